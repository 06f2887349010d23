// Attention of drafts over the paged cache: the nodes of a tree of guessed tokens
// behind a sequence's context, checked in one pass.  The kernel is the prompts'
// (prompts.hpp), a tree's node for a token.
#include <hip/hip_runtime.h>

#include "prompts.hpp"

namespace accel {

hipError_t launch_paged_tree(Device* d, hipStream_t st, const KvCache& c, const Drafts& a,
                             int* status) {
    return launch_prompts(d, st, c, a, status);
}

}  // namespace accel
