// Attention of drafts over the paged cache: the nodes of a tree of guessed tokens
// behind a sequence's context, checked in one pass.  The kernel is the prompts'
// (prompts.hpp), a tree's node for a token.
//
// Here the rows are few and the contexts long and uneven, so the work is cut evenly
// whatever the lengths: the steps (a tile of keys against a tile of rows) of all drafts
// in one line a key-value head, a workgroup an equal stretch of a head's line (16 to 64
// nodes over 32 contexts of 300 to 8000, 32/8 heads of 128 in bf16: 193 us, 243 with the
// prompts' shares).
//
// What bounds it: issue, as the prompts (those trees run at 460 TFLOP/s, the prompts at
// 600; 16 of 64 nodes after 4096 at 570, the keys' bytes are half of the time); for one
// small tree a chain.  8 nodes after 56 positions, one step, are 10.7 us, each further
// step of the one busy wave 1.4 to 1.5, a join 2.3 (8 steps, two pieces of four: 17.3).
// Past 128 dims one workgroup a CU, and registers spill: 16 trees of 16 to 64 nodes after
// 300 to 4000, 16/4 heads of 256 in bf16 104 us (32/8 heads of 128, as many products, 72),
// in f32 214 over bf16 and 173 over f16 (106 and 103).
// Tried and left: eight waves a workgroup, keys and values read once for up to 256 rows
// (the batch above 217 us instead of 222 call upon call, 9 drafts seen through a window of
// 333 28.6 instead of 24.7); three tiles of keys on their way instead of one (219 and 214);
// values read some products ahead, pages asked for beside the parents (the same).
#include <hip/hip_runtime.h>

#include "prompts.hpp"

namespace accel {
namespace {

// The entries' steps summed up, for more entries than a wave has lanes.  One workgroup.
template <int KT>
__global__ __launch_bounds__(1024) void draft_sums_kernel(KvCache c, Attention a, int tokens,
                                                          uint32_t* sums, uint32_t* fault) {
    __shared__ uint32_t sh[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int base = 0; base < a.n; base += 1024) {
        const int i = base + threadIdx.x;
        uint32_t v = 0;
        if (i < a.n) {
            const DraftWork w =
                work_of<KT>(a, held_by(c, a, i, fault).len, rows_of(a, i).count, tokens);
            v = w.tiles * w.steps;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d, 64);
            if (lane >= d) v = more_steps(v, up);
        }
        __syncthreads();
        if (lane == 63) sh[wave] = v;
        __syncthreads();
        uint32_t before = carry;
        for (int w = 0; w < 16; w++) {
            before = w < wave ? more_steps(before, sh[w]) : before;
            carry = more_steps(carry, sh[w]);
        }
        if (i < a.n) sums[i] = more_steps(before, v);
    }
}

// Key-value heads' lines, and rows of a tile.
struct Lines {
    int tokens;
    uint32_t heads;
};
Lines lines_of(const KvCache& c, const Attention& a) {
    const int group = a.heads / c.heads, per = prompt_heads(group);
    return {prompt_tokens(group), (uint32_t)(c.heads * ((group + per - 1) / per))};
}
constexpr int key_tile(int dim) { return dim <= 128 ? 64 : 32; }

}  // namespace

bool paged_tree_counts(const KvCache& c, const Attention& a) {
    const uint64_t tiles = (uint64_t)a.rows / lines_of(c, a).tokens + a.n;
    const uint64_t steps = ((uint64_t)c.slots << c.shift) / key_tile(c.dim) + 3;
    return tiles <= (kTooMany - 1) / steps;
}

hipError_t launch_paged_tree(Device* d, hipStream_t st, const KvCache& c, const Drafts& a,
                             int* status) {
    *status = ACCEL_OK;
    const Lines lines = lines_of(c, a);
    // two workgroups a CU of a 16-bit type up to 128 dims, else one
    const uint32_t slots = (uint32_t)d->cu_count * (!a.q_f32 && c.dim <= 128 ? 2 : 1);
    const uint32_t stretches = slots > lines.heads ? slots / lines.heads : 1;
    const uint32_t grid = lines.heads * stretches;
    const int wide = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    // a line of one stretch is not cut, so there are no joins and no tickets
    const size_t part_words =
        stretches > 1 ? 2 * (size_t)grid * 256 * (wide / 32 * 16 + 2) : 0;
    const bool summed = a.n > 64;
    const size_t sums_words = summed ? ((size_t)a.n + 1) & ~(size_t)1 : 0;
    uint32_t *tickets = nullptr, *sums = nullptr;
    float* parts = nullptr;
    if (part_words + sums_words) {
        char* ws = static_cast<char*>(workspace(d, st, (part_words + sums_words) * 4, status));
        if (!ws) return hipSuccess;
        tickets = reinterpret_cast<uint32_t*>(ws);
        parts = reinterpret_cast<float*>(ws + kWorkspaceCounterBytes);
        if (summed) sums = reinterpret_cast<uint32_t*>(parts + part_words);
    }
    if (summed) {
        if (key_tile(c.dim) == 64)
            hipLaunchKernelGGL(draft_sums_kernel<64>, dim3(1), dim3(1024), 0, st, c, a,
                               lines.tokens, sums, d->fault_dev);
        else
            hipLaunchKernelGGL(draft_sums_kernel<32>, dim3(1), dim3(1024), 0, st, c, a,
                               lines.tokens, sums, d->fault_dev);
    }
    const uint32_t stride = grid ? (uint32_t)(kWorkspaceCounterBytes / 4) / grid : 0;
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, c, a, sums, 0u, stretches, 0u,
                           tickets, stride, parts, d->fault_dev);
    };
    const bool full = c.dim == 64 || c.dim == 128 || c.dim == 256;
    const auto dims = [&](auto bf16, auto qt, auto pt) {
        constexpr bool B = decltype(bf16)::value;
        constexpr int Q = decltype(qt)::value, P = decltype(pt)::value;
        if (c.dim <= 64)
            full ? go(paged_prefill_kernel<B, Q, P, 64, true, 64, Drafts>)
                 : go(paged_prefill_kernel<B, Q, P, 64, false, 64, Drafts>);
        else if (c.dim <= 128)
            full ? go(paged_prefill_kernel<B, Q, P, 128, true, 64, Drafts>)
                 : go(paged_prefill_kernel<B, Q, P, 128, false, 64, Drafts>);
        else
            full ? go(paged_prefill_kernel<B, Q, P, 256, true, 32, Drafts>)
                 : go(paged_prefill_kernel<B, Q, P, 256, false, 32, Drafts>);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 3> three;
    if (a.q_f32) {
        if (c.bf16) dims(std::true_type(), three, three);
        else dims(std::false_type(), two, two);
    } else {
        if (c.bf16) dims(std::true_type(), one, one);
        else dims(std::false_type(), one, one);
    }
    return hipGetLastError();
}

}  // namespace accel
