// What follows the attention of drafts: the walk down a tree along the tokens that
// were sampled, and the accepted nodes' keys and values moved up behind their
// context.  Both are chains of a few dependent reads (a walk 2.2 us, of 256 trees of up
// to 64 nodes 4.2); the second's bytes are those of the rows that move, in every layer
// (8 of up to 64 nodes of 48 sequences, 16 layers, 8 heads of 128: 20 MB read and written
// together in 7.8 us after a plan of 3.7).  A launch of its own for the plan: whether a
// sequence is served, and its pages shared, has to be known before the first row moves.
#include <hip/hip_runtime.h>

#include "internal.hpp"
#include "kvcache.hpp"

namespace accel {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Workgroups of a launch, at most; the kernels walk over more work than that.
constexpr int64_t kGrid = 1 << 22;
dim3 grid_of(int64_t blocks) { return dim3((unsigned)(blocks < kGrid ? blocks : kGrid)); }

// An entry's rows, [first, first + count) of all.
struct Rows {
    uint32_t first, count;
};
__device__ __forceinline__ Rows rows_of(const uint32_t* offsets, uint32_t all, int64_t i) {
    const uint32_t x = offsets[i], y = offsets[i + 1];
    const uint32_t lo = x < all ? x : all, hi = y < all ? y : all;
    return {lo, hi > lo ? hi - lo : 0};
}

// A wave a draft, its nodes in the lanes' registers: a step asks all nodes at once
// whether they are the next, and the lowest that is becomes the place.  A child is
// past its parent, so the walk ends.
constexpr int kEach = ACCEL_DRAFT_NODES / 64;

__global__ __launch_bounds__(64) void tree_accept_kernel(
    const uint32_t* tokens, const uint32_t* parents, const uint32_t* offsets,
    const uint32_t* sampled, uint32_t rows, int64_t n, uint32_t width, uint32_t* path,
    uint32_t* counts, uint32_t* next, uint32_t* fault) {
    const uint32_t lane = threadIdx.x;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const Rows r = rows_of(offsets, rows, i);
        uint32_t* out = path + (size_t)i * width;
        uint32_t count = 0, last = ACCEL_KV_NONE;
        const bool refused = r.count > ACCEL_DRAFT_NODES;
        if (refused) {
            if (lane == 0) report(fault, kFaultDraft);
        } else if (r.count) {
            uint32_t token[kEach], parent[kEach], drawn[kEach];
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                const uint32_t t = e * 64 + lane;
                const bool in = t < r.count;
                token[e] = in ? tokens[r.first + t] : 0;
                parent[e] = in ? parents[r.first + t] : ACCEL_KV_NONE;
                drawn[e] = in ? sampled[r.first + t] : ACCEL_KV_NONE;
            }
            uint32_t at = 0;
            for (;;) {
                uint32_t mine = drawn[0];
#pragma unroll
                for (int e = 1; e < kEach; e++) mine = at >> 6 == (uint32_t)e ? drawn[e] : mine;
                last = __builtin_amdgcn_readlane(mine, at & 63);
                if (lane == 0) out[count] = at;
                count++;
                if (count == width || last == ACCEL_KV_NONE) break;
                uint32_t found = ACCEL_KV_NONE;
#pragma unroll
                for (int e = kEach - 1; e >= 0; e--) {
                    const uint64_t fits = __ballot(parent[e] == at && token[e] == last &&
                                                   e * 64 + lane > at);
                    if (fits) found = e * 64 + __builtin_ctzll(fits);
                }
                if (found == ACCEL_KV_NONE) break;
                at = found;
            }
        }
        // a count of 0 alone would have the keep take all of the sequence's nodes back
        for (uint32_t c = count + lane; c < width; c += 64)
            out[c] = refused && c == 0 ? ACCEL_DRAFT_REFUSED : ACCEL_KV_NONE;
        if (lane == 0) {
            counts[i] = count;
            next[i] = last;
        }
    }
}

// What an entry of a keep does.  count is kLeave for one that stays as it is.
constexpr uint32_t kLeave = 0xffffffffu;
// A sequence's length while its entry is at work: no table holds as many.
constexpr uint32_t kClaimed = 0xffffffffu;
struct Keep {
    uint32_t seq, before, after;      // its length, and its length then
    uint32_t count;                   // rows kept
};

// A wave an entry.  A sequence is claimed by exchanging its length, so of two
// entries that name it one is served.  pages [n, width]: where row c comes from and
// goes to; the same page and place where it stays.
__global__ __launch_bounds__(64) void kv_keep_plan_kernel(KvCache c, const uint32_t* seqs,
                                                          const uint32_t* offsets,
                                                          const uint32_t* path, uint32_t width,
                                                          const uint32_t* counts, int64_t n,
                                                          Keep* plan, uint2* pages,
                                                          uint32_t* fault) {
    const uint32_t lane = threadIdx.x;
    const uint32_t cap = c.slots << c.shift;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const uint32_t s = sequence_of(c, seqs, (int)i, lane ? nullptr : fault);
        Keep k = {s, 0, 0, kLeave};
        if (s != kNoSequence) {
            const uint32_t count = counts[i];
            const uint32_t x = offsets[i], y = offsets[i + 1], nodes = y > x ? y - x : 0;
            uint32_t len = 0;
            if (lane == 0)
                len = __hip_atomic_exchange(c.lens + s, kClaimed, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
            len = __builtin_amdgcn_readfirstlane(len);
            uint32_t wrong = 0;
            if (len == kClaimed) {
                k.seq = kNoSequence;      // the other entry gives it its length
                wrong = kFaultKvSequence;
            } else if (len > cap || nodes > len) {
                wrong = kFaultKvPage;
            } else if (count > width || count > nodes ||
                       (count == 0 && path[(size_t)i * width] == ACCEL_DRAFT_REFUSED)) {
                wrong = kFaultDraft;
            } else {
                const uint32_t first = len - nodes;
                const uint32_t* table = c.tables + (size_t)s * c.slots;
                for (uint32_t j = lane; j < count; j += 64) {
                    const uint32_t* p = path + (size_t)i * width + j;
                    const uint32_t t = p[0];
                    uint2 page = {0, 0};
                    if (t >= nodes || (j && p[-1] >= t)) {
                        wrong |= kFaultDraft;
                    } else if (t != j) {
                        page = {table[(first + t) >> c.shift], table[(first + j) >> c.shift]};
                        if (page.x >= c.pages || page.y >= c.pages) wrong |= kFaultKvPage;
                        // a page that another sequence reads too
                        else if (c.refs[page.y] != 1) wrong |= kFaultDraft;
                    }
                    pages[(size_t)i * width + j] = page;
                }
            }
            k.before = k.after = len;
            if (!__any(wrong != 0)) {
                k.count = count;
                k.after = len - nodes + count;
            } else if (wrong) {
                report(fault, wrong);
            }
        }
        if (lane == 0) plan[i] = k;
    }
}

// A wave an entry's keys or values of one head and layer: lanes 16 bytes apart over
// the rows that move, up to kDeep loads in flight a lane.  A row's target is never
// past its source and paths ascend, so no row is written over before the loads that
// a later step makes of it.  The first wave of an entry then sets its length and
// gives back its pages; the places are in the plan, so no wave needs the table.
constexpr int kDeep = 4;

__global__ __launch_bounds__(256) void kv_keep_kernel(KvCache c, const uint32_t* path,
                                                      uint32_t width, int64_t n,
                                                      const Keep* plan, const uint2* pages) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t chunks = (uint32_t)c.dim >> 3;
    const uint32_t parts = 2 * (uint32_t)c.layers * (uint32_t)c.heads;
    const uint32_t mask = (1u << c.shift) - 1;
    const uint64_t work = (uint64_t)n * parts;
    for (uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); w < work;
         w += (uint64_t)gridDim.x * 4) {
        const uint64_t i = w / parts;
        const uint32_t part = (uint32_t)(w - i * parts);
        const Keep k = plan[i];
        if (k.seq == kNoSequence) continue;
        if (k.count != kLeave) {
            const uint32_t plane = part & 1, lh = part >> 1;
            const uint32_t layer = lh / (uint32_t)c.heads, head = lh - layer * (uint32_t)c.heads;
            uint16_t* base = (plane ? c.values : c.keys) +
                             (size_t)layer * c.pages * c.page_elems() +
                             (((size_t)head << c.shift) * c.dim);
            const uint32_t first = k.after - k.count, items = k.count * chunks;
            for (uint32_t x0 = 0; x0 < items; x0 += 64 * kDeep) {
                u32x4 v[kDeep];
                uint16_t* to[kDeep];
#pragma unroll
                for (int e = 0; e < kDeep; e++) {
                    const uint32_t x = x0 + e * 64 + lane;
                    to[e] = nullptr;
                    if (x >= items) continue;
                    const uint32_t j = x / chunks, d = (x - j * chunks) * 8;
                    const uint32_t t = path[(size_t)i * width + j];
                    if (t == j) continue;
                    const uint2 page = pages[(size_t)i * width + j];
                    const auto at = [&](uint32_t pg, uint32_t pos) {
                        return base + pg * c.page_elems() + (size_t)(pos & mask) * c.dim + d;
                    };
                    v[e] = *reinterpret_cast<const u32x4*>(at(page.x, first + t));
                    to[e] = at(page.y, first + j);
                }
                // all loads of the step before its stores
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __builtin_amdgcn_s_waitcnt(0x0f70);
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
                for (int e = 0; e < kDeep; e++)
                    if (to[e]) *reinterpret_cast<u32x4*>(to[e]) = v[e];
            }
        }
        if (part == 0) {
            const uint32_t lo = (k.after + mask) >> c.shift, hi = (k.before + mask) >> c.shift;
            uint32_t* row = c.tables + (size_t)k.seq * c.slots;
            if (k.count != kLeave)
                for (uint32_t j = lo + lane; j < hi && j < c.slots; j += 64) {
                    const uint32_t page = row[j];
                    row[j] = ACCEL_KV_NONE;
                    if (page < c.pages)
                        __hip_atomic_fetch_sub(c.refs + page, 1u, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT);
                }
            if (lane == 0) c.lens[k.seq] = k.after;
        }
    }
}

}  // namespace

hipError_t launch_tree_accept(Device* d, hipStream_t st, const uint32_t* tokens,
                              const uint32_t* parents, const uint32_t* offsets,
                              const uint32_t* sampled, int64_t rows, int64_t n, int64_t width,
                              uint32_t* path, uint32_t* counts, uint32_t* next) {
    hipLaunchKernelGGL(tree_accept_kernel, grid_of(n), dim3(64), 0, st, tokens, parents, offsets,
                       sampled, (uint32_t)rows, n, (uint32_t)width, path, counts, next,
                       d->fault_dev);
    return hipGetLastError();
}

hipError_t launch_kv_keep(Device* d, hipStream_t st, const KvCache& c, const uint32_t* seqs,
                          const uint32_t* offsets, const uint32_t* path, int64_t width,
                          const uint32_t* counts, int64_t n, int* status) {
    const size_t plan_bytes = (size_t)n * sizeof(Keep);
    char* ws = static_cast<char*>(
        workspace(d, st, plan_bytes + (size_t)n * width * sizeof(uint2), status));
    if (!ws) return hipSuccess;
    Keep* plan = reinterpret_cast<Keep*>(ws + kWorkspaceCounterBytes);
    uint2* pages = reinterpret_cast<uint2*>(ws + kWorkspaceCounterBytes + plan_bytes);
    hipLaunchKernelGGL(kv_keep_plan_kernel, grid_of(n), dim3(64), 0, st, c, seqs, offsets, path,
                       (uint32_t)width, counts, n, plan, pages, d->fault_dev);
    const int64_t work = n * 2 * c.layers * c.heads;
    hipLaunchKernelGGL(kv_keep_kernel, grid_of((work + 3) / 4), dim3(256), 0, st, c, path,
                       (uint32_t)width, n, plan, pages);
    return hipGetLastError();
}

}  // namespace accel
