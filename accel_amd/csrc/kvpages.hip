// The paged cache's bookkeeping and the moves of its pages: reservation,
// appended rows, branches, pages given back, compaction.
//
// Allocation takes the lowest free pages in a fixed order, so the same calls
// give the same tables whatever the schedule: one workgroup plans a call (a
// prefix sum over the entries' needs, then one over the free pages), and a
// second launch moves the data, which is all that takes bytes.
#include <hip/hip_runtime.h>

#include "internal.hpp"
#include "kvcache.hpp"

namespace accel {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPlan = 1024;            // lanes of a planning workgroup
constexpr int kPlanWaves = kPlan / 64;
constexpr int kScan = 16;              // pages a lane tests at once

// Workgroups of a launch, at most: one of 256 lanes holds fewer than 2^24, as a
// grid's lanes are counted in 32 bits.  The kernels below walk over more work
// than that.
constexpr int64_t kGrid = 1 << 22;
dim3 grid_of(size_t blocks) { return dim3((unsigned)(blocks < (size_t)kGrid ? blocks : kGrid)); }

// A word another lane of the workgroup changed with an atomic: read past the
// vector cache, which may hold the line as it was.
__device__ __forceinline__ uint32_t load_fresh(const uint32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The exclusive sum of v over the workgroup's lanes before this one; *total
// the sum of all.  sh holds kPlanWaves words.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sh, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, 64);
        if (lane >= d) incl += up;
    }
    __syncthreads();
    if (lane == 63) sh[wave] = incl;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
        before += w < wave ? sh[w] : 0u;
        sum += sh[w];
    }
    *total = sum;
    return before + incl - v;
}

// Pages first .. last that are free (FREE) or in use, in order, into list (up
// to `most`); returns how many there are, or most once there are as many.  A
// wave tests 64 consecutive pages a step, so the loads are whole lines and a
// page's rank is a population count of the wave's ballot.
// `ahead` are the first step's counts, where they have been read already.
struct Counts {
    uint32_t r[kScan];
};
__device__ __forceinline__ Counts read_counts(const uint32_t* refs, uint32_t base, uint32_t last,
                                              uint32_t past) {
    Counts c;
#pragma unroll
    for (int j = 0; j < kScan; j++) {
        const uint32_t page =
            base + (threadIdx.x >> 6) * 64 * kScan + j * 64 + (threadIdx.x & 63);
        c.r[j] = page < last ? refs[page] : past;
    }
    return c;
}
// The pool's first counts, which a search for free pages starts from: asked for
// before what the call needs is known, so the two wait for memory together.
__device__ __forceinline__ Counts read_ahead(const KvCache& c) {
    return read_counts(c.refs, 0, c.pages, 1);
}
template <bool FREE>
__device__ uint32_t list_pages(const uint32_t* refs, uint32_t first, uint32_t last, uint32_t* list,
                               uint32_t most, uint32_t* sh, const Counts* ahead = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t found = 0;
    for (uint32_t base = first; base < last && found < most; base += kPlan * kScan) {
        uint64_t hit[kScan];
        uint32_t count = 0;
        const uint32_t at = base + (uint32_t)wave * 64 * kScan;
        const Counts c = ahead && base == first
                             ? *ahead : read_counts(refs, base, last, FREE ? 1u : 0u);
#pragma unroll
        for (int j = 0; j < kScan; j++) {
            hit[j] = __ballot(FREE ? c.r[j] == 0 : c.r[j] != 0);
            count += __popcll(hit[j]);
        }
        uint32_t total;
        // a wave's count on its first lane alone, so that the scan's value
        // there is the sum of the waves before
        const uint32_t mine = block_scan(lane == 0 ? count : 0u, sh, &total);
        uint32_t rank = found + __shfl(mine, 0, 64);
#pragma unroll
        for (int j = 0; j < kScan; j++) {
            const uint32_t k = rank + __popcll(hit[j] & ((1ull << lane) - 1));
            if ((hit[j] >> lane & 1) && k < most) list[k] = at + j * 64 + lane;
            rank += __popcll(hit[j]);
        }
        found += total;
    }
    return found < most ? found : most;
}

// A planning workgroup's scratch in LDS, for calls small enough: each round trip
// to memory it saves is most of a microsecond.
constexpr uint32_t kNearMarks = 4096, kNearList = 2048;
struct PlanScratch {
    uint32_t sums[kPlanWaves];
    uint32_t marks[kNearMarks];
    uint32_t list[kNearList];
};

// For each sequence the first entry that names it, in sh or `far` [sequences];
// the whole workgroup calls it for all entries at once.
struct Marks {
    PlanScratch* sh;
    uint32_t* far;
    bool near;
    __device__ uint32_t first(uint32_t s) const {
        return near ? sh->marks[s] : load_fresh(far + s);
    }
};
__device__ Marks mark_first(const KvCache& c, const uint32_t* seqs, int n, PlanScratch* sh,
                            uint32_t* far) {
    const Marks m = {sh, far, c.sequences <= kNearMarks};
    if (m.near) {
        for (uint32_t s = threadIdx.x; s < c.sequences; s += kPlan) sh->marks[s] = 0xffffffffu;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kPlan)
            if (seqs[i] < c.sequences) atomicMin(&sh->marks[seqs[i]], (uint32_t)i);
    } else {
        for (int i = threadIdx.x; i < n; i += kPlan)
            if (seqs[i] < c.sequences)
                __hip_atomic_store(far + seqs[i], 0xffffffffu, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kPlan)
            if (seqs[i] < c.sequences)
                __hip_atomic_fetch_min(far + seqs[i], (uint32_t)i, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return m;
}

__global__ __launch_bounds__(256) void kv_fill_kernel(uint32_t* p, size_t n, uint32_t v) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = v;
}

// Pages for the positions each entry grows by.  Scratch: list [pages], first
// [n] (an entry's first place in the list), mark [sequences].
__global__ __launch_bounds__(kPlan) void kv_reserve_kernel(KvCache c, const uint32_t* seqs,
                                                           const uint32_t* grow, int n,
                                                           uint32_t* list, uint32_t* first,
                                                           uint32_t* mark, uint32_t* fault) {
    __shared__ PlanScratch sh;
    __shared__ uint32_t short_sh[2];
    const uint32_t cap = c.slots << c.shift, up = (1u << c.shift) - 1;
    const Counts ahead = read_ahead(c);
    Marks marks = {};
    if (seqs) marks = mark_first(c, seqs, n, &sh, mark);
    const auto need_of = [&](uint32_t s, int i) {
        const uint32_t len = c.lens[s];
        return ((len + grow[i] + up) >> c.shift) - ((len + up) >> c.shift);
    };
    // what each entry needs, and where its pages begin in the list; an entry
    // that cannot be served is marked and needs none
    constexpr uint32_t kLeftOut = 0xffffffffu;
    uint32_t needed = 0;
    for (int base = 0; base < n; base += kPlan) {
        const int i = base + threadIdx.x;
        uint32_t need = 0;
        bool ok = false;
        if (i < n) {
            const uint32_t s = sequence_of(c, seqs, i, fault);
            if (s != kNoSequence) {
                if (seqs && marks.first(s) != (uint32_t)i) {
                    report(fault, kFaultKvSequence);
                } else {
                    const uint32_t len = c.lens[s], g = grow[i];
                    if (len > cap || g > cap - len) {
                        report(fault, kFaultKvRoom);
                    } else {
                        need = need_of(s, i);
                        ok = true;
                    }
                }
            }
        }
        // the sum stays below sequences * slots, which is below 2^31
        uint32_t total;
        const uint32_t at = needed + block_scan(need, sh.sums, &total);
        if (i < n) first[i] = ok ? at : kLeftOut;
        needed += total;
    }
    const uint32_t want = needed < c.pages ? needed : c.pages;
    if (want <= kNearList) list = sh.list;
    __syncthreads();
    const uint32_t found =
        want ? list_pages<true>(c.refs, 0, c.pages, list, want, sh.sums, &ahead) : 0;
    __syncthreads();
    if (found < needed) {
        // The pool is short: the entries are gone through in order, each served
        // that fits into what those before it left.  A pass over the entries at
        // hand serves those before the first that does not fit, and leaves out
        // that one and whatever needs more than is left then; so a pass that
        // serves few leaves out much, and few passes are usual (600 entries
        // made to need one each: 0.5 ms).
        uint32_t left = found;
        for (int base = 0; base < n; base += kPlan) {
            const int i = base + threadIdx.x;
            bool open = i < n && first[i] != kLeftOut;
            const uint32_t need = open ? need_of(seqs ? seqs[i] : (uint32_t)i, i) : 0;
            for (;;) {
                if (open && need > left) {
                    open = false;
                    first[i] = kLeftOut;
                    report(fault, kFaultKvRoom);
                }
                // the scan's barriers stand between the last pass's reads of
                // short_sh and this one's reset
                uint32_t total;
                const uint32_t at = block_scan(open ? need : 0u, sh.sums, &total);
                if (threadIdx.x == 0) short_sh[0] = kPlan, short_sh[1] = 0;
                __syncthreads();
                const bool over = open && (at > left || need > left - at);
                if (over) atomicMin(&short_sh[0], (uint32_t)threadIdx.x);
                __syncthreads();
                const uint32_t stop = short_sh[0];
                if (open && threadIdx.x < stop) {
                    first[i] = found - left + at;
                    open = false;
                    atomicMax(&short_sh[1], at + need);
                }
                __syncthreads();
                left -= short_sh[1];
                if (stop == kPlan) break;
            }
        }
        __syncthreads();
    }
    // a wave an entry: the slots of a long prompt are filled side by side
    const int lane = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < n; i += kPlanWaves) {
        const uint32_t at = first[i];
        if (at == kLeftOut) continue;
        const uint32_t s = seqs ? seqs[i] : (uint32_t)i;
        const uint32_t len = c.lens[s], g = grow[i];
        const uint32_t have = (len + up) >> c.shift, need = need_of(s, i);
        for (uint32_t j = lane; j < need; j += 64) {
            const uint32_t page = list[at + j];
            c.tables[(size_t)s * c.slots + have + j] = page;
            c.refs[page] = 1;
        }
        if (lane == 0 && g) c.lens[s] = len + g;
    }
}

// f32 or 16-bit values, eight of them, as the cache's 16-bit type.
__device__ __forceinline__ uint16_t narrow(float f, bool bf16) {
    if (bf16) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// One lane eight elements of a row of keys and of values: 16 bytes stored to
// each.  HBM-bound; a row's [kv_heads, dim] goes to kv_heads places of dim
// elements, and rows of one sequence follow each other within a head's part of
// the page, so stores fill whole lines.
__device__ __forceinline__ void append_item(const KvCache& c, size_t layer_elems, const void* k,
                                            const void* v, int32_t dtype, const uint32_t* seqs,
                                            const uint32_t* offsets, int n, uint32_t row,
                                            uint32_t part, uint32_t* fault) {
    int e = row;
    uint32_t left = 1;                  // rows of the entry from this one on
    if (offsets) {
        e = entry_of(offsets, n, row);
        if (e < 0) return;
        left = offsets[e + 1] - row;
    }
    const uint32_t s = sequence_of(c, seqs, e, fault);
    if (s == kNoSequence) return;
    const uint32_t len = length_of(c, s);
    if (left > len) {
        report(fault, kFaultKvPage);
        return;
    }
    const uint32_t pos = len - left;
    const uint32_t page = c.tables[(size_t)s * c.slots + (pos >> c.shift)];
    if (page >= c.pages) {
        report(fault, kFaultKvPage);
        return;
    }
    const uint32_t chunks = c.dim >> 3, h = part / chunks, d = (part - h * chunks) * 8;
    // A sequence that was shortened may end in a page that a branch has too: no row is
    // stored there.  Asked for beside the row, which is as far away.
    const uint32_t names = c.refs[page];
    const size_t from = ((size_t)row * c.heads + h) * c.dim + d;
    const size_t to = layer_elems +
                      ((((size_t)page * c.heads + h) << c.shift) + (pos & ((1u << c.shift) - 1))) *
                          c.dim + d;
    u32x4 out[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const void* src = x ? v : k;
        u32x4& o = out[x];
        if (dtype == ACCEL_F32) {
            const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(src) + from);
            const u32x4 a = p[0], b = p[1];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u32x4 w = j < 2 ? a : b;
                const float f0 = __uint_as_float(w[2 * (j & 1)]);
                const float f1 = __uint_as_float(w[2 * (j & 1) + 1]);
                o[j] = narrow(f0, c.bf16) | (uint32_t)narrow(f1, c.bf16) << 16;
            }
        } else {
            o = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(src) + from);
            if ((dtype == ACCEL_BF16) != c.bf16) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[j] = narrow(widen((uint16_t)o[j], !c.bf16), c.bf16) |
                           (uint32_t)narrow(widen((uint16_t)(o[j] >> 16), !c.bf16), c.bf16) << 16;
            }
        }
    }
    if (names > 1) {
        report(fault, kFaultKvPage);
        return;
    }
    *reinterpret_cast<u32x4*>(c.keys + to) = out[0];
    *reinterpret_cast<u32x4*>(c.values + to) = out[1];
}
__global__ __launch_bounds__(256) void kv_append_kernel(KvCache c, size_t layer_elems,
                                                        const void* k, const void* v,
                                                        int32_t dtype, const uint32_t* seqs,
                                                        const uint32_t* offsets, int n, int rows,
                                                        uint32_t* fault) {
    const uint32_t per = (uint32_t)c.heads * (c.dim >> 3);
    const size_t items = (size_t)rows * per;
    for (size_t item = (size_t)blockIdx.x * 256 + threadIdx.x; item < items;
         item += (size_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(item / per);
        append_item(c, layer_elems, k, v, dtype, seqs, offsets, n, row,
                    (uint32_t)(item - (size_t)row * per), fault);
    }
}

// A branch as planned: how many whole pages it shares, and the copy of the
// last one (from, to; ACCEL_KV_NONE: none).  ok: its length and one, 0 for an
// entry left out.
struct Branch {
    uint32_t whole, from, to, ok;
};

// Plans the branches and gives the children their lengths and last pages.
// Scratch: list [n] free pages, plan [n], mark [sequences].
__global__ __launch_bounds__(kPlan) void kv_fork_plan_kernel(KvCache c, const uint32_t* parents,
                                                             const uint32_t* children, int n,
                                                             uint32_t* list, Branch* plan,
                                                             uint32_t* mark, uint32_t* fault) {
    __shared__ PlanScratch sh;
    const Counts ahead = read_ahead(c);
    const Marks marks = mark_first(c, children, n, &sh, mark);
    uint32_t needed = 0, child = kNoSequence;
    Branch b = {};
    for (int base = 0; base < n; base += kPlan) {
        const int i = base + threadIdx.x;
        b = {0, ACCEL_KV_NONE, ACCEL_KV_NONE, 0};
        if (i < n) {
            const uint32_t p = parents[i], s = child = children[i];
            if (p < c.sequences && s < c.sequences) {
                if (marks.first(s) != (uint32_t)i || c.lens[s] != 0) {
                    report(fault, kFaultKvSequence);
                } else {
                    const uint32_t len = length_of(c, p);
                    b.ok = len + 1;
                    b.whole = len >> c.shift;
                    if (len & ((1u << c.shift) - 1)) {
                        const uint32_t last = c.tables[(size_t)p * c.slots + b.whole];
                        if (last < c.pages) b.from = last;
                        else report(fault, kFaultKvPage), b.ok = 0;
                    }
                }
            } else if ((p >= c.sequences && p != ACCEL_KV_NONE) ||
                       (s >= c.sequences && s != ACCEL_KV_NONE)) {
                report(fault, kFaultKvSequence);
            }
        }
        uint32_t total;
        const bool wants = b.ok && b.from != ACCEL_KV_NONE;
        const uint32_t at = needed + block_scan(wants ? 1u : 0u, sh.sums, &total);
        // the place in the list until the list is there
        if (i < n) {
            b.to = wants ? at : ACCEL_KV_NONE;
            if (n > kPlan) plan[i] = b;
        }
        needed += total;
    }
    const uint32_t want = needed < c.pages ? needed : c.pages;
    if (want <= kNearList) list = sh.list;
    __syncthreads();
    const uint32_t found =
        want ? list_pages<true>(c.refs, 0, c.pages, list, want, sh.sums, &ahead) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlan) {
        if (n > kPlan) {
            b = plan[i];
            child = children[i];
        }
        if (b.ok && b.to != ACCEL_KV_NONE) {
            if (b.to < found) {
                b.to = list[b.to];
                c.refs[b.to] = 1;
            } else {
                report(fault, kFaultKvRoom);
                b = {0, ACCEL_KV_NONE, ACCEL_KV_NONE, 0};
            }
        }
        plan[i] = b;
        if (b.ok > 1) c.lens[child] = b.ok - 1;
    }
}

// Copies one page's part of one layer: lanes 16 bytes apart, eight loads in
// flight a lane.
__device__ __forceinline__ void copy_page(const uint16_t* from, uint16_t* to, size_t elems) {
    const u32x4* src = reinterpret_cast<const u32x4*>(from);
    u32x4* dst = reinterpret_cast<u32x4*>(to);
    const uint32_t n = (uint32_t)(elems >> 3);
    for (uint32_t base = threadIdx.x; base < n; base += 256 * 8) {
        u32x4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (base + 256 * j < n) v[j] = src[base + 256 * j];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (base + 256 * j < n) dst[base + 256 * j] = v[j];
    }
}

// The copy of pair k's page in part `part` (a layer's keys or values).
__device__ __forceinline__ void copy_part(const KvCache& c, uint32_t from, uint32_t to,
                                          uint32_t part) {
    const size_t elems = c.page_elems();
    const size_t layer = (size_t)(part >> 1) * c.pages;
    uint16_t* base = part & 1 ? c.values : c.keys;
    copy_page(base + (layer + from) * elems, base + (layer + to) * elems, elems);
}

// Blocks 2 * layers a branch: its last page's copy; and one more a branch for
// its row of the table and the shared pages' counts.  (Blocks in all: below 2^31.)
__global__ __launch_bounds__(256) void kv_fork_kernel(KvCache c, const uint32_t* parents,
                                                      const uint32_t* children,
                                                      const Branch* plan, int n) {
    const uint32_t parts = 2 * (uint32_t)c.layers + 1, work = (uint32_t)n * parts;
    for (uint32_t w = blockIdx.x; w < work; w += gridDim.x) {
        const uint32_t i = w / parts, part = w - i * parts;
        const Branch b = plan[i];
        if (!b.ok) continue;
        if (part + 1 < parts) {
            if (b.to != ACCEL_KV_NONE) copy_part(c, b.from, b.to, part);
            continue;
        }
        const uint32_t* from = c.tables + (size_t)parents[i] * c.slots;
        uint32_t* to = c.tables + (size_t)children[i] * c.slots;
        for (uint32_t j = threadIdx.x; j < b.whole; j += 256) {
            const uint32_t page = from[j];
            to[j] = page < c.pages ? page : ACCEL_KV_NONE;
            if (page < c.pages)
                __hip_atomic_fetch_add(c.refs + page, 1u, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
        }
        if (threadIdx.x == 0 && b.to != ACCEL_KV_NONE) to[b.whole] = b.to;
    }
}

// Blocks 2 * layers a pair, below 2^31 in all.
__global__ __launch_bounds__(256) void kv_copy_kernel(KvCache c, const uint32_t* src,
                                                      const uint32_t* dst, int n,
                                                      uint32_t* fault) {
    const uint32_t parts = 2 * (uint32_t)c.layers, work = (uint32_t)n * parts;
    for (uint32_t w = blockIdx.x; w < work; w += gridDim.x) {
        const uint32_t i = w / parts, part = w - i * parts;
        const uint32_t from = src[i], to = dst[i];
        if (from >= c.pages || to >= c.pages) {
            if (from != ACCEL_KV_NONE && to != ACCEL_KV_NONE && threadIdx.x == 0)
                report(fault, kFaultKvSequence);
            continue;
        }
        if (from != to) copy_part(c, from, to, part);
    }
}

// A block a sequence.  An entry is claimed by exchanging it for ACCEL_KV_NONE,
// so a sequence named twice gives each page back once.
__global__ __launch_bounds__(256) void kv_free_kernel(KvCache c, const uint32_t* seqs, int n,
                                                      int64_t window, int64_t sinks,
                                                      uint32_t* fault) {
    for (uint32_t i = blockIdx.x; i < (uint32_t)n; i += gridDim.x) {
        const uint32_t s = sequence_of(c, seqs, (int)i, fault);
        if (s == kNoSequence) continue;
        uint32_t lo = 0, hi = c.slots;
        if (window) {
            // slots wholly past the sinks and wholly before the window of the
            // query at the last position
            const int64_t len = length_of(c, s);
            const int64_t first = (sinks + (1 << c.shift) - 1) >> c.shift;
            lo = (uint32_t)(first < (int64_t)c.slots ? first : (int64_t)c.slots);
            hi = len > window ? (uint32_t)((len - window) >> c.shift) : 0;
        }
        uint32_t* row = c.tables + (size_t)s * c.slots;
        for (uint32_t j = lo + threadIdx.x; j < hi; j += 256) {
            if (row[j] == ACCEL_KV_NONE) continue;
            const uint32_t page = __hip_atomic_exchange(row + j, ACCEL_KV_NONE, __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT);
            if (page < c.pages)
                __hip_atomic_fetch_sub(c.refs + page, 1u, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
        }
        if (!window && threadIdx.x == 0) c.lens[s] = 0;
    }
}

// The moves of a compaction.  Scratch: head[0] = how many, head[1] = pages in
// use, to [pages] the free pages below, from [pages] the pages that move, remap
// [pages] the new number of each page at or past head[1] (its own if it was
// not in use).
__global__ __launch_bounds__(kPlan) void kv_compact_plan_kernel(KvCache c, uint32_t* head,
                                                                uint32_t* to, uint32_t* from,
                                                                uint32_t* remap, uint32_t* live) {
    __shared__ uint32_t sh[kPlanWaves];
    uint32_t count = 0;
    for (uint32_t base = 0; base < c.pages; base += kPlan * kScan) {
#pragma unroll
        for (int j = 0; j < kScan; j++) {
            const uint32_t page = base + j * kPlan + threadIdx.x;
            count += page < c.pages && c.refs[page] != 0 ? 1u : 0u;
        }
    }
    uint32_t used;
    block_scan(count, sh, &used);
    for (uint32_t p = used + threadIdx.x; p < c.pages; p += kPlan) remap[p] = p;
    const uint32_t holes = list_pages<true>(c.refs, 0, used, to, c.pages, sh);
    __syncthreads();
    list_pages<false>(c.refs, used, c.pages, from, c.pages, sh);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < holes; k += kPlan) {
        const uint32_t a = from[k], b = to[k];
        remap[a] = b;
        c.refs[b] = c.refs[a];
        c.refs[a] = 0;
    }
    if (threadIdx.x == 0) {
        head[0] = holes;
        head[1] = used;
        if (live) *live = used;
    }
}

// A persistent grid over the planned copies; then the tables' entries.
__global__ __launch_bounds__(256) void kv_compact_kernel(KvCache c, const uint32_t* head,
                                                         const uint32_t* to,
                                                         const uint32_t* from,
                                                         const uint32_t* remap) {
    const uint32_t moves = head[0], used = head[1];
    if (moves == 0) return;
    const uint32_t parts = 2 * (uint32_t)c.layers;
    const size_t work = (size_t)moves * parts;
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const uint32_t k = (uint32_t)(w / parts);
        copy_part(c, from[k], to[k], (uint32_t)(w - (size_t)k * parts));
    }
    const size_t entries = (size_t)c.sequences * c.slots;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < entries;
         i += (size_t)gridDim.x * 256) {
        const uint32_t page = c.tables[i];
        if (page >= used && page < c.pages) c.tables[i] = remap[page];
    }
}

}  // namespace

hipError_t launch_kv_clear(hipStream_t st, const KvCache& c) {
    const size_t entries = (size_t)c.sequences * c.slots;
    const auto fill = [st](uint32_t* p, size_t n, uint32_t v) {
        hipLaunchKernelGGL(kv_fill_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p,
                           n, v);
    };
    fill(c.refs, c.pages, 0);
    fill(c.tables, entries, ACCEL_KV_NONE);
    fill(c.lens, c.sequences, 0);
    return hipGetLastError();
}

namespace {
// Scratch words past the workspace's counters.
uint32_t* scratch_words(Device* d, hipStream_t st, size_t words, int* status) {
    char* ws = static_cast<char*>(workspace(d, st, words * 4, status));
    return ws ? reinterpret_cast<uint32_t*>(ws + kWorkspaceCounterBytes) : nullptr;
}
}  // namespace

hipError_t launch_kv_reserve(Device* d, hipStream_t st, const KvCache& c, const uint32_t* seqs,
                             const uint32_t* grow, int n, int* status) {
    uint32_t* w = scratch_words(d, st, (size_t)c.pages + n + (seqs ? c.sequences : 0), status);
    if (!w) return hipSuccess;
    hipLaunchKernelGGL(kv_reserve_kernel, dim3(1), dim3(kPlan), 0, st, c, seqs, grow, n, w,
                       w + c.pages, w + c.pages + n, d->fault_dev);
    return hipGetLastError();
}

hipError_t launch_kv_append(Device* d, hipStream_t st, const KvCache& c, int64_t layer,
                            const void* k, const void* v, int32_t dtype, const uint32_t* seqs,
                            const uint32_t* offsets, int n, int rows) {
    const size_t items = (size_t)rows * c.heads * (c.dim >> 3);
    hipLaunchKernelGGL(kv_append_kernel, grid_of((items + 255) / 256), dim3(256), 0, st, c,
                       (size_t)layer * c.pages * c.page_elems(), k, v, dtype, seqs, offsets, n,
                       rows, d->fault_dev);
    return hipGetLastError();
}

hipError_t launch_kv_fork(Device* d, hipStream_t st, const KvCache& c, const uint32_t* parents,
                          const uint32_t* children, int n, int* status) {
    uint32_t* w = scratch_words(d, st, (size_t)n * 5 + c.sequences, status);
    if (!w) return hipSuccess;
    Branch* plan = reinterpret_cast<Branch*>(w);
    uint32_t* list = w + (size_t)n * 4;
    hipLaunchKernelGGL(kv_fork_plan_kernel, dim3(1), dim3(kPlan), 0, st, c, parents, children, n,
                       list, plan, list + n, d->fault_dev);
    hipLaunchKernelGGL(kv_fork_kernel, grid_of((size_t)n * (2 * c.layers + 1)), dim3(256), 0, st, c,
                       parents, children, plan, n);
    return hipGetLastError();
}

hipError_t launch_kv_free(Device* d, hipStream_t st, const KvCache& c, const uint32_t* seqs,
                          int n, int64_t window, int64_t sinks) {
    hipLaunchKernelGGL(kv_free_kernel, grid_of((size_t)n), dim3(256), 0, st, c, seqs, n, window,
                       sinks, d->fault_dev);
    return hipGetLastError();
}

hipError_t launch_kv_compact(Device* d, hipStream_t st, const KvCache& c, uint32_t* live,
                             int* status) {
    uint32_t* w = scratch_words(d, st, (size_t)c.pages * 3 + 4, status);
    if (!w) return hipSuccess;
    uint32_t *head = w, *to = w + 4, *from = to + c.pages, *remap = from + c.pages;
    hipLaunchKernelGGL(kv_compact_plan_kernel, dim3(1), dim3(kPlan), 0, st, c, head, to, from,
                       remap, live);
    hipLaunchKernelGGL(kv_compact_kernel, dim3((unsigned)(d->cu_count * 8)), dim3(256), 0, st, c,
                       head, to, from, remap);
    return hipGetLastError();
}

hipError_t launch_kv_copy(Device* d, hipStream_t st, const KvCache& c, const uint32_t* src,
                          const uint32_t* dst, int n) {
    hipLaunchKernelGGL(kv_copy_kernel, grid_of((size_t)n * (2 * c.layers)), dim3(256), 0, st, c,
                       src, dst, n, d->fault_dev);
    return hipGetLastError();
}

}  // namespace accel
