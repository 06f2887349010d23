// Attention over the paged cache: for the query at position p of a sequence,
//
//   out = sum_j e_j v_j / sum_j e_j,   e_j = exp(scale q.k_j - m),
//
// m the largest score, over the keys j <= p with p - j < window or j < sinks
// (all j <= p without a window).
//
// One new token a sequence (paged_decode_kernel).  The bytes of the keys and
// values bound it: each is read once for up to 16 query heads of its group, once
// more for every further 16.  A wave takes 32 keys at a time against those heads as
// S^T = K Q^T and O^T += V^T P^T on the matrix cores, everything in registers:
//
// - K goes from memory to the A operand as it is (a lane 16 bytes of one key a
//   step).  Which key is which row is free, and is chosen so that a lane's
//   eight scores (C layout: column = query, rows 4 (lane / 16) + i of two
//   tiles) are eight consecutive keys: exactly its part of P^T's B operand.
// - A lane loads V for those eight keys, DIM / 16 consecutive dims of each, and
//   turns the block by byte permutes (half an instruction an element) into A
//   operands with the eight keys along k; which dim is which row is free too.
// - The running maximum is only moved when some weight would pass 2^8 of it (over
//   an f16 cache 2^6: kOver, kLift), so most steps have no exchange between
//   lanes.  A lane sums its own weights.
//
// Weights are split into two 16-bit terms (f32 queries: three bf16 or two f16
// terms, queries too), so a 16-bit call rounds only its result and an f32 call
// keeps 2^-22 of each (over an f16 cache, where the last term's steps end, 2^-34 of
// the row's largest weight); the matrix cores have the time.
//
// The work is cut evenly over the workgroups whatever the lengths: the tiles of
// 32 keys of all sequences in one line a key-value head, a workgroup an equal
// stretch of a head's line, its waves the tiles in turn.  A sequence that
// crosses stretches is joined by the workgroup that finishes last, in the
// stretches' order, so the result does not depend on the schedule.
//
// Measured (32 query and 8 key-value heads of 128, pages of 16): 64 sequences of
// 1 to 8192 tokens in bf16 194 us, 5.5 TB/s of keys and values (a copy of 4 GiB
// moves 4.6); one of 32768 in f32 35 us, 3.9 TB/s; one of 200 tokens 8 us, four
// dependent reads of memory (length, table, keys, then the way out through
// LDS).  Many sequences of a few tiles are bound by that chain too, so runs of
// them go to a wave each (kAlone).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "bf16split.hpp"
#include "internal.hpp"
#include "kvcache.hpp"
#include "splitk.hpp"

namespace accel {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two f32 values as TERMS pairs of 16-bit values whose sum they are, up to the
// last term's rounding.
template <bool BF16, int TERMS>
__device__ __forceinline__ void terms16(float a, float b, uint32_t (&t)[TERMS]) {
    if constexpr (BF16) {
        split_terms<TERMS>(a, b, t);
    } else {
#pragma unroll
        for (int i = 0; i < TERMS; i++) {
            const f16x2 h = {(_Float16)a, (_Float16)b};
            t[i] = __builtin_bit_cast(uint32_t, h);
            a -= (float)h[0];
            b -= (float)h[1];
        }
    }
}

// Values that are not finite.  What the definition gives for one that is seen, as
// every weight is more than 0, is itself; a weight's terms of either sign, and
// weights that are 0 in 32 bits or fewer, make it NaN in a product.  So a pass over
// the keys whose result is not finite, or near that, is made again with such values
// apart: taken out of the products and added as they are.  Where all is finite that costs the
// look at the result and a barrier: 0.4 us of a window over 33 sequences' 14.4, 0.7 of
// a prompt; f32 prompts of 136 to 256 dims, whose registers spill, 4 to 5%.

// A factor of sums: with INF they may hold an infinity, which 0 would make NaN; the
// smallest number instead leaves what is finite as it was.
template <bool INF>
__device__ __forceinline__ float kept(float f) {
    return INF ? fmaxf(f, 0x1p-149f) : f;
}

// Whether a sum of weights or of values is, or of values so large (2^110) that sums
// of them may not be: products that leave the range then, by fours of an operand's
// rows that count.
template <int N, typename V, typename F>
__device__ __forceinline__ bool not_finite(float sum, const V (&o)[N], F counts) {
    float odd = sum * 0x1p18f;
#pragma unroll
    for (int e = 0; e < N; e++)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / 16); i++) {
            float x = o[e][4 * i] * 0x1p18f;
#pragma unroll
            for (int k = 1; k < 4; k++) x = __builtin_fmaf(o[e][4 * i + k], 0x1p18f, x);
            odd += counts(e, i) ? x : 0.0f;
        }
    return !(fabsf(odd) < INFINITY);
}

// A score in units of log 2 and its weight, each rounded by itself: the largest
// score's weight is what it is to be, however large they are.
__device__ __forceinline__ float scaled(float s, float factor) {
#pragma clang fp contract(off)
    return s * factor;
}
__device__ __forceinline__ float weight_of(float y, float m) {
#pragma clang fp contract(off)
    return __builtin_amdgcn_exp2f(y - m);
}

// Takes the values that are not finite out of eight.  One whose exponent is all
// ones carries into the sign's place.
template <bool BF16>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
    constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t kOne = BF16 ? 0x00800080u : 0x04000400u;
    return ((w & kExp) + kOne) & 0x80008000u;
}
template <bool BF16>
__device__ __forceinline__ u32x4 take_odd(u32x4& f) {
    u32x4 odd;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t mask = (odd_bits<BF16>(f[i]) >> 15) * 0xffffu;
        odd[i] = f[i] & mask;
        f[i] &= ~mask;
    }
    return odd;
}
template <bool BF16>
__device__ __forceinline__ u32x4 ones() {
    constexpr uint32_t k = BF16 ? 0x3f803f80u : 0x3c003c00u;
    return (u32x4){k, k, k, k};
}

// Keys that are not finite, under f32 queries: the first of the query's terms, the
// largest, gives the score there; those of either sign together give NaN.  It has
// the query's sign, however small the query: what would round to 0 is the term's
// smallest number instead (2^-38 of the row's largest magnitude).
template <bool BF16, bool CAREFUL>
__device__ __forceinline__ float signed_first(float v) {
    constexpr float kLeast = BF16 ? 0x1p-126f : 0x1p-24f;
    return CAREFUL && v != 0 && fabsf(v) < kLeast ? copysignf(kLeast, v) : v;
}

// f16 terms of f32 queries: the power of two that takes a row's largest magnitude
// to [2^14, 2^15), less where the scores' factor, which takes it back, would leave
// the normal range: scores hidden as -infinity are multiplied by it.
__device__ __forceinline__ int query_shift(float top, float factor) {
    const int ex = top > 0 && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
    const int most = 125 + __builtin_amdgcn_frexp_expf(factor);
    return ex < most ? ex : most;
}

__device__ __forceinline__ void store_result(const KvCache& c, const Attention& a, size_t i,
                                             float v) {
    if (a.q_f32) static_cast<float*>(a.out)[i] = v;
    else if (c.bf16) static_cast<__bf16*>(a.out)[i] = (__bf16)v;
    else static_cast<_Float16*>(a.out)[i] = (_Float16)v;
}

// ---- one new token a sequence ---------------------------------------------------

constexpr int kTile = 32;             // keys a wave step
// A weight is 2^(score - m), where m is the running maximum less kOver, and m moves
// when some score exceeds it by more than kOver + kLift.  f16 holds 2^-14 to 2^16 in
// full and steps of 2^-24 below: weights of 2^9 to 2^15 for the largest leave those
// down to 2^-23 of it all their bits, and half a step is 2^-34 of it.  (f16 prompt of
// 2048 with 7 + 8, 9 + 6 and 11 + 4: 60.0, 60.4 and 61.3 us, 59.0 with the largest at
// 1; f32 of 1000: 49.0, 49.8 and 51.1.)  A second pass over a bf16 cache takes 2^-40
// for the largest: 2^31 values of up to 2^128 stay in f32's range.
template <bool BF16, bool CAREFUL>
constexpr float kOver = !BF16 ? 9.0f : CAREFUL ? -40.0f : 0.0f;
template <bool BF16>
constexpr float kLift = BF16 ? 8.0f : 6.0f;
constexpr float kLowest = -__FLT_MAX__;   // m before any key
// A cut this near to a sequence's first or last tile moves there: a join costs
// about two steps of eight waves.  One sequence of 4096, eight heads of 128: 20.6
// us with 24, 15.5 with 12 or 8; 33 sequences seen through a window of 1000, 33
// tiles each: 13.7, 14.3 and 15.5.
constexpr uint32_t kNear = 12;

// Sequences of up to this many tiles are taken by a wave each where as many of
// them follow each other (256 of 50 to 150 tokens 59 -> 37 us; 200 of 1 to 300
// 56 -> 45 with up to 8 tiles, 40 with 12 or 16).
constexpr uint32_t kAlone = 12;
constexpr int kManyAlone = 3;

// m for a maximum.  Where f32's steps are 16, 9 less is 16 less.
template <bool BF16, bool CAREFUL>
__device__ __forceinline__ float below(float top) {
    constexpr float over = kOver<BF16, CAREFUL>;
    const float m = top - over;
    return top - m > over + kLift<BF16> ? top : m;
}

// The keys a query at position n - 1 sees: [0, first) and [lo, n); the tiles
// that hold them, in order.
struct Span {
    uint32_t n, lo, first, sink_tiles, start, tiles;
};
__device__ __forceinline__ Span span_of(const Attention& a, uint32_t n) {
    Span s;
    s.n = n;
    s.lo = a.window && n > a.window ? n - a.window : 0;
    s.first = a.sinks < s.lo ? a.sinks : s.lo;
    s.sink_tiles = (s.first + kTile - 1) / kTile;
    s.start = s.lo / kTile > s.sink_tiles ? s.lo / kTile : s.sink_tiles;
    const uint32_t end = (n + kTile - 1) / kTile;
    s.tiles = s.sink_tiles + (end > s.start ? end - s.start : 0);
    return s;
}

// Entry i's sequence and what its table holds of it (0: nothing to see).
struct Held {
    uint32_t seq, len;
};
__device__ __forceinline__ Held held_by(const KvCache& c, const Attention& a, int i,
                                        uint32_t* fault) {
    const uint32_t s = sequence_of(c, a.seqs, i, fault);
    return {s, s == kNoSequence ? 0 : length_of(c, s)};
}

// A prompt entry's rows of q: [first, first + count).
struct Rows {
    uint32_t first, count;
};
__device__ __forceinline__ Rows rows_of(const Attention& a, int i) {
    const uint32_t all = (uint32_t)a.rows;
    const uint32_t x = a.offsets[i], y = a.offsets[i + 1];
    const uint32_t lo = x < all ? x : all, hi = y < all ? y : all;
    return {lo, hi > lo ? hi - lo : 0};
}

// The entries' tiles summed up, for more entries than a wave has lanes:
// sums[i] = tiles of entries 0 .. i, of keys (tokens 0) or of so many of a
// prompt's tokens.  One workgroup.
__global__ __launch_bounds__(1024) void paged_sums_kernel(KvCache c, Attention a, uint32_t tokens,
                                                          uint32_t* sums, uint32_t* fault) {
    __shared__ uint32_t sh[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int base = 0; base < a.n; base += 1024) {
        const int i = base + threadIdx.x;
        uint32_t v = 0;
        if (i < a.n)
            v = tokens ? (rows_of(a, i).count + tokens - 1) / tokens
                       : span_of(a, held_by(c, a, i, fault).len).tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d, 64);
            if (lane >= d) v += up;
        }
        __syncthreads();
        if (lane == 63) sh[wave] = v;
        __syncthreads();
        uint32_t before = carry;
        for (int w = 0; w < 16; w++) {
            before += w < wave ? sh[w] : 0u;
            carry += sh[w];
        }
        if (i < a.n) sums[i] = before + v;
    }
}

// Where the line of tiles is cut.  Up to 64 entries: what is known of an entry
// is in the lane of its number, read once; more: in memory, the tiles summed up
// by the launch before.
struct Cut {
    uint32_t tiles;         // of all entries
    uint32_t chunk;         // tiles a workgroup
    uint32_t lane_sum;      // up to 64 entries: the running sum of this lane's
    Held lane_held;         // and its sequence
    const uint32_t* sums;   // more entries: the running sums
    int n;
};

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// The entry whose tiles hold x of the line (an entry in any case: sums over
// offsets that do not ascend may wrap); *start its first tile.
__device__ __forceinline__ int find_entry(const Cut& k, uint32_t x, uint32_t* start) {
    const int lane = threadIdx.x & 63;
    if (!k.sums) {
        int i = __popcll(__ballot(lane < k.n && k.lane_sum <= x));
        i = i < k.n ? i : k.n - 1;
        *start = i ? lane_value(k.lane_sum, i - 1) : 0;
        return i;
    }
    // 64 ways a step
    int lo = 0, size = k.n;
    while (size > 64) {
        const int step = (size + 63) / 64;
        const int at = lo + (lane + 1) * step - 1;
        const uint64_t below = __ballot(at < lo + size && at < k.n && k.sums[at] <= x);
        const int skip = __popcll(below) * step;
        lo += skip;
        size = size - skip < step ? size - skip : step;
    }
    const uint64_t below = __ballot(lane < size && k.sums[lo + lane] <= x);
    int i = __builtin_amdgcn_readfirstlane(lo + __popcll(below));
    i = i < k.n ? i : k.n - 1;
    *start = i ? __builtin_amdgcn_readfirstlane(k.sums[i - 1]) : 0;
    return i;
}

__device__ __forceinline__ Held entry_held(const Cut& k, const KvCache& c, const Attention& a,
                                           int i) {
    if (!k.sums) return {lane_value(k.lane_held.seq, i), lane_value(k.lane_held.len, i)};
    const Held h = held_by(c, a, i, nullptr);
    return {(uint32_t)__builtin_amdgcn_readfirstlane(h.seq),
            (uint32_t)__builtin_amdgcn_readfirstlane(h.len)};
}

// Where cut w of the line is made.
__device__ __forceinline__ uint32_t cut_at(const Cut& k, const KvCache& c, const Attention& a,
                                           uint64_t w) {
    if (w * k.chunk >= k.tiles) return k.tiles;
    const uint32_t x = (uint32_t)(w * k.chunk);
    uint32_t start;
    const int i = find_entry(k, x, &start);
    const uint32_t end = start + span_of(a, entry_held(k, c, a, i).len).tiles;
    return x - start <= kNear ? start : end - x <= kNear ? end : x;
}

// The join of a sequence's parts (of workgroups w0, w0 + 1 .. of the head) by the
// whole workgroup: sum and values scaled to the largest maximum and added in the
// parts' order.  A part is (maximum, sum) of each column, then the columns'
// values.  The maxima of all parts are read at once and the parts' factors kept
// in LDS (`room` floats), then a lane takes two dims of a column, BATCH parts'
// loads in flight.
template <int WAVES, int BATCH>
__device__ void join_parts(const KvCache& c, const Attention& a, float* parts, size_t slot_size,
                           uint32_t w0, uint32_t heads, uint32_t head, int count, int cols,
                           int dim, size_t qrow, float* sh, int room) {
    const auto slot = [&](int p) {
        return parts + (2 * ((w0 + p) * (size_t)heads + head) + (p == 0 ? 1 : 0)) * slot_size;
    };
    const auto load2 = [](float* p) {
        return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<uint64_t*>(p),
                                                           __ATOMIC_RELAXED,
                                                           __HIP_MEMORY_SCOPE_AGENT));
    };
    const int half = dim / 2;
    // as many columns a pass as the factors fit
    const int fit = room / (count + 1);
    for (int g0 = 0; g0 < cols; g0 += fit) {
        const int gs = cols - g0 < fit ? cols - g0 : fit;
        float* factor = sh;                // [gs][count]
        float* den = sh + gs * count;      // [gs]
        __syncthreads();
        for (int g = threadIdx.x >> 6; g < gs; g += WAVES) {
            // a wave a column
            const int lane = threadIdx.x & 63;
            float top = kLowest;
            for (int p = lane; p < count; p += 64)
                top = fmaxf(top, load2(slot(p) + 2 * (g0 + g))[0]);
            for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
            float sum = 0;
            for (int p0 = 0; p0 < count; p0 += 64) {
                const int p = p0 + lane;
                float term = 0;
                if (p < count) {
                    const f32x2 ml = load2(slot(p) + 2 * (g0 + g));
                    const float f = kept<true>(__builtin_amdgcn_exp2f(ml[0] - top));
                    factor[g * count + p] = f;
                    term = f * ml[1];
                }
                for (int x = 32; x; x >>= 1) term += __shfl_xor(term, x, 64);
                sum += term;
            }
            if (lane == 0) den[g] = sum;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < gs * half; i += 64 * WAVES) {
            const int g = i / half, d = (i - g * half) * 2;
            const uint32_t at = (uint32_t)(2 * cols + (g0 + g) * dim + d);
            f32x2 num = {0, 0};
            for (int p0 = 0; p0 < count; p0 += BATCH) {
                f32x2 v[BATCH];
#pragma unroll
                for (int x = 0; x < BATCH; x++)
                    v[x] = load2(slot(p0 + x < count ? p0 + x : p0) + at);
#pragma unroll
                for (int x = 0; x < BATCH; x++) {
                    const float f = p0 + x < count ? factor[g * count + p0 + x] : 0.0f;
                    num[0] += p0 + x < count ? f * v[x][0] : 0.0f;
                    num[1] += p0 + x < count ? f * v[x][1] : 0.0f;
                }
            }
            const float l = den[g];
            const size_t o = qrow + (size_t)(g0 + g) * dim + d;
            store_result(c, a, o, l == 0 ? 0.0f : num[0] / l);
            store_result(c, a, o + 1, l == 0 ? 0.0f : num[1] / l);
        }
    }
}

// Waves a workgroup, one workgroup a CU: eight, as the registers of up to 128
// dims allow; past that four.
template <int DIM>
constexpr int kWaves = DIM > 128 ? 4 : 8;

// MANY: a workgroup may have a run of short sequences.
template <bool BF16, int QT, int PT, int DIM, bool FULL, bool MANY>
__global__ __launch_bounds__(64 * kWaves<DIM>) void paged_decode_kernel(
    KvCache c, Attention a, const uint32_t* sums, uint32_t stretches, uint32_t* tickets,
    uint32_t ticket_stride, float* parts, uint32_t* fault) {
    constexpr int W = kWaves<DIM>;
    constexpr int NJ = DIM / 32;       // steps of 32 dims of a score
    constexpr int VD = DIM / 16;       // dims of a value a lane holds
    constexpr int VW = VD / 2;         // and words
    constexpr bool F32 = QT > 1;
    __shared__ float acc_sh[W][16][DIM + 4];
    __shared__ float max_sh[W][16], sum_sh[W][16];
    __shared__ int last_sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int dim = FULL ? DIM : c.dim;
    const int group = a.heads / c.heads;
    const int group_tiles = (group + 15) / 16;
    const uint32_t heads = (uint32_t)(c.heads * group_tiles);
    const uint32_t stretch = blockIdx.x / heads, head_tile = blockIdx.x - stretch * heads;
    const uint32_t head = head_tile / group_tiles;
    const int g0 = (int)(head_tile - head * group_tiles) * 16;
    const int cols = group - g0 < 16 ? group - g0 : 16;

    // the line of tiles
    Cut cut;
    cut.n = a.n;
    cut.sums = sums;
    if (!sums) {
        cut.lane_held = {kNoSequence, 0};
        if (lane < a.n) cut.lane_held = held_by(c, a, lane, blockIdx.x ? nullptr : fault);
        uint32_t v = span_of(a, cut.lane_held.len).tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d, 64);
            if (lane >= d) v += up;
        }
        cut.lane_sum = v;
        cut.tiles = lane_value(v, 63);
    } else {
        cut.tiles = __builtin_amdgcn_readfirstlane(sums[a.n - 1]);
    }
    // entries that see nothing
    for (int base = wave * 64; stretch + (uint64_t)stretches * base < (uint64_t)a.n;
         base += 64 * W) {
        const uint64_t i = stretch + (uint64_t)stretches * (base + lane);
        uint32_t len = 1;
        if (!sums) len = __shfl(cut.lane_held.len, (int)i & 63, 64);
        else if (i < (uint64_t)a.n) len = held_by(c, a, (int)i, nullptr).len;
        for (uint64_t none = __ballot(i < (uint64_t)a.n && len == 0); none; none &= none - 1) {
            const size_t row = stretch + (size_t)stretches * (base + __builtin_ctzll(none));
            for (int x = lane; x < cols * dim; x += 64)
                store_result(c, a, (row * a.heads + head * group + g0) * dim + x, 0.0f);
        }
    }
    // a tile a wave at least
    const uint32_t even = (uint32_t)(((uint64_t)cut.tiles + stretches - 1) / stretches);
    cut.chunk = even > W ? even : W;
    uint32_t u = cut_at(cut, c, a, stretch);
    const uint32_t u_end = cut_at(cut, c, a, stretch + 1);

    const size_t layer = (size_t)a.layer * c.pages * c.page_elems();
    while (u < u_end) {
        uint32_t item;
        int entry = find_entry(cut, u, &item);
        Held held = entry_held(cut, c, a, entry);
        Span sp = span_of(a, held.len);
        uint32_t t0 = u - item;
        uint32_t t1 = sp.tiles - t0 <= u_end - u ? sp.tiles : t0 + (u_end - u);
        uint32_t u_next = u + (t1 - t0);
        // Short sequences one after the other: a wave each, so that the waves'
        // chains of reads run side by side.  A lane an entry from this one on:
        // those up to the first that is too long, or not wholly in the stretch.
        uint64_t mine = 1;
        bool alone = false;
        Held lane_held = {kNoSequence, 0};
        if (MANY && t0 == 0 && t1 == sp.tiles && sp.tiles <= kAlone && u_next < u_end) {
            const int e = entry + lane;
            if (!sums)
                lane_held = {__shfl(cut.lane_held.seq, e & 63, 64),
                             __shfl(cut.lane_held.len, e & 63, 64)};
            else if (e < a.n)
                lane_held = held_by(c, a, e, nullptr);
            const uint32_t own = e < a.n ? span_of(a, lane_held.len).tiles : 0;
            uint32_t past = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(past, d, 64);
                if (lane >= d) past += up;
            }
            const uint64_t stop = __ballot(e >= a.n || own > kAlone || past > u_end - u);
            const int run = stop ? __builtin_ctzll(stop) : 64;
            const uint64_t items = __ballot(lane < run && own != 0);
            alone = __popcll(items) >= kManyAlone;
            if (alone) {
                const int rank = __popcll(items & ((1ull << lane) - 1));
                mine = __ballot((items >> lane & 1) && rank % W == wave);
                u_next = u + lane_value(past, run - 1);
            }
        }
        const int entry0 = entry;
        for (; mine; mine &= mine - 1) {
            uint32_t t_first = t0 + wave, stride = W;
            if (alone) {
                const int l = __builtin_ctzll(mine);
                entry = entry0 + l;
                held = {lane_value(lane_held.seq, l), lane_value(lane_held.len, l)};
                sp = span_of(a, held.len);
                t0 = 0, t1 = sp.tiles, t_first = 0, stride = 1;
            }
            const uint32_t seq = held.seq;
            const size_t qrow = ((size_t)entry * a.heads + head * group + g0) * dim;

            // A first pass takes the values as they are; where something in it is
            // not finite the wave goes over its keys again, carefully.
            f32x4 o[VD];
            float m, sum;
            const auto pass = [&](auto careful) {
                constexpr bool CAREFUL = decltype(careful)::value;
                // queries: the B operand, column = query head
                u32x4 q[QT][NJ];
                float factor = a.scale * 1.44269504088896340736f;
                if constexpr (F32) {
                    const float* src = static_cast<const float*>(a.q) + qrow + (size_t)col * dim;
                    float v[NJ][8];
                    float top = 0;
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        const int d = j * 32 + quad * 8;
                        const bool in = col < cols && d < dim;
                        f32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
                        if (in) {
                            lo = *reinterpret_cast<const f32x4*>(src + d);
                            hi = *reinterpret_cast<const f32x4*>(src + d + 4);
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            v[j][e] = e < 4 ? lo[e] : hi[e - 4];
                            top = fmaxf(top, fabsf(v[j][e]));
                        }
                    }
                    if constexpr (!BF16) {
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const int ex = query_shift(top, factor);
                        factor = ldexpf(factor, -ex);
#pragma unroll
                        for (int j = 0; j < NJ; j++)
#pragma unroll
                            for (int e = 0; e < 8; e++) v[j][e] = ldexpf(v[j][e], ex);
                    }
#pragma unroll
                    for (int j = 0; j < NJ; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t t[QT];
                            terms16<BF16, QT>(signed_first<BF16, CAREFUL>(v[j][2 * e]),
                                              signed_first<BF16, CAREFUL>(v[j][2 * e + 1]), t);
#pragma unroll
                            for (int k = 0; k < QT; k++) q[k][j][e] = t[k];
                        }
                } else {
                    const uint16_t* src = static_cast<const uint16_t*>(a.q) + qrow + (size_t)col * dim;
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        const int d = j * 32 + quad * 8;
                        q[0][j] = col < cols && d < dim ? *reinterpret_cast<const u32x4*>(src + d)
                                                        : (u32x4){0, 0, 0, 0};
                    }
                }

#pragma unroll
                for (int e = 0; e < VD; e++) o[e] = (f32x4){0, 0, 0, 0};
                m = kLowest, sum = 0;

                const uint32_t* table = c.tables + (size_t)seq * c.slots;
                const uint32_t row_mask = (1u << c.shift) - 1;
                const uint32_t kv_row = head << c.shift;      // rows before this head's in a page
                const int k_block = col >> 2;
                // first position of tile t
                const auto tile_pos = [&](uint32_t t) {
                    return (t < sp.sink_tiles ? t : sp.start + (t - sp.sink_tiles)) * kTile;
                };
                // the page of eight positions from pos (a multiple of 8) on, where a
                // key among them is seen; ~0 where it names none
                const auto seen8 = [&](uint32_t pos) {
                    return pos < sp.n && (pos + 8 > sp.lo || pos < sp.first);
                };
                const auto page_of = [&](uint32_t pos) {
                    uint32_t p = 0;
                    if (seen8(pos)) p = table[pos >> c.shift];
                    return p;
                };
                const auto k_rows = [&](uint32_t page, uint32_t pos) {
                    const uint32_t p = page < c.pages ? page : 0;
                    return c.keys + layer +
                           ((size_t)p * ((size_t)c.heads << c.shift) + kv_row +
                            ((pos + k_block * 8 + (col & 3)) & row_mask)) * dim + quad * 8;
                };
                const auto v_rows = [&](uint32_t page, uint32_t pos) {
                    const uint32_t p = page < c.pages ? page : 0;
                    const int d = FULL || col * VD < dim ? col * VD : 0;
                    return c.values + layer +
                           ((size_t)p * ((size_t)c.heads << c.shift) + kv_row +
                            ((pos + quad * 8) & row_mask)) * dim + d;
                };
                u32x4 k[2][NJ];
                uint32_t v[8][VW];
                const auto load_k = [&](uint32_t page, uint32_t pos) {
                    const uint16_t* p = k_rows(page, pos);
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int j = 0; j < NJ; j++) {
                            if (FULL || j * 32 + quad * 8 < dim)
                                k[t][j] = *reinterpret_cast<const u32x4*>(p + t * 4 * dim + j * 32);
                            else
                                k[t][j] = (u32x4){0, 0, 0, 0};
                        }
                };
                const auto load_v = [&](uint32_t page, uint32_t pos) {
                    const uint16_t* p = v_rows(page, pos);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if constexpr (VW == 2) {
                            const u32x2 w = *reinterpret_cast<const u32x2*>(p + i * dim);
                            v[i][0] = w[0], v[i][1] = w[1];
                        } else {
#pragma unroll
                            for (int h = 0; h < VW / 4; h++) {
                                // a head may end inside a lane's sixteen dims
                                const int d = FULL || h == 0 || col * VD + h * 8 < dim ? h * 8 : 0;
                                const u32x4 w = *reinterpret_cast<const u32x4*>(p + i * dim + d);
#pragma unroll
                                for (int e = 0; e < 4; e++) v[i][4 * h + e] = w[e];
                            }
                        }
                    }
                };

                uint32_t t = t_first;
                uint32_t pos = 0, k_page = 0, v_page = 0, k_next = 0, v_next = 0;
                if (t < t1) {
                    pos = tile_pos(t);
                    k_page = page_of(pos + k_block * 8);
                    v_page = page_of(pos + quad * 8);
                    if (t + stride < t1) {
                        k_next = page_of(tile_pos(t + stride) + k_block * 8);
                        v_next = page_of(tile_pos(t + stride) + quad * 8);
                    }
                    load_k(k_page, pos);
                    load_v(v_page, pos);
                }
                for (; t < t1; t += stride) {
                    const bool more = t + stride < t1;
                    const uint32_t pos_next = more ? tile_pos(t + stride) : 0;
                    // scores
                    f32x4 s[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        s[i] = (f32x4){0, 0, 0, 0};
                        f32x4 low = {0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < NJ; j++)
#pragma unroll
                            for (int x = QT - 1; x >= 0; x--) {
                                f32x4& to = CAREFUL && x ? low : s[i];
                                to = mfma16<BF16>(k[i][j], q[x][j], to);
                            }
                        if constexpr (CAREFUL)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                s[i][e] += fabsf(s[i][e]) < INFINITY ? low[e] : 0.0f;
                    }
                    const uint32_t page_now = v_page;
                    if (more) load_k(k_next, pos_next);
                    // which of them are seen
                    const bool all = pos + kTile <= sp.n && (pos >= sp.lo || pos + kTile <= sp.first) &&
                                     !__any(page_now >= c.pages);
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = scaled(s[e >> 2][e & 3], factor);
                    uint32_t hidden = 0;
                    if (!all) {
                        const uint32_t p0 = pos + quad * 8;
                        if (page_now >= c.pages) report(fault, kFaultKvPage);
                        // conditions without branches, a select each: joined with &&
                        // and || an earlier form did not hide y[0] of a key behind the
                        // window (why was not found; the window tests hold this one)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const bool ok = (p0 + e < sp.n) &
                                            ((p0 + e >= sp.lo) | (p0 + e < sp.first)) &
                                            (page_now < c.pages);
                            hidden |= ok ? 0u : 1u << e;
                            y[e] = ok ? y[e] : -INFINITY;
                        }
                    }
                    float top = y[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) top = fmaxf(top, y[e]);
                    if (__any(top - m > kOver<BF16, CAREFUL> + kLift<BF16>)) {
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const float up = fmaxf(m, below<BF16, CAREFUL>(top));
                        const float keep = kept<CAREFUL>(__builtin_amdgcn_exp2f(m - up));
                        m = up;
                        sum *= keep;
#pragma unroll
                        for (int e = 0; e < VD; e++) o[e] *= keep;
                    }
                    u32x4 w[PT];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float a0 = weight_of(y[2 * e], m);
                        const float a1 = weight_of(y[2 * e + 1], m);
                        sum += a0 + a1;
                        uint32_t x[PT];
                        terms16<BF16, PT>(a0, a1, x);
#pragma unroll
                        for (int i = 0; i < PT; i++) w[i][e] = x[i];
                    }
                    // values of keys that are not seen count as 0, whatever they hold
                    if (!all) {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (hidden >> i & 1) {
#pragma unroll
                                for (int e = 0; e < VW; e++) v[i][e] = 0;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < VD; e++) {
                        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                        u32x4 f;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            f[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], sel);
                        if constexpr (CAREFUL) {
                            const u32x4 odd = take_odd<BF16>(f);
                            o[e] = mfma16<BF16>(odd, ones<BF16>(), o[e]);
                        }
#pragma unroll
                        for (int i = PT - 1; i >= 0; i--) o[e] = mfma16<BF16>(f, w[i], o[e]);
                    }
                    if (more) {
                        load_v(v_next, pos_next);
                        v_page = v_next;
                        pos = pos_next;
                        if (t + 2 * stride < t1) {
                            const uint32_t after = tile_pos(t + 2 * stride);
                            k_next = page_of(after + k_block * 8);
                            v_next = page_of(after + quad * 8);
                        }
                    }
                }
            };
            pass(std::false_type());
            if (__any(not_finite(sum, o, [](int, int) { return true; }))) pass(std::true_type());
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (alone) {
                const float out = sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < VD; e++) {
                        const int d = (quad * 4 + i) * VD + e;
                        if (col < cols && (FULL || d < dim))
                            store_result(c, a, qrow + (size_t)col * dim + d,
                                         sum == 0 ? 0.0f : o[e][i] * out);
                    }
                continue;
            }

            // the waves' parts of this pair
            __syncthreads();
            if (col < cols) {
                if (quad == 0) max_sh[wave][col] = m, sum_sh[wave][col] = sum;
#pragma unroll
                for (int e = 0; e < VD; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        acc_sh[wave][col][(quad * 4 + i) * VD + e] = o[e][i];
            }
            __syncthreads();
            const bool whole = t0 == 0 && t1 == sp.tiles;
            const uint32_t per = (uint32_t)(cols * dim);
            const size_t slot_size = (size_t)(group < 16 ? group : 16) * (dim + 2);
            float* part = parts + (2 * (size_t)blockIdx.x + (t0 == 0 ? 1 : 0)) * slot_size;
            for (uint32_t i = threadIdx.x; i < per; i += 64 * W) {
                const int g = (int)(i / dim), d = (int)(i - g * dim);
                float top = max_sh[0][g];
#pragma unroll
                for (int x = 1; x < W; x++) top = fmaxf(top, max_sh[x][g]);
                float den = 0, num = 0;
#pragma unroll
                for (int x = 0; x < W; x++) {
                    const float f = kept<true>(__builtin_amdgcn_exp2f(max_sh[x][g] - top));
                    den += f * sum_sh[x][g];
                    num += f * acc_sh[x][g][d];
                }
                if (whole) {
                    store_result(c, a, qrow + (size_t)g * dim + d, den == 0 ? 0.0f : num / den);
                } else {
                    store_device(part + 2 * cols + i, num);
                    if (d == 0) {
                        store_device(part + 2 * g, top);
                        store_device(part + 2 * g + 1, den);
                    }
                }
            }
            if (!whole) {
                // the stretches that hold a part: w0, whose end is the first cut
                // farther than kNear from the sequence's ends, to w1, whose start
                // is the last; the one to arrive last joins them all
                const uint64_t end = (uint64_t)item + sp.tiles;
                const uint32_t w0 = (uint32_t)(((uint64_t)item + kNear) / cut.chunk);
                const uint32_t w1 = (uint32_t)((end - kNear + cut.chunk - 1) / cut.chunk) - 1;
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __builtin_amdgcn_s_waitcnt(0);
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __syncthreads();
                uint32_t* ticket = tickets + ((size_t)w0 * heads + head_tile) * ticket_stride;
                if (threadIdx.x == 0)
                    last_sh = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT) == w1 - w0;
                __syncthreads();
                if (last_sh) {
                    join_parts<W, 16>(c, a, parts, slot_size, w0, heads, head_tile,
                                      (int)(w1 - w0) + 1, cols, dim, qrow, &acc_sh[0][0][0],
                                      W * 16 * (DIM + 4));
                    if (threadIdx.x == 0)
                        __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
        u = u_next;
    }
}

// ---- prompts ------------------------------------------------------------------------
//
// A workgroup takes 128 rows, 32 a wave: (token, query head of one group) pairs,
// as many whole tokens as fit, so a tile of keys and values serves the group's
// heads at once.  Tiles of KT keys go through LDS as they lie, loaded straight
// there a tile ahead; V is read turned (ds_read_b64_tr_b16).  A wave computes
// S^T = K Q^T and O^T += V^T P^T with 32 x 32 x 16 MFMAs; a lane has one row's
// scores and sums (its column), half of the keys, and the other half is 32
// lanes on.  As in the decode kernel the keys' order in K's rows is chosen so that
// a lane's scores are its part of P^T's operand, and the running maximum moves
// as rarely.
//
// Weights of a 16-bit call are rounded to its type once (the sum of them is not):
// half a step of each, in f16 no less than 2^-34 of the row's largest, as the
// product's operands have to be 16 bits; f32 calls split queries and weights as the
// decode kernel does.
//
// What bounds it is issue: with two waves a SIMD the MFMAs take 38% of a step's
// cycles and some 280 VALU instructions a wave most of the rest; 2048 tokens
// (32/8 heads of 128, bf16) run in 57 us, 600 TFLOP/s of what is seen, 8192
// through a window of 1024 in 186 us, 695 (an 8192 cube in bf16 reaches 1200).
// Tried and left: eight waves a workgroup (taller tiles hide more of what they
// compute, one barrier holds all: 208 us against 196), wave priorities around the
// products (58 against 56), weights first and the maximum after (S outlives
// them: spills, 98 against 64).

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr int kRows = 128;            // rows a workgroup

// s_waitcnt vmcnt(0), as an instruction that the compiler counts itself; reads of
// what the loads brought to LDS stay behind it.
__device__ __forceinline__ void wait_loads() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Four keys of one dim: see the kernel's v_from.
__device__ __forceinline__ u32x2 read_turned(const char* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4*)p));
}

// Tiles of keys that are worth a workgroup and its part of a join (5 tokens after
// 8192, 16-bit: 48 us with two, 31 with four, 29 with eight; 42 tokens a tile of
// 8 tiles: 25.4 with four, 26.4 with eight).
template <bool F32>
constexpr int kTilesAShare = F32 ? 2 : 4;

// Tokens of a tile of rows, and the query heads of one.
__host__ __device__ inline int prompt_heads(int group) { return group < kRows ? group : kRows; }
__host__ __device__ inline int prompt_tokens(int group) { return kRows / prompt_heads(group); }

template <bool BF16, int QT, int PT, int DIM, bool FULL, int KT>
__global__ __launch_bounds__(256, QT == 1 && DIM <= 128 ? 2 : 1) void paged_prefill_kernel(
    KvCache c, Attention a, const uint32_t* sums, uint32_t fold, uint32_t splits, uint32_t place0,
    uint32_t* tickets, uint32_t ticket_stride, float* parts, uint32_t* fault) {
    constexpr int NS = DIM / 16;            // MFMA steps of a score
    constexpr int NC = DIM / 8;             // 16-byte chunks of a key
    constexpr int SUB = KT / 32;            // 32-key parts of a tile
    constexpr int DT = DIM / 32;            // 32-dim parts of a row of values
    constexpr int BLOCKS = KT / 8;          // eight keys lie in one page
    constexpr int KL = KT * NC / 256;       // chunks of K, and of V, a lane stages
    constexpr bool F32 = QT > 1;
    __shared__ __attribute__((aligned(256))) char k_sh[2][KT * NC * 16];
    __shared__ __attribute__((aligned(256))) char v_sh[2][KT * NC * 16];
    // keys of a tile with values that are not finite: tile t's in place t % 3,
    // which is cleared two steps before it is read, a barrier before it is set
    __shared__ uint32_t odd_sh[3][2];
    __shared__ uint32_t again_sh;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int dim = FULL ? DIM : c.dim;
    const int group = a.heads / c.heads;
    const int per = prompt_heads(group), tokens = prompt_tokens(group);
    const int group_tiles = (group + per - 1) / per;
    const uint32_t heads = (uint32_t)(c.heads * group_tiles);
    // shares are the slow index: those that have nothing to do come last
    const uint32_t places = gridDim.x / splits;
    const uint32_t split = blockIdx.x / places, place = place0 + blockIdx.x - split * places;
    const uint32_t order = place / heads, head_tile = place - order * heads;
    const uint32_t head = head_tile / group_tiles;
    const int g0 = (int)(head_tile - head * group_tiles) * per;
    const int gs = group - g0 < per ? group - g0 : per;

    // this workgroup's tile of rows: the longest (last) ones first; where all
    // tiles run at once, two a CU, the second half of them shortest first, so
    // that a long one shares its CU with a short one (two prompts of 1024, 64
    // dims: 32 -> 28 us)
    Cut cut;
    cut.n = a.n;
    cut.sums = sums;
    if (!sums) {
        // lengths are asked for beside the offsets, not after them
        cut.lane_held = {kNoSequence, 0};
        if (lane < a.n) cut.lane_held = held_by(c, a, lane, blockIdx.x ? nullptr : fault);
        uint32_t v = lane < a.n ? (rows_of(a, lane).count + tokens - 1) / tokens : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d, 64);
            if (lane >= d) v += up;
        }
        cut.lane_sum = v;
        cut.tiles = lane_value(v, 63);
    } else {
        cut.tiles = __builtin_amdgcn_readfirstlane(sums[a.n - 1]);
    }
    if (order >= cut.tiles) return;
    const uint32_t tile = cut.tiles <= 2 * fold && order >= fold ? order - fold
                                                                 : cut.tiles - 1 - order;
    uint32_t item;
    const int entry = find_entry(cut, tile, &item);
    const Rows rows = rows_of(a, entry);
    const uint32_t tok0 = (tile - item) * tokens;
    if (tok0 >= rows.count) return;      // offsets that do not ascend
    const uint32_t toks = rows.count - tok0 < (uint32_t)tokens ? rows.count - tok0 : tokens;
    const Held held = sums ? held_by(c, a, entry, threadIdx.x ? nullptr : fault)
                           : entry_held(cut, c, a, entry);
    // the position of the tile's first token; below 0 it sees nothing
    const int base = (int)held.len - (int)rows.count + (int)tok0;
    const int window = a.window ? (int)a.window : 0x7fffffff;
    const int sinks = a.window ? (int)a.sinks : 0;

    // this lane's row
    const int r = wave * 32 + col;
    const int tok = r / per, g = r - tok * per;
    const bool real = tok < (int)toks && g < gs;
    const int p = real && base + tok > -1 ? base + tok : -1;
    const size_t qrow = ((size_t)(rows.first + tok0 + (real ? tok : 0)) * a.heads + head * group +
                         g0 + (real ? g : 0)) * dim;
    // the wave's first and last position, and the workgroup's
    const int tok_a = wave * 32 / per, tok_b = (wave * 32 + 31) / per;
    const bool busy = tok_a < (int)toks;
    const int p_a = base + tok_a > -1 ? base + tok_a : -1;
    const int p_last = base + (tok_b < (int)toks ? tok_b : (int)toks - 1);
    const int p_b = p_last > -1 ? p_last : -1;
    const int p_end = base + (int)toks;           // past the workgroup's last

    // tiles of keys: those of the sinks, then those from the first window's
    // start to the last position
    const int lo = base + 1 > window ? base + 1 - window : 0;
    const int near = sinks < lo ? sinks : lo;
    const int sink_tiles = (near + KT - 1) / KT;
    const int start = lo / KT > sink_tiles ? lo / KT : sink_tiles;
    const int last = p_end > 0 ? (p_end - 1) / KT + 1 : 0;
    const int count = p_end > 0 ? sink_tiles + (last > start ? last - start : 0) : 0;
    // this workgroup's share of them: where the rows are few, a tile of rows has
    // several workgroups, each with at least kShare tiles of keys
    constexpr int kShare = kTilesAShare<F32>;
    const int shares = count / kShare < (int)splits ? (count / kShare > 0 ? count / kShare : 1)
                                                    : (int)splits;
    const int share = (count + shares - 1) / shares;
    const int held_shares = count > 0 ? (count + share - 1) / share : 1;
    if ((int)split >= held_shares) return;
    const int t_begin = (int)split * share;
    const int t_end = t_begin + share < count ? t_begin + share : count;
    const auto tile_pos = [&](int t) {
        return (t < sink_tiles ? t : start + (t - sink_tiles)) * KT;
    };
    const uint32_t* table = c.tables + (size_t)held.seq * c.slots;
    const uint64_t page_bytes = c.page_elems() * 2;
    const uint32_t row_mask = (1u << c.shift) - 1;
    const uint32_t head_row = head << c.shift;    // below 2^24
    const size_t layer = (size_t)a.layer * c.pages * c.page_elems();
    const char* keys = reinterpret_cast<const char*>(c.keys + layer);
    const char* values = reinterpret_cast<const char*>(c.values + layer);
    // the page of the eight positions from pos on, for a lane a block; one that
    // some row of the workgroup sees has to name a page
    const auto page_of = [&](int pos) {
        uint32_t page = 0;
        const int x = pos + (lane & (BLOCKS - 1)) * 8;
        if (x < p_end && (x + 8 > lo || x < near)) page = table[(uint32_t)x >> c.shift];
        return page;
    };
    // Where chunks lie: linear in the bits of their numbers under exclusive or,
    // so a lane's address is its own part, exchanged with a constant's.  K's
    // sixteen rows a read takes at once, and V's four times 64 bytes, fall in
    // different banks.
    const auto k_swap = [](int key) { return NC >= 16 ? key & 15 : key >> 1 & 7; };
    const auto v_swap = [](int key) { return NC >= 16 ? (key & 3) << 2 : (key >> 1 & 1) << 2; };
    const auto k_byte = [&](int key, int ch) { return (key * NC + (ch ^ k_swap(key))) * 16; };
    const auto v_byte = [&](int key, int ch) { return (key * NC + (ch ^ v_swap(key))) * 16; };
    // what a lane stages, straight to LDS: a wave 64 consecutive chunks a step
    // (what the lane reads follows from where it lands); bytes from the row of
    // the block's first key, or none past the head's dims
    constexpr uint32_t kNoChunk = 0xffffffffu;
    uint32_t k_off[KL], v_off[KL];
#pragma unroll
    for (int i = 0; i < KL; i++) {
        const int at = (wave * KL + i) * 64 + lane, key = at / NC;
        const int kc = at % NC ^ k_swap(key), vc = at % NC ^ v_swap(key);
        k_off[i] = FULL || kc * 8 < dim ? (uint32_t)((key & 7) * dim + kc * 8) * 2 : kNoChunk;
        v_off[i] = FULL || vc * 8 < dim ? (uint32_t)((key & 7) * dim + vc * 8) * 2 : kNoChunk;
    }
    // the lanes of blocks 0 .. hold the byte offset of their block's first row
    // in a plane, from which a load's uniform part is read
    const uint32_t row_bytes = (uint32_t)dim * 2;
    const auto block_rows = [&](uint32_t pages, int pos) {
        const uint32_t at = (uint32_t)head_row +
                            (((uint32_t)pos + (lane & (BLOCKS - 1)) * 8) & row_mask);
        return (pages < c.pages ? pages : 0) * page_bytes + (uint64_t)at * row_bytes;
    };
    const auto block_row = [&](uint64_t rows, int b) {
        return (uint64_t)lane_value((uint32_t)rows, b) |
               (uint64_t)lane_value((uint32_t)(rows >> 32), b) << 32;
    };
    const auto to_lds = [](const char* from, char* to) {
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)from,
            (__attribute__((address_space(3))) void*)to, 16, 0, 0);
    };
    const auto load = [&](uint32_t pages, int pos, auto buf) {
        constexpr int B = decltype(buf)::value;
        const uint64_t rows = block_rows(pages, pos);
#pragma unroll
        for (int i = 0; i < KL; i++) {
            // a step's keys lie in one block of eight
            const int at = (wave * KL + i) * 64;
            const uint64_t row = block_row(rows, at / NC / 8);
            if (FULL || k_off[i] != kNoChunk) to_lds(keys + row + k_off[i], k_sh[B] + at * 16);
            if (FULL || v_off[i] != kNoChunk) to_lds(values + row + v_off[i], v_sh[B] + at * 16);
        }
    };
    // whether every row of the workgroup sees all of the tile
    const auto plain = [&](int pos) {
        return pos + KT <= base + 1 && (pos > p_end - 1 - window || pos + KT <= sinks);
    };
    const auto arrive = [&](uint32_t pages, int pos, int odd, auto buf, auto careful) {
        constexpr int B = decltype(buf)::value;
        constexpr bool CAREFUL = decltype(careful)::value;
        // what this wave staged is in LDS before the barrier that follows
        wait_loads();
        if (!CAREFUL && plain(pos) && !__any(pages >= c.pages)) return;
        // values no row sees count as 0, whatever they hold; those that are not
        // finite are left out of the product, where a row that does not see them
        // would meet them, and added apart
#pragma unroll
        for (int i = 0; i < KL; i++) {
            const int at = (wave * KL + i) * 64 + lane, key = at / NC;
            const int x = pos + key;
            const uint32_t page = __shfl(pages, key >> 3, 64);
            const bool seen = (x < p_end) & ((x >= lo) | (x < near)) & (page < c.pages);
            u32x4* chunk = reinterpret_cast<u32x4*>(v_sh[B] + at * 16);
            if (!FULL && v_off[i] == kNoChunk) continue;
            u32x4 w = {0, 0, 0, 0};
            if (seen) {
                w = *chunk;
                u32x4 over;
#pragma unroll
                for (int e = 0; e < 4; e++) over[e] = odd_bits<BF16>(w[e]);
                if ((over[0] | over[1] | over[2] | over[3]) == 0) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] &= ~((over[e] >> 15) * 0xffffu);
                atomicOr(&odd_sh[odd][key >> 5], 1u << (key & 31));
            }
            *chunk = w;
        }
    };

    // dims past the head's: K's chunks there are no load's target and stay 0
    if constexpr (!FULL) {
        for (int i = threadIdx.x; i < 2 * KT * NC; i += 256)
            reinterpret_cast<u32x4*>(k_sh)[i] = (u32x4){0, 0, 0, 0};
    }
    // A first pass takes the values of tiles that all rows see as they are; where
    // something in it is not finite, or scores are large, the workgroup goes over
    // its keys again.
    f32x16 o[DT];
    float m, sum;
    bool unnamed = false;       // a page some row sees and the table does not name
    const auto pass = [&](auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        // queries: the B operand, column = row
        u32x4 q[QT][NS];
        float factor = a.scale * 1.44269504088896340736f;
        if constexpr (F32) {
            const float* src = static_cast<const float*>(a.q) + qrow;
            float top = 0;
            if constexpr (!BF16) {
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    const int d = j * 16 + half * 8;
                    if (real && d < dim)
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(src[d + e]));
                }
                top = fmaxf(top, __shfl_xor(top, 32, 64));
            }
            const int ex = BF16 ? 0 : query_shift(top, factor);
            if constexpr (!BF16) factor = ldexpf(factor, -ex);
#pragma unroll
            for (int j = 0; j < NS; j++) {
                const int d = j * 16 + half * 8;
                f32x4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                if (real && d < dim) {
                    x[0] = *reinterpret_cast<const f32x4*>(src + d);
                    x[1] = *reinterpret_cast<const f32x4*>(src + d + 4);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float y0 = x[e >> 1][2 * (e & 1)], y1 = x[e >> 1][2 * (e & 1) + 1];
                    if constexpr (!BF16) y0 = ldexpf(y0, ex), y1 = ldexpf(y1, ex);
                    uint32_t t[QT];
                    terms16<BF16, QT>(signed_first<BF16, CAREFUL>(y0),
                                      signed_first<BF16, CAREFUL>(y1), t);
#pragma unroll
                    for (int k = 0; k < QT; k++) q[k][j][e] = t[k];
                }
            }
        } else {
            const uint16_t* src = static_cast<const uint16_t*>(a.q) + qrow;
#pragma unroll
            for (int j = 0; j < NS; j++) {
                const int d = j * 16 + half * 8;
                q[0][j] = real && d < dim ? *reinterpret_cast<const u32x4*>(src + d)
                                          : (u32x4){0, 0, 0, 0};
            }
        }

#pragma unroll
        for (int e = 0; e < DT; e++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[e][i] = 0;
        m = kLowest, sum = 0;
        uint32_t pages = 0, pages_next = 0;
        if (threadIdx.x < 6) odd_sh[threadIdx.x >> 1][threadIdx.x & 1] = 0;
        __syncthreads();
        if (t_begin < t_end) {
            pages = page_of(tile_pos(t_begin));
            if (t_begin + 1 < t_end) pages_next = page_of(tile_pos(t_begin + 1));
            load(pages, tile_pos(t_begin), std::integral_constant<int, 0>());
            arrive(pages, tile_pos(t_begin), 0, std::integral_constant<int, 0>(), careful);
        }
        // the lane's part of what it reads: row 8 x + 4 h + b of K's operand holds
        // key 16 (x / 2) + 8 h + 4 (x % 2) + b
        const int k_from = k_byte(16 * (col >> 4) + 8 * (col >> 2 & 1) + 4 * (col >> 3 & 1) + (col & 3),
                                  half);
        // values through the transposing read: of sixteen lanes four take 32 bytes
        // of one key's dims, and each receives one dim of the four keys
        const int v_from = v_byte(half * 8 + (col >> 2 & 3), (col >> 4) * 2 + (col >> 1 & 1)) +
                           (col & 1) * 8;
        // the queries have arrived: without this the loop's first product waits for
        // every load in flight, each time
        wait_loads();
        int odd_at = 0;
        const auto step = [&](int t, auto buf) {
            constexpr int B = decltype(buf)::value;
            const std::integral_constant<int, B ^ 1> other;
            const int pos = tile_pos(t);
            const bool more = t + 1 < t_end;
            unnamed |= pages >= c.pages;
            __syncthreads();
            const uint32_t odd0 = odd_sh[odd_at][0], odd1 = odd_sh[odd_at][1];
            const int odd_next = odd_at == 2 ? 0 : odd_at + 1;
            if (threadIdx.x < 2) odd_sh[odd_next == 2 ? 0 : odd_next + 1][threadIdx.x] = 0;
            odd_at = odd_next;
            if (more) load(pages_next, tile_pos(t + 1), other);
            // a whole step ahead of its use
            const uint32_t pages_after = t + 2 < t_end ? page_of(tile_pos(t + 2)) : 0;
            // a wave none of whose rows sees the tile only stages
            if (busy && pos <= p_b && (pos + KT > p_a + 1 - window || pos < sinks)) {
                f32x16 s[SUB];
#pragma unroll
                for (int i = 0; i < SUB; i++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[i][e] = 0;
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    u32x4 kf[SUB];
#pragma unroll
                    for (int i = 0; i < SUB; i++)
                        kf[i] = *reinterpret_cast<const u32x4*>(
                            k_sh[B] + (k_from ^ k_byte(0, 2 * j)) + k_byte(i * 32, 0));
#pragma unroll
                    for (int x = QT - 1; x >= 0; x--)
#pragma unroll
                        for (int i = 0; i < SUB; i++) s[i] = mfma32<BF16>(kf[i], q[x][j], s[i]);
                }
                if constexpr (CAREFUL && F32) {
                    // first terms alone where the score is not finite
#pragma unroll
                    for (int i = 0; i < SUB; i++) {
                        f32x16 first;
#pragma unroll
                        for (int e = 0; e < 16; e++) first[e] = 0;
#pragma unroll
                        for (int j = 0; j < NS; j++)
                            first = mfma32<BF16>(
                                *reinterpret_cast<const u32x4*>(
                                    k_sh[B] + (k_from ^ k_byte(0, 2 * j)) + k_byte(i * 32, 0)),
                                q[0][j], first);
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            s[i][e] = fabsf(first[e]) < INFINITY ? s[i][e] : first[e];
                    }
                }
                // reads three products ahead of their use
                if constexpr (QT == 1) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 3 * SUB, 0);
#pragma unroll
                    for (int j = 0; j < NS - 3; j++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, SUB, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, SUB, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, 3 * SUB, 0);
                }
                // keys a row does not see, by a key's place x in the tile: past the
                // row's position, behind its window, on a page without a number
                const int here = pos + half * 8;
                const int until = p - here;
                const auto hide = [&](auto seen) {
#pragma unroll
                    for (int i = 0; i < SUB; i++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            s[i][e] = seen(i * 32 + (e >> 3) * 16 + (e & 7)) ? s[i][e] : -INFINITY;
                };
                if (pos + KT > p_a + 1) hide([&](int x) { return x <= until; });
                if (!(pos > p_b - window || pos + KT <= sinks)) {
                    // the first place the row's window holds; none where it is all past
                    const int from = until < window ? -KT : until - window + 1;
                    if (pos >= sinks) {
                        hide([&](int x) { return x >= from; });
                    } else {
                        const int kept = sinks - here;
                        hide([&](int x) { return (x >= from) | (x < kept); });
                    }
                }
                const uint64_t named = __ballot(pages < c.pages);   // bit b: block b's page
                if (~named & ((1ull << BLOCKS) - 1)) {
                    const uint32_t mine = (uint32_t)named >> half;
                    hide([&](int x) { return (mine >> (x >> 3) & 1) != 0; });
                }
                // two chains of three-way maxima
                float top = s[0][0], top1 = s[0][1];
#pragma unroll
                for (int i = 0; i < SUB; i++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        top = fmaxf(fmaxf(top, s[i][e]), s[i][e + 1]);
                        top1 = fmaxf(fmaxf(top1, s[i][e + 2]), s[i][e + 3]);
                    }
                top = scaled(fmaxf(top, top1), factor);
                if (__any(top - m > kOver<BF16, CAREFUL> + kLift<BF16>)) {
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float up = fmaxf(m, below<BF16, CAREFUL>(top));
                    const float keep = kept<CAREFUL>(__builtin_amdgcn_exp2f(m - up));
                    m = up;
                    sum *= keep;
#pragma unroll
                    for (int e = 0; e < DT; e++) o[e] *= keep;
                }
                u32x4 w[PT][SUB][2];
                float part[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < SUB; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float w0, w1;
                        if constexpr (CAREFUL) {
                            w0 = weight_of(scaled(s[i][2 * e], factor), m);
                            w1 = weight_of(scaled(s[i][2 * e + 1], factor), m);
                        } else {
                            w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][2 * e], factor, -m));
                            w1 = __builtin_amdgcn_exp2f(
                                __builtin_fmaf(s[i][2 * e + 1], factor, -m));
                        }
                        part[e & 3] += w0 + w1;
                        uint32_t x[PT];
                        terms16<BF16, PT>(w0, w1, x);
#pragma unroll
                        for (int k = 0; k < PT; k++) w[k][i][e >> 2][e & 3] = x[k];
                    }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
                for (int i = 0; i < SUB; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int e = 0; e < DT; e++) {
                            u32x2 part[2];
#pragma unroll
                            for (int x = 0; x < 2; x++)
                                part[x] = read_turned(v_sh[B] + (v_from ^ v_byte(0, e * 4)) +
                                                      (i * 32 + j * 16 + x * 4) * NC * 16);
                            const u32x4 vf = {part[0][0], part[0][1], part[1][0], part[1][1]};
#pragma unroll
                            for (int x = PT - 1; x >= 0; x--) o[e] = mfma32<BF16>(vf, w[x][i][j], o[e]);
                        }
                // the values that are not finite, for the rows that see them: whatever
                // the weight, the sum is what they are
                for (uint64_t odd = odd0 | (uint64_t)odd1 << 32; odd; odd &= odd - 1) {
                    const int x = pos + (int)__builtin_ctzll(odd);
                    const bool ok = (x <= p) & ((x > p - window) | (x < sinks));
                    const uint32_t page = table[(uint32_t)x >> c.shift];
                    const uint16_t* src = reinterpret_cast<const uint16_t*>(
                        values + (page < c.pages ? page : 0) * page_bytes +
                        (uint64_t)(head_row + ((uint32_t)x & row_mask)) * row_bytes);
#pragma unroll
                    for (int y = 0; y < DT; y++)
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const int d = y * 32 + 8 * z + 4 * half;
                            u32x2 f = {0, 0};
                            if (FULL || d < dim) f = *reinterpret_cast<const u32x2*>(src + d);
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float v = widen((uint16_t)(f[e >> 1] >> 16 * (e & 1)), BF16);
                                o[y][4 * z + e] += ok && !(fabsf(v) < INFINITY) ? v : 0.0f;
                            }
                        }
                }
            }
            if (more) {
                // every wave has passed the barrier above, so none reads this buffer
                pages = pages_next;
                arrive(pages, tile_pos(t + 1), odd_next, other, careful);
                pages_next = pages_after;
            }
        };
        for (int t = t_begin; t < t_end; t += 2) {
            step(t, std::integral_constant<int, 0>());
            if (t + 1 < t_end) step(t + 1, std::integral_constant<int, 1>());
        }
    };
    if (threadIdx.x == 0) again_sh = 0;
    pass(std::false_type());
    // past the head's dims there is whatever LDS held
    const auto counts = [&](int e, int i) { return FULL || e * 32 + 8 * i + 4 * half < dim; };
    // nor do scores from 2^20 on stand in one fused step with their maximum, which
    // is rounded: what that leaves out is 2^-4 there and soon past any weight
    const bool large = fabsf(m) >= 0x1p20f && m > kLowest;
    if (__any(real && (large || not_finite(sum, o, counts)))) again_sh = 1;
    __syncthreads();
    if (again_sh) pass(std::true_type());
    if (unnamed && wave == 0) report(fault, kFaultKvPage);
    if (held_shares > 1) {
        // a share's maximum, sum and values as the lanes hold them; the share to
        // arrive last adds them all, in the shares' order
        constexpr int kWords = DT * 16 + 2;
        const auto part = [&](int x) {
            return reinterpret_cast<uint64_t*>(parts) +
                   ((size_t)place * splits + x) * (kWords / 2 * 256) + threadIdx.x;
        };
        const auto put = [](uint64_t* p, float x, float y) {
            __hip_atomic_store(p, __builtin_bit_cast(uint64_t, (f32x2){x, y}), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        };
        const auto get = [](uint64_t* p) {
            return __builtin_bit_cast(
                f32x2, __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        uint64_t* mine = part((int)split);
        if (real) {
            put(mine, m, sum);
#pragma unroll
            for (int e = 0; e < DT; e++)
#pragma unroll
                for (int x = 0; x < 8; x++)
                    put(mine + (1 + e * 8 + x) * 256, o[e][2 * x], o[e][2 * x + 1]);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        uint32_t* ticket = tickets + (size_t)place * ticket_stride;
        if (threadIdx.x == 0)
            odd_sh[0][0] = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (odd_sh[0][0] != (uint32_t)held_shares - 1) return;
        if (threadIdx.x == 0)
            __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!real) return;
        m = kLowest;
        for (int x = 0; x < held_shares; x++) m = fmaxf(m, get(part(x))[0]);
        sum = 0;
#pragma unroll
        for (int e = 0; e < DT; e++)
#pragma unroll
            for (int z = 0; z < 16; z++) o[e][z] = 0;
        // two shares' loads in flight
        for (int x = 0; x < held_shares; x += 2) {
            uint64_t* from[2] = {part(x), part(x + 1 < held_shares ? x + 1 : x)};
            f32x2 ml[2], v[2][DT * 8];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                ml[y] = get(from[y]);
#pragma unroll
                for (int z = 0; z < DT * 8; z++) v[y][z] = get(from[y] + (1 + z) * 256);
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                if (x + y >= held_shares) break;
                const float f = kept<true>(__builtin_amdgcn_exp2f(ml[y][0] - m));
                sum += f * ml[y][1];
#pragma unroll
                for (int z = 0; z < DT * 8; z++) {
                    o[z >> 3][2 * (z & 7)] += f * v[y][z][0];
                    o[z >> 3][2 * (z & 7) + 1] += f * v[y][z][1];
                }
            }
        }
    }
    if (!real) return;
    sum += __shfl_xor(sum, 32, 64);
    const float scale = sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < DT; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = e * 32 + 8 * i + 4 * half;
            if (!FULL && d >= dim) continue;
            f32x4 v;
#pragma unroll
            for (int x = 0; x < 4; x++) v[x] = sum == 0 ? 0.0f : o[e][4 * i + x] * scale;
            if constexpr (F32) {
                *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + qrow + d) = v;
            } else {
                uint32_t x[2][1];
                terms16<BF16, 1>(v[0], v[1], x[0]);
                terms16<BF16, 1>(v[2], v[3], x[1]);
                *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + qrow + d) =
                    (u32x2){x[0][0], x[1][0]};
            }
        }
}

template <bool BF16, int QT, int PT, int DIM, bool FULL, bool MANY>
void decode(Device* d, hipStream_t st, const KvCache& c, const Attention& a, const uint32_t* sums,
            uint32_t heads, uint32_t stretches, uint32_t* tickets, float* parts) {
    const uint32_t grid = heads * stretches;
    hipLaunchKernelGGL((paged_decode_kernel<BF16, QT, PT, DIM, FULL, MANY>), dim3(grid),
                       dim3(64 * kWaves<DIM>), 0, st, c, a, sums, stretches, tickets,
                       (uint32_t)(kWorkspaceCounterBytes / 4) / grid, parts, d->fault_dev);
}

template <bool BF16, int QT, int PT, bool MANY>
void decode_dims(Device* d, hipStream_t st, const KvCache& c, const Attention& a,
                 const uint32_t* sums, uint32_t heads, uint32_t stretches, uint32_t* tickets,
                 float* parts) {
    const auto go = [&](auto f) { f(d, st, c, a, sums, heads, stretches, tickets, parts); };
    if (c.dim == 64) go(decode<BF16, QT, PT, 64, true, MANY>);
    else if (c.dim < 64) go(decode<BF16, QT, PT, 64, false, MANY>);
    else if (c.dim == 128) go(decode<BF16, QT, PT, 128, true, MANY>);
    else if (c.dim < 128) go(decode<BF16, QT, PT, 128, false, MANY>);
    else if (c.dim == 256) go(decode<BF16, QT, PT, 256, true, MANY>);
    else go(decode<BF16, QT, PT, 256, false, MANY>);
}

}  // namespace

bool paged_attention_counts(const KvCache& c, const Attention& a) {
    const uint64_t tiles = (((uint64_t)c.slots << c.shift) + 2 * kTile - 1) / kTile + 1;
    return (uint64_t)a.n * tiles <= 0xffffffffu;
}

hipError_t launch_paged_attention(Device* d, hipStream_t st, const KvCache& c,
                                  const Attention& a, int* status) {
    *status = ACCEL_OK;
    const int group = a.heads / c.heads;
    // a workgroup a CU holds as many loads in flight as the memory answers;
    // one a head is never cut, so past as many heads as CUs there are no joins
    // and no tickets
    const uint32_t heads = (uint32_t)(c.heads * ((group + 15) / 16));
    const uint32_t stretches = (uint32_t)d->cu_count > heads ? (uint32_t)d->cu_count / heads : 1;
    const size_t slot = (size_t)(group < 16 ? group : 16) * (c.dim + 2);
    const size_t part_words = stretches > 1 ? 2 * (size_t)heads * stretches * slot : 0;
    const bool summed = a.n > 64;
    const size_t sums_words = summed ? (((size_t)a.n + 63) & ~(size_t)63) : 0;
    char* ws = static_cast<char*>(
        workspace(d, st, (sums_words + part_words) * 4, status));
    if (!ws) return hipSuccess;
    uint32_t* sums = reinterpret_cast<uint32_t*>(ws + kWorkspaceCounterBytes);
    float* parts = reinterpret_cast<float*>(sums + sums_words);
    if (summed)
        hipLaunchKernelGGL(paged_sums_kernel, dim3(1), dim3(1024), 0, st, c, a, 0u, sums,
                           d->fault_dev);
    const auto go = [&](auto f) {
        f(d, st, c, a, summed ? sums : nullptr, heads, stretches,
          reinterpret_cast<uint32_t*>(ws), parts);
    };
    // Runs of short sequences need more than one a stretch, on average two; with
    // fewer the search for them costs 0.3 us and finds nothing (one of 200 tokens
    // 8.1 against 8.5 us).
    const bool many = (uint64_t)a.n * heads >= 2 * (uint64_t)d->cu_count;
    if (a.q_f32) {
        if (c.bf16) many ? go(decode_dims<true, 3, 3, true>) : go(decode_dims<true, 3, 3, false>);
        else many ? go(decode_dims<false, 2, 2, true>) : go(decode_dims<false, 2, 2, false>);
    } else {
        if (c.bf16) many ? go(decode_dims<true, 1, 2, true>) : go(decode_dims<true, 1, 2, false>);
        else many ? go(decode_dims<false, 1, 2, true>) : go(decode_dims<false, 1, 2, false>);
    }
    return hipGetLastError();
}

hipError_t launch_paged_prefill(Device* d, hipStream_t st, const KvCache& c, const Attention& a,
                                int* status) {
    *status = ACCEL_OK;
    const int group = a.heads / c.heads;
    const int per = prompt_heads(group), tokens = prompt_tokens(group);
    const uint32_t heads = (uint32_t)(c.heads * ((group + per - 1) / per));
    // an entry's last tile may be partly filled
    const uint64_t tiles = (uint64_t)a.rows / tokens + (a.n < a.rows ? a.n : a.rows);
    const uint64_t bound = tiles * heads;
    // two workgroups a CU of a 16-bit type up to 128 dims, else one; with fewer
    // tiles of rows than that, several workgroups share one
    const uint32_t slots = (uint32_t)d->cu_count * (!a.q_f32 && c.dim <= 128 ? 2 : 1);
    uint32_t splits = bound < slots ? (uint32_t)(slots / bound) : 1;
    // as many as the longest sequence's keys can be worth
    const int64_t kt = c.dim <= 128 ? 64 : 32;
    int64_t most = ((int64_t)c.slots << c.shift) / kt + 1;
    if (a.window) {
        const int64_t near = ((int64_t)a.window + tokens) / kt + a.sinks / kt + 3;
        most = near < most ? near : most;
    }
    const int64_t worth = most / (a.q_f32 ? kTilesAShare<true> : kTilesAShare<false>);
    splits = worth < (int64_t)splits ? (uint32_t)(worth > 1 ? worth : 1) : splits;
    const int wide = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    const size_t part_words =
        splits > 1 ? (size_t)(bound * splits) * 256 * (wide / 32 * 16 + 2) : 0;
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
    if (summed)
        hipLaunchKernelGGL(paged_sums_kernel, dim3(1), dim3(1024), 0, st, c, a, (uint32_t)tokens,
                           sums, d->fault_dev);
    const uint32_t fold = slots > (uint32_t)d->cu_count ? (uint32_t)d->cu_count / heads : 0;
    const uint32_t stride = (uint32_t)(kWorkspaceCounterBytes / 4) / slots;
    // a launch of 256 lanes a workgroup holds fewer than 2^24 of them, as a
    // grid's lanes are counted in 32 bits; that many places are not split
    constexpr uint64_t kPlaces = 1 << 22;
    const auto go = [&](auto kernel) {
        for (uint64_t place = 0; place < bound; place += kPlaces) {
            const uint64_t places = bound - place < kPlaces ? bound - place : kPlaces;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(places * splits)), dim3(256), 0, st, c, a,
                               sums, fold, splits, (uint32_t)place, tickets, stride, parts,
                               d->fault_dev);
        }
    };
    const bool full = c.dim == 64 || c.dim == 128 || c.dim == 256;
    const auto dims = [&](auto bf16, auto qt, auto pt) {
        constexpr bool B = decltype(bf16)::value;
        constexpr int Q = decltype(qt)::value, P = decltype(pt)::value;
        if (c.dim <= 64)
            full ? go(paged_prefill_kernel<B, Q, P, 64, true, 64>)
                 : go(paged_prefill_kernel<B, Q, P, 64, false, 64>);
        else if (c.dim <= 128)
            full ? go(paged_prefill_kernel<B, Q, P, 128, true, 64>)
                 : go(paged_prefill_kernel<B, Q, P, 128, false, 64>);
        else
            full ? go(paged_prefill_kernel<B, Q, P, 256, true, 32>)
                 : go(paged_prefill_kernel<B, Q, P, 256, false, 32>);
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
