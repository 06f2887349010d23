// What the kernels of attention over the paged cache share: products on the
// matrix cores, terms of f32 values, values that are not finite, the running
// maximum, and where a call's work is cut.  Included into one anonymous namespace
// per translation unit.
#pragma once

#include <hip/hip_runtime.h>

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

}  // namespace
}  // namespace accel
