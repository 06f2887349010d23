// A token of each row of logits, drawn from what its settings leave: in the order
// (value descending, index ascending), w_j = exp((x_j - max x) / T), the first k, of
// those the fewest whose sum reaches p of theirs, of those the w_j >= m, and of what
// is left the first whose running sum passes u of the sum.
//
// Nothing is sorted but what lies near a border.  All borders are places in one
// order, so a histogram over it finds them: with e = x log2(e) / T, the bin of a
// logit is 16 e rounded, i, and its weight 2^(i / 16) 2^(r / 16), |r| <= 1/2 the
// rest.  A pass over the logits adds up each bin's count and its 2^(r / 16), both in
// one 64-bit word, as whole numbers: the sums are exact and the same in any order.
// Sums over bins then say in which bins the borders of k, p, m and u lie; the logits
// of those few are gathered, sorted and weighed one by one.
//
// Bins are absolute, not relative to the row's largest, so one pass is enough: a ring
// of 1024 bins (64 factors of two) whose top follows the largest seen.  Weights below
// 2^-60 of the largest are left out.
#include <hip/hip_runtime.h>

#include "internal.hpp"

namespace accel {
namespace {

// A logit as a key: unsigned numbers in the logits' order, both zeros alike; a NaN
// is minus infinity, the lowest.
constexpr uint32_t kNoKey = 0x007fffffu;       // minus infinity's
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b >> 31 ? ~b : b | 0x80000000u;
    return x == x ? k : kNoKey;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

template <int DT>
__device__ __forceinline__ float logit(const void* p, size_t i) {
    if constexpr (DT == ACCEL_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == ACCEL_F16) return (float)static_cast<const _Float16*>(p)[i];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

// A number that all lanes have, for a scalar register.
__device__ __forceinline__ float uniform(float x) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}
__device__ __forceinline__ double uniform(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(
        double, (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) << 32 |
                    (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b));
}

// A row's settings, in range.
struct Rules {
    double temperature, top_p, min_p, u;
    uint32_t top_k;
    bool greedy;
};
__device__ __forceinline__ Rules rules_of(const Sampling& s, uint32_t row) {
    Rules r;
    const float t = s.temperature ? s.temperature[row] : 1.0f;
    r.greedy = !(t > 0);
    r.temperature = uniform((double)t);
    const float p = s.top_p ? s.top_p[row] : 1.0f;
    r.top_p = uniform((double)(p < 1 ? fmaxf(p, 0.0f) : 1.0f));
    const float m = s.min_p ? s.min_p[row] : 0.0f;
    r.min_p = uniform((double)(m > 0 ? fminf(m, 1.0f) : 0.0f));
    const float u = s.u[row];
    r.u = uniform((double)(u > 0 ? fminf(u, 1.0f - 0x1p-24f) : 0.0f));
    const uint32_t k = s.top_k ? s.top_k[row] : 0u;
    r.top_k = k ? k : 0xffffffffu;
    return r;
}

constexpr int kLanes = 1024, kWaves = kLanes / 64;
constexpr int kDigit = 11, kBins = 1 << kDigit;

struct RowScratch {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    uint64_t found_mass;
    uint32_t found_count, found, first, last;
};

// Weights are whole numbers, of 2^bits for the largest logit's: their sums are exact
// and the same in any order.
struct Weigher {
    double top, temperature, one;
    bool infinite;
    __device__ double share(uint32_t key) const {
        const float x = value_of(key);
        if (infinite) return x == INFINITY ? 1.0 : 0.0;
        if (x == -INFINITY) return 0.0;
        if (temperature == (double)INFINITY) return 1.0;
        return exp(((double)x - top) / temperature);
    }
    __device__ uint64_t operator()(uint32_t key) const {
        return (uint64_t)__double2ull_rn(share(key) * one);
    }
};

// The bin, from the highest down, in which `crosses(count, mass)` of the sums up to
// its end comes true; the last that holds anything where it never does.
template <typename F>
__device__ __forceinline__ uint32_t find_bin(RowScratch& sh, uint64_t mass0, uint32_t count0,
                                             F crosses) {
    constexpr int kPer = kBins / kLanes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) sh.first = 0xffffffffu, sh.last = 0;
    uint64_t mass = 0;
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const uint32_t b = kBins - 1 - (threadIdx.x * kPer + i);
        mass += sh.mass[b];
        count += sh.count[b];
    }
    uint64_t up_mass = mass;
    uint32_t up_count = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t m = __shfl_up(up_mass, d, 64);
        const uint32_t c = __shfl_up(up_count, d, 64);
        if (lane >= d) up_mass += m, up_count += c;
    }
    __syncthreads();
    if (lane == 63) sh.wave_mass[wave] = up_mass, sh.wave_count[wave] = up_count;
    __syncthreads();
    mass = mass0 + up_mass - mass;
    count = count0 + up_count - count;
    for (int w = 0; w < wave; w++) mass += sh.wave_mass[w], count += sh.wave_count[w];
    uint64_t mass_at[kPer];
    uint32_t count_at[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const uint32_t at = threadIdx.x * kPer + i, b = kBins - 1 - at;
        mass_at[i] = mass, count_at[i] = count;
        mass += sh.mass[b];
        count += sh.count[b];
        if (sh.count[b]) {
            atomicMax(&sh.last, at);
            if (crosses(count, mass)) atomicMin(&sh.first, at);
        }
    }
    __syncthreads();
    const uint32_t at = sh.first != 0xffffffffu ? sh.first : sh.last;
    if (at / kPer == threadIdx.x) {
        sh.found_mass = mass_at[at % kPer];
        sh.found_count = count_at[at % kPer];
    }
    __syncthreads();
    return kBins - 1 - at;
}

// Where in the order (value descending, index ascending) sums cross a border: a key,
// and what lies before the first logit of that key.
struct Place {
    uint32_t key, before;
    uint64_t mass;
};

// Which logits are still in: those above `key`, and of it the first `ties`, with a
// weight share of min_p or more.
struct Kept {
    uint32_t key, ties;
};

template <int DT, typename F>
__device__ Place cross_at(const void* row, uint32_t width, const Weigher& weigh, RowScratch& sh,
                          F crosses) {
    Place p = {0, 0, 0};
    int shift = 32;
    while (shift > 0) {
        const int bits = shift > kDigit ? kDigit : shift, low = shift - bits;
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += kLanes) sh.mass[b] = 0, sh.count[b] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < width; i += kLanes) {
            const uint32_t key = key_of(logit<DT>(row, i));
            if (key <= kNoKey || (shift < 32 && key >> shift != p.key >> shift)) continue;
            const uint32_t b = key >> low & ((1u << bits) - 1);
            atomicAdd(&sh.count[b], 1u);
            atomicAdd((unsigned long long*)&sh.mass[b], (unsigned long long)weigh(key));
        }
        __syncthreads();
        const uint32_t b = find_bin(sh, p.mass, p.before, crosses);
        p.key |= b << low;
        p.mass = sh.found_mass;
        p.before = sh.found_count;
        shift = low;
    }
    __syncthreads();
    return p;
}

// The workgroup's sum.
__device__ __forceinline__ uint64_t sum_of(RowScratch& sh, uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kWaves; w++) v += sh.wave_mass[w];
    __syncthreads();
    return v;
}

// The index of the logit of `key` that `nth` others of it come before.
template <int DT>
__device__ uint32_t index_of(const void* row, uint32_t width, uint32_t key, uint32_t nth,
                             RowScratch& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t per = ((width + kWaves - 1) / kWaves + 63) & ~63u;
    const uint32_t lo = wave * per, hi = lo + per < width ? lo + per : width;
    uint32_t count = 0;
    for (uint32_t i = lo; i < hi; i += 64)
        count += __popcll(__ballot(i + lane < hi && key_of(logit<DT>(row, i + lane)) == key));
    __syncthreads();
    if (lane == 0) sh.wave_count[wave] = count;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += sh.wave_count[w];
    if (nth >= before && nth < before + count) {
        for (uint32_t i = lo; i < hi; i += 64) {
            const uint64_t hit =
                __ballot(i + lane < hi && key_of(logit<DT>(row, i + lane)) == key);
            const uint32_t here = __popcll(hit);
            if (nth < before + here) {
                if ((hit >> lane & 1) &&
                    (uint32_t)__popcll(hit & ((1ull << lane) - 1)) == nth - before)
                    sh.found = i + lane;
                break;
            }
            before += here;
        }
    }
    __syncthreads();
    const uint32_t at = sh.found;
    __syncthreads();
    return at;
}


// ---- the histogram ------------------------------------------------------------

constexpr int kRing = 1024;            // bins of the ring: a lane each
constexpr int kCopies = 8;             // of each bin's word, for lanes that meet in it
constexpr int kReach = 960;            // bins below the largest's that count
constexpr int kList = 2048;            // logits near the borders, at most

// A bin's word: 2^49 for each logit, and 2^39 (2^(r / 16) - kLeast).  Up to 2^14 of
// them: the lower sum stays below 2^39 0.0434 2^14 < 2^49.
constexpr int kUnit = 39, kCount = 49;
constexpr double kLeast = 1002.0 / 1024;               // below 2^(-1 / 32)
constexpr uint64_t kLeastUnits = 1002ull << (kUnit - 10);
constexpr uint32_t kMostEach = 1u << 14;

// A logit's bin and its part of the bin's word.  2^(r / 16) to the fifth power of its
// series: off by (ln 2 / 32)^6 / 720 = 2^-42.7 of it, and rounded by 2^-40.  Bins have
// to be the same wherever they are asked for, so no sum is fused here that is not
// written so.
struct Binned {
    int bin;
    uint64_t word;
};
__device__ __forceinline__ Binned binned(float x, double per) {
#pragma clang fp contract(off)
    constexpr double kMagic = 6755399441055744.0;      // 3 * 2^51: the sum's low word is whole
    constexpr double z = 0.69314718055994530942 / 16;
    constexpr double c1 = z, c2 = z * z / 2, c3 = z * z * z / 6, c4 = z * z * z * z / 24,
                     c5 = z * z * z * z * z / 120;
    constexpr double kBase = 8192.0;                   // its last place is 2^-39
    const double e = (double)x * per;
    const double t = e + kMagic;
    const double r = e - (t - kMagic);
    double q = __builtin_fma(c5, r, c4);
    q = __builtin_fma(q, r, c3);
    q = __builtin_fma(q, r, c2);
    q = __builtin_fma(q, r, c1);
    q = __builtin_fma(q, r, kBase + (1 - kLeast));
    return {(int)(uint32_t)__builtin_bit_cast(uint64_t, t),
            __builtin_bit_cast(uint64_t, q) -
                (__builtin_bit_cast(uint64_t, kBase) - (1ull << kCount))};
}
// Logits per bin's width: 16 log2(e) / T.
__device__ __forceinline__ double bins_per(const Rules& r) {
    return uniform(16 * 1.44269504088896340736 / r.temperature);
}
// A weight in units of 2^-39 of 2^(bin / 16), exact.
__device__ __forceinline__ uint64_t units(uint64_t count, uint64_t rest) {
    return count * kLeastUnits + rest;
}
__device__ __forceinline__ uint64_t units_of(const Binned& b) {
    return units(1, b.word & ((1ull << kCount) - 1));
}

// A row as aligned blocks of 16 bytes; what its ends leave of the first and the last
// is no number.
template <int DT>
struct Blocks {
    static constexpr int kEach = DT == ACCEL_F32 ? 4 : 8;
    const char* base;
    uint32_t before, end;              // places of the row's first logit and past its last
    uint32_t count;
    __device__ Blocks(const Sampling& s, uint32_t row) {
        constexpr int size = 16 / kEach;
        const uintptr_t at = (uintptr_t)s.logits + (size_t)row * s.width * size;
        base = reinterpret_cast<const char*>(at & ~(uintptr_t)15);
        before = (uint32_t)(at & 15) / size;
        end = before + s.width;
        count = (end + kEach - 1) / kEach;
    }
    __device__ void read(uint32_t b, float* x) const {
        const uint32_t place = b * kEach;
        const char* at = base + (size_t)b * 16;
        if (place >= before && place + kEach <= end) {
            const uint4 w = *reinterpret_cast<const uint4*>(at);
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < kEach; e++) x[e] = part(v, e);
        } else {
#pragma unroll
            for (int e = 0; e < kEach; e++)
                x[e] = place + e >= before && place + e < end ? logit<DT>(at, e) : -INFINITY;
        }
    }
    static __device__ float part(const uint32_t (&v)[4], int e) {
        if constexpr (DT == ACCEL_F32) return __uint_as_float(v[e]);
        else if constexpr (DT == ACCEL_BF16)
            return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[e >> 1] >> 16 * (e & 1)));
    }
};
constexpr int kTile = 16;              // logits a lane reads at once

// Tile t's logits of this lane, of the blocks [first, last).
template <int DT>
__device__ __forceinline__ void read_tile(const Blocks<DT>& row, uint32_t first, uint32_t last,
                                          uint32_t t, float (&x)[kTile]) {
    constexpr int E = Blocks<DT>::kEach;
#pragma unroll
    for (int q = 0; q < kTile / E; q++) {
        const uint32_t b = first + (t * (kTile / E) + q) * kLanes + threadIdx.x;
        if (b < last) row.read(b, x + q * E);
        else
#pragma unroll
            for (int e = 0; e < E; e++) x[q * E + e] = -INFINITY;
    }
}
template <int DT>
__device__ __forceinline__ uint32_t index_in(const Blocks<DT>& row, uint32_t first, uint32_t t,
                                             int e) {
    constexpr int E = Blocks<DT>::kEach;
    return (first + (t * (kTile / E) + e / E) * kLanes + threadIdx.x) * E + e % E - row.before;
}
__device__ __forceinline__ float largest(const float (&x)[kTile]) {
    float m = fmaxf(x[0], x[1]);
#pragma unroll
    for (int e = 2; e < kTile; e++) m = fmaxf(m, x[e]);
    return m;
}

// Sums of a row's bins, from the largest's down, and where its borders lie.
struct Span {
    int lo, hi;                        // bins below the largest's
};
struct Plan {
    float top;                         // the row's largest logit
    uint32_t listed;                   // logits of the bins below
    double all;                        // the row's sum
    Span k, p, m, s;                   // an empty one: hi < lo
};
struct Sums {
    double mass[kRing];                // up to the bin's end
    uint32_t count[kRing];
};
struct Scratch {
    union {
        uint64_t ring[kRing * kCopies + kCopies];      // the last: logits of no bin
        struct {
            Sums sums;
            uint64_t list[kList];
            double upto[kList];         // the row's sum up to a listed logit's end
            uint32_t rank[kList];       // its place in the order
            int bin[kList];
        };
        RowScratch slow;
    };
    Plan plan;
    double wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float wave_top[kWaves];
    int first[4];
    uint32_t listed, last;
};

__device__ __forceinline__ float top_of(Scratch& sh, float m) {
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if ((threadIdx.x & 63) == 0) sh.wave_top[threadIdx.x >> 6] = m;
    __syncthreads();
    m = sh.wave_top[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) m = fmaxf(m, sh.wave_top[w]);
    __syncthreads();
    return uniform(m);
}

// Bins below a window's top that its ring holds, whatever the edges' roundings.
constexpr int kLow = 1008;
// The ring's window: bins up to top, and the logits that fall into it.
struct Window {
    int top;
    float low, high;
    __device__ void set(int bin, double per) {
        top = __builtin_amdgcn_readfirstlane(bin);
        high = uniform((float)((top - 1) / per));
        low = uniform((float)((top - (kLow - 1)) / per));
    }
};
// Whether a row's bins are whole numbers near which it can be weighed: places are
// right to 2^-36 of a bin up to here, weights to 2^-40.5.
__device__ __forceinline__ bool has_bins(float top, double per) {
    return fabs((double)top * per) < 0x1p17 && per > 0x1p-60;
}

__device__ __forceinline__ void clear_ring(Scratch& sh) {
    uint4* p = reinterpret_cast<uint4*>(sh.ring);
#pragma unroll
    for (int i = 0; i < kRing * kCopies / 2 / kLanes; i++)
        p[i * kLanes + threadIdx.x] = make_uint4(0, 0, 0, 0);
}
// Adds a lane's logits that are in; the others' words go where nobody reads, without a
// branch a logit.
template <typename F>
__device__ __forceinline__ void add_to_ring(Scratch& sh, const float (&x)[kTile], double per,
                                            F in) {
    uint64_t* mine = sh.ring + (threadIdx.x & (kCopies - 1));
#pragma unroll
    for (int e = 0; e < kTile; e++) {
        const Binned b = binned(x[e], per);
        const int slot = in(x[e]) ? b.bin & (kRing - 1) : kRing;
        atomicAdd((unsigned long long*)(mine + slot * kCopies), (unsigned long long)b.word);
        // a few at a time: registers
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}
// This lane's bin, so many below top: its copies' sum.
__device__ __forceinline__ void read_ring(const Scratch& sh, int top, uint32_t* count,
                                          uint64_t* rest) {
    const uint64_t* p = &sh.ring[((top - (int)threadIdx.x) & (kRing - 1)) * kCopies];
    *count = 0, *rest = 0;
#pragma unroll
    for (int i = 0; i < kCopies; i++) {
        *count += (uint32_t)(p[i] >> kCount);
        *rest += p[i] & ((1ull << kCount) - 1);
    }
}

// The first lane for which it holds, or `none`; all lanes call it.
template <int N>
__device__ __forceinline__ void first_lanes(Scratch& sh, const bool (&is)[N], int none,
                                            int (&at)[N]) {
    if (threadIdx.x < N) sh.first[threadIdx.x] = none;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t b = __ballot(is[i]);
        if (b && (threadIdx.x & 63) == 0)
            atomicMin(&sh.first[i], (int)(threadIdx.x & ~63u) + (int)__builtin_ctzll(b));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) at[i] = sh.first[i];
    __syncthreads();
}

// Where the borders lie, from each lane's bin (so many below the largest's).  What a
// border leaves or cuts off of its bin is not known yet, so a sum behind it lies
// between two, and the bins where the next border may be with it.
__device__ void make_plan(Scratch& sh, const Rules& rules, float top, double per, uint32_t count,
                          uint64_t rest) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = threadIdx.x;
    const Binned big = binned(top, per);
    const uint64_t one = units_of(big);
    double mass = 0;
    if (d >= kReach) count = 0, rest = 0;
    if (count) {
        const uint64_t all = units(count, rest);
        // the largest's own bin in whole weights and their rest, so that equal logits'
        // sums are whole
        if (d == 0) mass = (double)(all / one) + (double)(all % one) / (double)one;
        else mass = (double)all / (double)one * exp2(-d / 16.0);
    }
    double up = mass;
    uint32_t up_count = count;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const double m = __shfl_up(up, x, 64);
        const uint32_t c = __shfl_up(up_count, x, 64);
        if (lane >= x) up += m, up_count += c;
    }
    if (lane == 63) sh.wave_mass[wave] = up, sh.wave_count[wave] = up_count;
    __syncthreads();                    // every lane has read the ring, too
    double before = 0;
    uint32_t before_count = 0;
    for (int w = 0; w < wave; w++) before += sh.wave_mass[w], before_count += sh.wave_count[w];
    const double inc = before + up;
    const uint32_t inc_count = before_count + up_count;
    sh.sums.mass[d] = inc;
    sh.sums.count[d] = inc_count;
    __syncthreads();
    const double all = sh.sums.mass[kRing - 1];
    const uint32_t all_count = sh.sums.count[kRing - 1];
    const auto mass_before = [&](int b) { return b > 0 ? sh.sums.mass[b - 1] : 0.0; };
    Plan plan;
    plan.top = top;
    plan.k = plan.p = plan.m = plan.s = {0, -1};
    double lo = all, hi = all;          // what is kept
    int end = kRing - 1;
    {
        const bool is[2] = {inc_count >= rules.top_k, inc_count >= all_count};
        int at[2];
        first_lanes<2>(sh, is, kRing - 1, at);
        end = at[1];                    // the last that holds any
        if (rules.top_k < all_count) {
            end = at[0];
            plan.k = {at[0], at[0]};
            lo = mass_before(at[0]), hi = sh.sums.mass[at[0]];
        }
    }
    if (rules.top_p < 1) {
        const bool is[2] = {inc >= rules.top_p * lo, inc >= rules.top_p * hi};
        int at[2];
        first_lanes<2>(sh, is, end, at);
        // an empty bin has its predecessor's sum, so a border is in one that holds any
        plan.p = {at[0] < end ? at[0] : end, at[1] < end ? at[1] : end};
        lo = mass_before(plan.p.lo);
        hi = sh.sums.mass[plan.p.hi];
        end = plan.p.hi;
    }
    if (rules.min_p > 0) {
        const double e = (double)top * per;
        const double r = e - rint(e);
        // bins before this one are kept whole, those past it not at all
        const double at = rint(-16 * log2(rules.min_p) - r);
        if (at <= end) {
            end = at > 0 ? (int)at : 0;
            plan.m = {end, end};
            lo = fmin(lo, mass_before(end));
            hi = fmin(hi, sh.sums.mass[end]);
        }
    }
    {
        const bool is[2] = {inc > rules.u * lo, inc > rules.u * hi};
        int at[2];
        first_lanes<2>(sh, is, end, at);
        plan.s = {at[0] < end ? at[0] : end, at[1] < end ? at[1] : end};
    }
    plan.all = all;
    const auto in = [](const Span& s, int b) { return b >= s.lo && b <= s.hi; };
    const bool need = in(plan.k, d) || in(plan.p, d) || in(plan.m, d) || in(plan.s, d);
    uint32_t listed = need ? count : 0;
#pragma unroll
    for (int x = 32; x; x >>= 1) listed += __shfl_xor(listed, x, 64);
    if (lane == 0) sh.wave_count[wave] = listed;
    __syncthreads();
    listed = 0;
    for (int w = 0; w < kWaves; w++) listed += sh.wave_count[w];
    plan.listed = listed;
    if (threadIdx.x == 0) sh.plan = plan;
    __syncthreads();
}
__device__ __forceinline__ bool needed(const Plan& p, int d) {
    return (d >= p.k.lo && d <= p.k.hi) || (d >= p.p.lo && d <= p.p.hi) ||
           (d >= p.m.lo && d <= p.m.hi) || (d >= p.s.lo && d <= p.s.hi);
}
__device__ __forceinline__ int last_needed(const Plan& p) {
    const int a = p.k.hi > p.p.hi ? p.k.hi : p.p.hi, b = p.m.hi > p.s.hi ? p.m.hi : p.s.hi;
    return a > b ? a : b;
}

// Place in the order, ascending.
__device__ __forceinline__ uint64_t placed(float x, uint32_t index) {
    return (uint64_t)~key_of(x) << 32 | index;
}

// Lists a lane's logits of the plan's bins, none of which holds one below low.
template <typename F>
__device__ __forceinline__ void list_near(Scratch& sh, const Plan& plan, int top, float low,
                                          double per, const float (&x)[kTile], F index) {
#pragma unroll
    for (int e = 0; e < kTile; e++)
        if (x[e] >= low && needed(plan, top - binned(x[e], per).bin)) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            if (at < kList) sh.list[at] = placed(x[e], index(e));
        }
}

// Sorts sh.list[0 .. n) up; n <= kList.  A lane an element up to kLanes, exchanged
// within a wave without LDS.
__device__ void sort_list(Scratch& sh, uint32_t n) {
    constexpr int kPer = kList / kLanes;
    const uint32_t size = n <= 64 ? 64 : 1u << (32 - __builtin_clz(n - 1));
    const int per = size > kLanes ? (int)(size / kLanes) : 1;
    for (uint32_t i = n + threadIdx.x; i < size; i += kLanes) sh.list[i] = ~0ull;
    __syncthreads();
    uint64_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++)
        v[i] = i < per && i * kLanes + threadIdx.x < size ? sh.list[i * kLanes + threadIdx.x] : ~0ull;
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t j = k >> 1; j; j >>= 1) {
            if (j >= 64) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kPer; i++)
                    if (i < per && i * kLanes + threadIdx.x < size)
                        sh.list[i * kLanes + threadIdx.x] = v[i];
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const uint32_t x = i * kLanes + threadIdx.x;
                if (j < 64 || (i < per && x < size)) {
                    const uint64_t o = j < 64 ? __shfl_xor(v[i], (int)j, 64) : sh.list[x ^ j];
                    const bool up = (x & k) == 0, low = (x & j) == 0;
                    if ((o < v[i]) == (up == low)) v[i] = o;
                }
            }
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; i++)
        if (i < per && i * kLanes + threadIdx.x < size) sh.list[i * kLanes + threadIdx.x] = v[i];
    __syncthreads();
}

// The first of the list's n elements, one past the other, for which it holds, or n.
template <typename F>
__device__ uint32_t first_listed(Scratch& sh, uint32_t n, F is) {
    __syncthreads();
    if (threadIdx.x == 0) sh.first[0] = (int)n;
    __syncthreads();
    for (uint32_t base = 0; base < n; base += kLanes) {
        const uint32_t i = base + threadIdx.x;
        const uint64_t b = __ballot(i < n && is(i));
        if (b && (threadIdx.x & 63) == 0)
            atomicMin(&sh.first[0], (int)(i + __builtin_ctzll(b)));
    }
    __syncthreads();
    return (uint32_t)sh.first[0];
}

// The token, from the sums over bins and the n logits of the plan's bins.
__device__ void draw(Scratch& sh, const Sampling& s, uint32_t row, const Rules& rules, double per,
                     uint32_t n) {
    sort_list(sh, n);
    const Plan plan = sh.plan;
    const Binned big = binned(plan.top, per);
    const double one = (double)units_of(big);
    const auto binned_at = [&](uint32_t i) {
        return binned(value_of(~(uint32_t)(sh.list[i] >> 32)), per);
    };
    const auto weight_of = [&](const Binned& b) {
        const int d = big.bin - b.bin;
        const double w = (double)units_of(b) / one;
        return d ? w * exp2(-d / 16.0) : w;
    };
    const auto mass_before = [&](int d) { return d ? sh.sums.mass[d - 1] : 0.0; };
    const auto count_before = [&](int d) { return d ? sh.sums.count[d - 1] : 0u; };
    // the first listed logit of bin d or one past it
    const auto start_of = [&](int d) {
        uint32_t lo = 0, hi = n;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (sh.bin[mid] < d) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    // running sums of the list, kLanes at a time, then of the row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double carry = 0;
    for (uint32_t base = 0; base < n; base += kLanes) {
        const uint32_t i = base + threadIdx.x;
        double up = 0;
        if (i < n) {
            const Binned b = binned_at(i);
            sh.bin[i] = big.bin - b.bin;
            up = weight_of(b);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const double m = __shfl_up(up, x, 64);
            if (lane >= x) up += m;
        }
        if (lane == 63) sh.wave_mass[wave] = up;
        __syncthreads();
        double before = carry;
        for (int w = 0; w < kWaves; w++) {
            if (w < wave) before += sh.wave_mass[w];
            carry += sh.wave_mass[w];
        }
        if (i < n) sh.upto[i] = before + up;
        __syncthreads();
    }
    double upto[kList / kLanes];
#pragma unroll
    for (int x = 0; x < kList / kLanes; x++) {
        const uint32_t i = x * kLanes + threadIdx.x;
        if (i >= n) continue;
        const int d = sh.bin[i];
        const uint32_t at = start_of(d);
        upto[x] = mass_before(d) + (sh.upto[i] - (at ? sh.upto[at - 1] : 0.0));
        sh.rank[i] = count_before(d) + (i - at);
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kList / kLanes; x++) {
        const uint32_t i = x * kLanes + threadIdx.x;
        if (i < n) sh.upto[i] = upto[x];
    }
    __syncthreads();
    double kept = plan.all;
    uint32_t count = sh.sums.count[kRing - 1];
    const auto cut = [&](double mass, uint32_t upto_count) {
        if (upto_count < count) kept = mass, count = upto_count;
    };
    if (plan.k.lo <= plan.k.hi) {
        const uint32_t i = start_of(plan.k.lo) + (rules.top_k - 1 - count_before(plan.k.lo));
        kept = sh.upto[i < n ? i : n - 1];
        count = rules.top_k;
    }
    // the first in a span of bins whose sum is past a border, or the span's last
    const auto crossing = [&](const Span& span, auto past) {
        const uint32_t lo = start_of(span.lo), hi = start_of(span.hi + 1);
        const uint32_t i =
            first_listed(sh, hi, [&](uint32_t x) { return x >= lo && past(sh.upto[x]); });
        return i < hi ? i : hi - 1;
    };
    if (plan.p.lo <= plan.p.hi) {
        const double border = rules.top_p * kept;
        const uint32_t i = crossing(plan.p, [&](double m) { return m >= border; });
        cut(sh.upto[i], sh.rank[i] + 1);
    }
    if (plan.m.lo <= plan.m.hi) {
        const int d = plan.m.lo;
        const uint32_t lo = start_of(d), hi = start_of(d + 1);
        const uint32_t i = first_listed(sh, hi, [&](uint32_t x) {
            return x >= lo && !(weight_of(binned_at(x)) >= rules.min_p);
        });
        if (i > lo) cut(sh.upto[i - 1], sh.rank[i - 1] + 1);
        else cut(mass_before(d), count_before(d));
    }
    const double border = rules.u * kept;
    uint32_t i = crossing(plan.s, [&](double m) { return m > border; });
    // sums of bins and of their logits are rounded apart
    while (i && sh.rank[i] >= count) i--;
    if (threadIdx.x == 0) {
        s.tokens[row] = (uint32_t)sh.list[i];
        if (s.logprobs) s.logprobs[row] = (float)log(weight_of(binned_at(i)) / kept);
    }
    __syncthreads();
}

// ---- the kernels ----------------------------------------------------------------

// A row that has no bins, or too many logits near its borders: place by place.
template <int DT>
__device__ __attribute__((noinline)) void draw_slowly(RowScratch& sh, const Sampling& s, uint32_t r, const Rules& rules,
                            float top) {
    const void* row = static_cast<const char*>(s.logits) +
                      (size_t)r * s.width * (DT == ACCEL_F32 ? 4 : 2);
    const Weigher weigh = {(double)top, rules.temperature,
                           (double)(1ull << (31 + __builtin_clz(s.width))),
                           top == INFINITY};
    // top-k, then the whole mass of what it leaves
    Kept kept = {kNoKey + 1, 0xffffffffu};
    uint64_t whole;
    if (rules.top_k < s.width) {
        const Place p = cross_at<DT>(row, s.width, weigh, sh, [&](uint32_t n, uint64_t) {
            return n >= rules.top_k;
        });
        // fewer than k: all of them
        kept = {p.key, rules.top_k - p.before};
        uint64_t ties = 0;
        for (uint32_t i = threadIdx.x; i < s.width; i += kLanes)
            ties += key_of(logit<DT>(row, i)) == p.key;
        ties = sum_of(sh, ties);
        if (ties < kept.ties) kept.ties = (uint32_t)ties;
        whole = p.mass + kept.ties * weigh(p.key);
    } else {
        uint64_t mass = 0;
        for (uint32_t i = threadIdx.x; i < s.width; i += kLanes) {
            const uint32_t key = key_of(logit<DT>(row, i));
            if (key > kNoKey) mass += weigh(key);
        }
        whole = sum_of(sh, mass);
    }
    if (rules.top_p < 1) {
        const double border = rules.top_p * (double)whole;
        const Place p = cross_at<DT>(row, s.width, weigh, sh, [&](uint32_t, uint64_t mass) {
            return (double)mass >= border;
        });
        // the fewest of its ties that reach the border
        const uint64_t w = weigh(p.key);
        const double need = w ? ceil((border - (double)p.mass) / (double)w) : 1.0;
        const uint32_t ties = need > 1 ? (uint32_t)fmin(need, 4294967295.0) : 1u;
        if (p.key > kept.key || (p.key == kept.key && ties < kept.ties)) kept = {p.key, ties};
    }
    uint64_t mass = 0;
    uint32_t ties = 0;
    for (uint32_t i = threadIdx.x; i < s.width; i += kLanes) {
        const uint32_t key = key_of(logit<DT>(row, i));
        if (key > kept.key && weigh.share(key) >= rules.min_p) mass += weigh(key);
        ties += key == kept.key;
    }
    mass = sum_of(sh, mass);
    ties = (uint32_t)sum_of(sh, ties);
    if (ties > kept.ties) ties = kept.ties;
    if (weigh.share(kept.key) >= rules.min_p) mass += ties * weigh(kept.key);
    else ties = 0;
    const double border = rules.u * (double)mass;
    const Place p = cross_at<DT>(row, s.width, weigh, sh, [&](uint32_t, uint64_t m) {
        return (double)m > border;
    });
    const uint64_t w = weigh(p.key);
    uint32_t nth = 0;
    if (w) {
        const double past = floor((border - (double)p.mass) / (double)w);
        nth = past > 0 ? (uint32_t)past : 0u;
    }
    // roundings of the division
    while (nth && (double)(p.mass + nth * w) > border) nth--;
    while ((double)(p.mass + (nth + 1) * w) <= border && w) nth++;
    if (p.key == kept.key && ties && nth >= ties) nth = ties - 1;
    const uint32_t at = index_of<DT>(row, s.width, p.key, nth, sh);
    if (threadIdx.x == 0) {
        s.tokens[r] = at;
        if (s.logprobs)
            s.logprobs[r] = (float)log(weigh.share(p.key) * weigh.one / (double)mass);
    }
    __syncthreads();
}

// The first of a row's order: its least place.
__device__ __forceinline__ uint64_t least_of(Scratch& sh, uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint64_t o = __shfl_xor(v, d, 64);
        v = o < v ? o : v;
    }
    if ((threadIdx.x & 63) == 0) sh.list[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.list[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) v = sh.list[w] < v ? sh.list[w] : v;
    __syncthreads();
    return v;
}
template <int DT>
__device__ __forceinline__ uint64_t least_in(const Blocks<DT>& row, uint32_t first, uint32_t last) {
    constexpr uint32_t kStep = kTile / Blocks<DT>::kEach * kLanes;
    float best = -INFINITY;
    uint32_t at = 0;
    for (uint32_t t = 0; t * kStep < last - first; t++) {
        float x[kTile];
        read_tile<DT>(row, first, last, t, x);
        // a lane's logits are read in their order, but for the blocks of a tile
#pragma unroll
        for (int e = 0; e < kTile; e++)
            if (x[e] > best) best = x[e], at = index_in<DT>(row, first, t, e);
    }
    return best > -INFINITY ? placed(best, at) : ~0ull;
}
__device__ __forceinline__ void give_first(const Sampling& s, uint32_t row, uint64_t least) {
    if (threadIdx.x) return;
    const bool any = least != ~0ull;
    s.tokens[row] = any ? (uint32_t)least : ACCEL_NO_TOKEN;
    if (s.logprobs) s.logprobs[row] = any ? 0.0f : -INFINITY;
}

// Rows of up to kTiles tiles, a workgroup each, two workgroups a CU.  Of each tile of a
// lane it is kept how far its largest logit is from the top, so the second look goes
// only to what may hold something near a border.
constexpr int kTiles = 8;
constexpr int kFar = 255;              // below the window; nearer ones are 253 at most
static_assert(kTiles * kTile * kLanes / kCopies <= kMostEach, "a word's count and sum");
static_assert(kTile * kLanes <= kMostEach, "the same, of a part's copies together");

template <int DT>
__global__ __launch_bounds__(kLanes, 8) void sample_whole_kernel(Sampling s, uint32_t first_row) {
    __shared__ Scratch sh;
    __shared__ uint8_t far[kTiles][kLanes];
    constexpr uint32_t kStep = kTile / Blocks<DT>::kEach * kLanes;
    const uint32_t r = first_row + blockIdx.x;
    const Rules rules = rules_of(s, r);
    const Blocks<DT> row(s, r);
    if (rules.greedy) {
        give_first(s, r, least_of(sh, least_in<DT>(row, 0, row.count)));
        return;
    }
    const double per = bins_per(rules);
    float x[kTile];
    read_tile<DT>(row, 0, row.count, 0, x);
    float top = largest(x);
    clear_ring(sh);
    // the window is set by the first tile, with room for the rest to pass it by a
    // factor of four; what passes it further is added afterwards
    const float first = top_of(sh, top);
    const bool bins = has_bins(first, per);
    Window w = {0, INFINITY, -INFINITY};
    if (bins) w.set(binned(first, per).bin + 32, per);
#pragma clang loop unroll(disable)
    for (uint32_t t = 0;;) {
        const float m = largest(x);
        top = fmaxf(top, m);
        // how far the lane's largest is from the window's top
        int code = kFar;
        if (m > w.high) code = 0;
        else if (m >= w.low) code = 1 + ((w.top - binned(m, per).bin) >> 2);
        far[t][threadIdx.x] = (uint8_t)code;
        add_to_ring(sh, x, per, [&](float v) { return v >= w.low && v <= w.high; });
        if (++t * kStep >= row.count) break;
        read_tile<DT>(row, 0, row.count, t, x);
    }
    top = top_of(sh, top);
    if (top == -INFINITY) {
        give_first(s, r, ~0ull);
        return;
    }
    bool listed = has_bins(top, per);
    if (listed) {
        const int bin = __builtin_amdgcn_readfirstlane(binned(top, per).bin);
        if (top > w.high) {
            const int past = bins ? bin - w.top : kRing;
            if (past >= kRing) {
                clear_ring(sh);
            } else if ((int)threadIdx.x < past) {
                uint64_t* p = &sh.ring[((bin - (int)threadIdx.x) & (kRing - 1)) * kCopies];
#pragma unroll
                for (int i = 0; i < kCopies; i++) p[i] = 0;
            }
            __syncthreads();
            const float low = (float)((bin - (kLow - 1)) / per);
#pragma clang loop unroll(disable)
            for (uint32_t t = 0; t * kStep < row.count; t++) {
                if (far[t][threadIdx.x]) continue;
                read_tile<DT>(row, 0, row.count, t, x);
                add_to_ring(sh, x, per, [&](float v) { return v > w.high && v >= low; });
            }
            __syncthreads();
        }
        uint32_t count;
        uint64_t rest;
        read_ring(sh, bin, &count, &rest);
        make_plan(sh, rules, top, per, count, rest);
        const Plan plan = sh.plan;
        listed = plan.listed && plan.listed <= kList;
        if (listed) {
            if (threadIdx.x == 0) sh.listed = 0;
            __syncthreads();
            const float low = (float)((bin - last_needed(plan) - 1) / per);
            const int most = bins ? 1 + ((w.top - bin + last_needed(plan)) >> 2) : 0;
#pragma clang loop unroll(disable)
            for (uint32_t t = 0; t * kStep < row.count; t++) {
                const int code = far[t][threadIdx.x];
                if (code && code > most) continue;
                read_tile<DT>(row, 0, row.count, t, x);
                list_near(sh, plan, bin, low, per, x,
                          [&](int e) { return index_in<DT>(row, 0, t, e); });
            }
            __syncthreads();
            draw(sh, s, r, rules, per, sh.listed < kList ? sh.listed : kList);
        }
    }
    if (!listed) draw_slowly<DT>(sh.slow, s, r, rules, top);
}

// Longer rows, and too few rows to fill the chip: a workgroup a part of up to one tile.
// The last of a row's parts to end adds up their bins and goes on as above.
constexpr int kBatch = 8;              // parts whose words are asked for at once
constexpr int kMostParts = ACCEL_SAMPLE_WIDTH / (kTile * kLanes) + kBatch;
struct Parts {
    uint64_t* rings;                   // [rows, parts, kRing]
    uint64_t* least;                   // [rows, parts]
    float* tops;                       // [rows, parts]
    uint8_t* far;                      // [rows, parts, kLanes]
    uint32_t* tickets;                 // [rows]: zero between calls
    uint32_t first, parts, blocks;     // the launch's first row; a part's blocks
};

template <typename T>
__device__ __forceinline__ void put(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of `parts` here; what they stored is there then.
__device__ __forceinline__ bool is_last(Scratch& sh, uint32_t* ticket, uint32_t parts) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.listed = 0;
        sh.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        if (sh.last) put(ticket, 0u);
    }
    __syncthreads();
    return sh.last != 0;
}

template <int DT>
__global__ __launch_bounds__(kLanes, 8) void sample_parts_kernel(Sampling s, Parts p) {
    __shared__ Scratch sh;
    __shared__ int bins[kMostParts];
    const uint32_t local = blockIdx.x / p.parts, part = blockIdx.x - local * p.parts;
    const uint32_t r = p.first + local;
    const Rules rules = rules_of(s, r);
    const Blocks<DT> row(s, r);
    const auto begin_of = [&](uint32_t i) {
        return i * p.blocks < row.count ? i * p.blocks : row.count;
    };
    const uint32_t begin = begin_of(part), end = begin_of(part + 1);
    const size_t slot0 = (size_t)local * p.parts, slot = slot0 + part;
    const double per = bins_per(rules);
    float x[kTile];
    if (rules.greedy) {
        const uint64_t least = least_of(sh, least_in<DT>(row, begin, end));
        if (threadIdx.x == 0) put(p.least + slot, least);
    } else {
        read_tile<DT>(row, begin, end, 0, x);
        clear_ring(sh);
        const float most = largest(x);
        const float top = top_of(sh, most);
        if (threadIdx.x == 0) put(p.tops + slot, top);
        if (top > -INFINITY && has_bins(top, per)) {
            Window w;
            w.set(binned(top, per).bin, per);
            int code = kFar;
            if (most >= w.low) code = (w.top - binned(most, per).bin) >> 2;
            put(p.far + slot * kLanes + threadIdx.x, (uint8_t)code);
            add_to_ring(sh, x, per, [&](float v) { return v >= w.low; });
            __syncthreads();
            uint32_t count;
            uint64_t rest;
            read_ring(sh, w.top, &count, &rest);
            put(p.rings + slot * kRing + ((w.top - (int)threadIdx.x) & (kRing - 1)),
                (uint64_t)count << kCount | rest);
        }
    }
    if (!is_last(sh, p.tickets + local, p.parts)) return;
    if (rules.greedy) {
        uint64_t least = ~0ull;
        for (uint32_t i = threadIdx.x; i < p.parts; i += kLanes) {
            const uint64_t v = get(p.least + slot0 + i);
            least = v < least ? v : least;
        }
        give_first(s, r, least_of(sh, least));
        return;
    }
    constexpr int kNone = 1 << 30;
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < p.parts; i += kLanes) {
        const float t = get(p.tops + slot0 + i);
        top = fmaxf(top, t);
        bins[i] = !(t > -INFINITY) ? -kNone : has_bins(t, per) ? binned(t, per).bin : kNone;
    }
    top = top_of(sh, top);
    for (uint32_t i = threadIdx.x; i < p.parts; i += kLanes) {
        if (bins[i] != kNone) continue;
        // far from zero: far from the row's largest too, or the row has no bins
        bins[i] = -kNone;
        if (!(((double)top - (double)get(p.tops + slot0 + i)) * per > 2 * kRing)) sh.listed = 1;
    }
    __syncthreads();
    if (top == -INFINITY) {
        give_first(s, r, ~0ull);
        return;
    }
    bool listed = has_bins(top, per) && !sh.listed;
    if (listed) {
        const int big = __builtin_amdgcn_readfirstlane(binned(top, per).bin);
        const int bin = big - (int)threadIdx.x;
        uint32_t count = 0;
        uint64_t rest = 0;
#pragma clang loop unroll(disable)
        for (uint32_t i = 0; i < p.parts; i += kBatch) {
            uint64_t v[kBatch];
            const uint64_t* ring = p.rings + (slot0 + i) * kRing + (bin & (kRing - 1));
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
                const bool has = i + j < p.parts && bins[i + j] - bin >= 0 &&
                                 bins[i + j] - bin < kRing;
                v[j] = has ? get(const_cast<uint64_t*>(ring) + (size_t)j * kRing) : 0;
            }
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
                count += (uint32_t)(v[j] >> kCount);
                rest += v[j] & ((1ull << kCount) - 1);
            }
        }
        make_plan(sh, rules, top, per, count, rest);
        const Plan plan = sh.plan;
        listed = plan.listed && plan.listed <= kList;
        if (listed) {
            const float low = (float)((big - last_needed(plan) - 1) / per);
            const int below = big - last_needed(plan);
#pragma clang loop unroll(disable)
            for (uint32_t i = 0; i < p.parts; i += kBatch) {
                uint32_t look = 0;
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    if (i + j >= p.parts || bins[i + j] < below) continue;
                    const int code = get(p.far + (slot0 + i + j) * kLanes + threadIdx.x);
                    look |= bins[i + j] - 4 * code >= below ? 1u << j : 0u;
                }
                while (look) {
                    const uint32_t at = i + __builtin_ctz(look);
                    look &= look - 1;
                    read_tile<DT>(row, begin_of(at), begin_of(at + 1), 0, x);
                    list_near(sh, plan, big, low, per, x, [&](int e) {
                        return index_in<DT>(row, begin_of(at), 0, e);
                    });
                }
            }
            __syncthreads();
            draw(sh, s, r, rules, per, sh.listed < kList ? sh.listed : kList);
        }
    }
    if (!listed) draw_slowly<DT>(sh.slow, s, r, rules, top);
}

template <int DT>
hipError_t launch(Device* d, hipStream_t st, const Sampling& s, int* status) {
    constexpr uint32_t E = Blocks<DT>::kEach;
    // a row's blocks, one of them for its start
    const uint32_t blocks = (s.width + E - 1) / E + 1;
    constexpr uint32_t kMost = kTile / E * kLanes;
    const uint32_t least = (blocks + kMost - 1) / kMost;
    if (least <= 1 || (least <= kTiles && s.rows >= (uint32_t)d->cu_count)) {
        // a grid's lanes are counted in 32 bits
        constexpr uint32_t kRows = 1u << 21;
        for (uint32_t first = 0; first < s.rows; first += kRows) {
            const uint32_t n = s.rows - first < kRows ? s.rows - first : kRows;
            hipLaunchKernelGGL(sample_whole_kernel<DT>, dim3(n), dim3(kLanes), 0, st, s, first);
        }
        return hipGetLastError();
    }
    uint32_t parts = 2 * (uint32_t)d->cu_count / s.rows;
    const uint32_t most = (blocks + kMost / 2 - 1) / (kMost / 2);
    parts = parts < most ? parts : most;
    parts = parts > least ? parts : least;
    Parts p{};
    p.blocks = (blocks + parts - 1) / parts;
    p.parts = (blocks + p.blocks - 1) / p.blocks;
    // launches of up to 64 MiB of rings, and of as many rows as there are tickets
    uint32_t rows = (64u << 20) / (p.parts * kRing * 8);
    constexpr uint32_t kTickets = kWorkspaceCounterBytes / 4;
    rows = rows < kTickets ? (rows ? rows : 1) : kTickets;
    rows = rows < s.rows ? rows : s.rows;
    const size_t slots = (size_t)rows * p.parts;
    char* ws = static_cast<char*>(
        workspace(d, st, slots * (kRing * 8 + 8 + 4 + kLanes), status));
    if (!ws) return hipSuccess;
    p.tickets = reinterpret_cast<uint32_t*>(ws);
    p.rings = reinterpret_cast<uint64_t*>(ws + kWorkspaceCounterBytes);
    p.least = p.rings + slots * kRing;
    p.tops = reinterpret_cast<float*>(p.least + slots);
    p.far = reinterpret_cast<uint8_t*>(p.tops + slots);
    for (uint32_t first = 0; first < s.rows; first += rows) {
        const uint32_t n = s.rows - first < rows ? s.rows - first : rows;
        p.first = first;
        hipLaunchKernelGGL(sample_parts_kernel<DT>, dim3(n * p.parts), dim3(kLanes), 0, st, s, p);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(Device* d, hipStream_t st, const Sampling& s, int* status) {
    *status = ACCEL_OK;
    return s.dtype == ACCEL_F32   ? launch<ACCEL_F32>(d, st, s, status)
           : s.dtype == ACCEL_F16 ? launch<ACCEL_F16>(d, st, s, status)
                                  : launch<ACCEL_BF16>(d, st, s, status);
}

}  // namespace accel
