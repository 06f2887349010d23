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
// Sums over bins then say in which bins the borders of k, p, m and u lie.  Where those
// hold up to 64 logits together, one more look gathers them, and a wave puts them in
// order and finds the borders.  Otherwise the borders are found one by one, each bin
// cut into 1024 by another histogram first if it holds more than 64.  Rows past what
// that serves (has_bins, kMostEach, kFew) go digit by digit of their keys, many passes of
// one workgroup: a row of 128000 near 60 below zero at a temperature of 0.005 in 960 us,
// 512 of them in 2000.
//
// Bins are absolute, not relative to the row's largest, so one pass is enough: a ring
// of 1024 bins (64 factors of two), set by the first logits seen.  Weights below 2^-46
// of the largest are left out.
//
// What bounds it: for many rows issue, 29 VALU instructions a logit and one atomic on
// LDS, of eight copies of a bin (512 rows of 128000 in f32 88 to 118 us, 262 MB at 2.2 to
// 3 TB/s; digit by digit of the keys, four looks a border, it was 1689).  A row's chain
// after its pass, some 20 us of barriers and a look, no other workgroup fills where all
// rows run at once.  For few rows that chain: one row of 128000 26 us, 64 of 100003 in
// bf16 48 to 53; nearly flat ones, with hundreds of logits in a border's bin and another
// look a border, 17 of 32001 in f16 51.  At a temperature of 0 only the largest is looked
// for: 512 rows of 128000 in 63 us (4.2 TB/s), one in 12.
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

constexpr int kLanes = 512, kWaves = kLanes / 64;
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
    constexpr int kPer = kBins / kLanes;      // digits a lane
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

constexpr int kRing = 1024;            // bins of the ring
constexpr int kPer = kRing / kLanes;   // consecutive ones a lane
constexpr int kCopies = 8;             // of each bin's word, for lanes that meet in it
constexpr int kReach = 736;            // bins below the largest's that count
constexpr int kFew = 64;               // logits that a wave puts in order

// A bin's word: 2^49 for each logit, and 2^38 (2^(r / 16) - kLeast).  Up to 30 2^10
// of them: their number is below 2^15 and the lower sum below 2^38 0.0434 30 2^10 < 2^49.
constexpr int kUnit = 38, kCount = 49;
constexpr double kLeast = 1002.0 / 1024;               // below 2^(-1 / 32)
constexpr uint64_t kLeastUnits = 1002ull << (kUnit - 10);
constexpr uint64_t kRest = (1ull << kCount) - 1;
constexpr uint32_t kMostEach = 30 << 10;

// 2^(r / 16), by the fifth power of its series: off by (ln 2 / 32)^6 / 720 = 2^-42.7 of
// it for |r| <= 1/2.  `one` is the series' first number.
__device__ __forceinline__ double sixteenth_of(double r, double one) {
    constexpr double z = 0.69314718055994530942 / 16;
    constexpr double c1 = z, c2 = z * z / 2, c3 = z * z * z / 6, c4 = z * z * z * z / 24,
                     c5 = z * z * z * z * z / 120;
    double q = __builtin_fma(c5, r, c4);
    q = __builtin_fma(q, r, c3);
    q = __builtin_fma(q, r, c2);
    q = __builtin_fma(q, r, c1);
    return __builtin_fma(q, r, one);
}
// A logit's bin, its place r in it and its part of the bin's word, rounded by 2^-39.
// Bins have to be the same wherever they are asked for, so no sum is fused here that is
// not written so.
struct Binned {
    int bin;
    double r;
    uint64_t word;
};
__device__ __forceinline__ Binned binned(float x, double per) {
#pragma clang fp contract(off)
    constexpr double kMagic = 6755399441055744.0;      // 3 * 2^51: the sum's low word is whole
    constexpr double kBase = 16384.0;                  // its last place is 2^-38
    const double e = (double)x * per;
    const double t = e + kMagic;
    const double r = e - (t - kMagic);
    const double q = sixteenth_of(r, kBase + (1 - kLeast));
    return {(int)(uint32_t)__builtin_bit_cast(uint64_t, t), r,
            __builtin_bit_cast(uint64_t, q) -
                (__builtin_bit_cast(uint64_t, kBase) - (1ull << kCount))};
}
// Bins a logit's unit: 16 log2(e) / T.
__device__ __forceinline__ double bins_per(const Rules& r) {
    return uniform(16 * 1.44269504088896340736 / r.temperature);
}
// A weight, or a sum of them, in units of 2^-38 of 2^(bin / 16), exact.
__device__ __forceinline__ uint64_t units(uint64_t count, uint64_t rest) {
    return count * kLeastUnits + rest;
}
__device__ __forceinline__ uint64_t units_of(const Binned& b) { return units(1, b.word & kRest); }
// 2^(-d / 16), to a few of its last places.
__device__ __forceinline__ double two_to(int d) {
    double t = d & 1 ? 0.9576032806985737 : 1.0;
    t *= d & 2 ? 0.9170040432046712 : 1.0;
    t *= d & 4 ? 0.8408964152537145 : 1.0;
    t *= d & 8 ? 0.7071067811865476 : 1.0;
    return __builtin_amdgcn_ldexp(t, -(d >> 4));
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
// Logits a lane reads at once; a tile is two such strips of all lanes.
constexpr int kStrip = 8;
template <int DT>
constexpr uint32_t kStripBlocks = kStrip / Blocks<DT>::kEach * kLanes;

// This lane's logits of strip t of the blocks [first, last).
template <int DT>
__device__ __forceinline__ void read_strip(const Blocks<DT>& row, uint32_t first, uint32_t last,
                                           uint32_t t, float (&x)[kStrip]) {
    constexpr int E = Blocks<DT>::kEach;
#pragma unroll
    for (int q = 0; q < kStrip / E; q++) {
        const uint32_t b = first + t * kStripBlocks<DT> + q * kLanes + threadIdx.x;
        if (b < last) row.read(b, x + q * E);
        else
#pragma unroll
            for (int e = 0; e < E; e++) x[q * E + e] = -INFINITY;
    }
}
// Those of strips t and t + 1.
template <int DT>
__device__ __forceinline__ void read_tile(const Blocks<DT>& row, uint32_t first, uint32_t last,
                                          uint32_t t, float (&x)[2 * kStrip]) {
    constexpr int E = Blocks<DT>::kEach;
#pragma unroll
    for (int q = 0; q < 2 * kStrip / E; q++) {
        const uint32_t b = first + t * kStripBlocks<DT> + q * kLanes + threadIdx.x;
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
    return (first + t * kStripBlocks<DT> + e / E * kLanes + threadIdx.x) * E + e % E - row.before;
}
__device__ __forceinline__ float largest(const float (&x)[kStrip]) {
    float m = fmaxf(x[0], x[1]);
#pragma unroll
    for (int e = 2; e < kStrip; e++) m = fmaxf(m, x[e]);
    return m;
}

constexpr uint32_t kHeld = 32;         // parts of a row whose distances are held
constexpr uint32_t kHold = 2560;       // logits of a bin held in LDS, at most
constexpr int kFirsts = 24;            // searches of a row: 7, and up to 4 a border
struct Scratch {
    union {
        uint64_t ring[kRing * kCopies + kCopies];      // the last: logits of no bin
        struct {
            double mass[kRing];        // the row's sum up to a bin's end, from the largest's
            uint32_t count[kRing];
            uint64_t fine[kRing];      // a bin's words, cut into 1024
            uint64_t list[kFew];
            uint8_t near[kRing];       // bins that a border may lie in
            uint8_t far[kHeld][kLanes];    // parts' lanes' distances
            uint64_t held[kHold];
        };
        RowScratch slow;
    };
    double wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float wave_top[kWaves];
    int first[kFirsts][kWaves];        // a search's each
    uint32_t listed, least, most, last;
    double kept, weight;               // what a wave found
    uint32_t kept_count, token;
};
__device__ __forceinline__ void clear_scratch(Scratch& sh) {
    uint4* p = reinterpret_cast<uint4*>(sh.ring);
#pragma unroll
    for (int i = 0; i < kRing * kCopies / 2 / kLanes; i++)
        p[i * kLanes + threadIdx.x] = make_uint4(0, 0, 0, 0);
}

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
    return fabs((double)top * per) < 0x1p17 && per > 0x1p-60 && per < 0x1p120;
}

// Adds a lane's logits that are in; the others' words go where nobody reads, without a
// branch a logit.
template <typename F>
__device__ __forceinline__ void add_to_ring(Scratch& sh, const float (&x)[kStrip], double per,
                                            F in) {
    uint64_t* mine = sh.ring + (threadIdx.x & (kCopies - 1));
#pragma unroll
    for (int e = 0; e < kStrip; e++) {
        const Binned b = binned(x[e], per);
        const int slot = in(x[e]) ? b.bin & (kRing - 1) : kRing;
        atomicAdd((unsigned long long*)(mine + slot * kCopies), (unsigned long long)b.word);
        // a few at a time: registers
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}
// A lane's bins: how many logits, and the rest of their weights.
struct Bins {
    uint32_t count[kPer];
    uint64_t rest[kPer];
};
// Those so many below top, from the ring: the copies' sums.
__device__ __forceinline__ Bins read_ring(const Scratch& sh, int top) {
    Bins b;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const int bin = top - (int)(threadIdx.x * kPer) - j;
        const uint64_t* p = &sh.ring[(bin & (kRing - 1)) * kCopies];
        b.count[j] = 0, b.rest[j] = 0;
#pragma unroll
        for (int i = 0; i < kCopies; i++) {
            b.count[j] += (uint32_t)(p[i] >> kCount);
            b.rest[j] += p[i] & kRest;
        }
    }
    return b;
}

// ---- the borders ----------------------------------------------------------------

// The first bin for which it holds, or `none`, N questions at once; all lanes call it,
// each time for another place of sh.first.  (A word a wave: an atomic minimum would be a
// loop over the lanes.)
template <int N>
__device__ __forceinline__ void first_bins(Scratch& sh, int& next, const bool (&is)[N][kPer],
                                           int none, int (&at)[N]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; i++) {
        int mine = kRing;
#pragma unroll
        for (int j = kPer - 1; j >= 0; j--) mine = is[i][j] ? (int)threadIdx.x * kPer + j : mine;
        const uint64_t b = __ballot(mine < kRing);
        const int first = __builtin_amdgcn_readlane(mine, b ? (int)__builtin_ctzll(b) : 0);
        if (lane == 0) sh.first[next + i][threadIdx.x >> 6] = first;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        int x = sh.first[next + i][lane & (kWaves - 1)];
#pragma unroll
        for (int d = kWaves / 2; d; d >>= 1) {
            const int o = __shfl_xor(x, d, 64);
            x = o < x ? o : x;
        }
        x = __builtin_amdgcn_readfirstlane(x);
        at[i] = x < none ? x : none;
    }
    next += N;
}

// Sums over bins up to and with each of this lane's.
struct Sums {
    double mass[kPer];
    uint32_t count[kPer];
};
__device__ __forceinline__ void sums_upto(Scratch& sh, Sums& x) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 1; j < kPer; j++) x.mass[j] += x.mass[j - 1], x.count[j] += x.count[j - 1];
    const double own = x.mass[kPer - 1];
    const uint32_t own_count = x.count[kPer - 1];
    double mass = own;
    uint32_t count = own_count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double m = __shfl_up(mass, d, 64);
        const uint32_t c = __shfl_up(count, d, 64);
        if (lane >= d) mass += m, count += c;
    }
    if (lane == 63) sh.wave_mass[wave] = mass, sh.wave_count[wave] = count;
    // the lanes before this one, not this sum less the lane's own: that would be rounded
    double before = __shfl_up(mass, 1, 64);
    uint32_t before_count = __shfl_up(count, 1, 64);
    if (lane == 0) before = 0, before_count = 0;
    __syncthreads();
    double waves = 0;
    uint32_t waves_count = 0;
#pragma unroll 1
    for (int w = 0; w < wave; w++) waves += sh.wave_mass[w], waves_count += sh.wave_count[w];
    before += waves, before_count += waves_count;
#pragma unroll
    for (int j = 0; j < kPer; j++) x.mass[j] += before, x.count[j] += before_count;
}

// Place in the order, ascending.
__device__ __forceinline__ uint64_t placed(float x, uint32_t index) {
    return (uint64_t)~key_of(x) << 32 | index;
}

// What a look over the row is for: bins lo .. hi below the largest's, of them (joint)
// those that are near a border; to cut them into 1024 (fine), or to list their logits,
// those of one of the 1024 where part is not -1; hold: and to hold them for the next.
struct Ask {
    int lo, hi, part;
    bool joint, fine, hold;
};
__device__ __forceinline__ int part_of(double r) {
    const int p = (int)((0.5 - r) * kRing);
    return p < 0 ? 0 : p < kRing ? p : kRing - 1;
}
// The logits between which those that are asked for lie.
struct Range {
    float low, high;
};
// The edges are rounded to a logit's type, by less than 2^-6 of a bin.
__device__ __forceinline__ Range range_of(const Ask& ask, int top, double per) {
    constexpr double kEdge = 1.0 / 64;
    double low = top - ask.hi - 0.5 - kEdge, high = top - ask.lo + 0.5 + kEdge;
    if (ask.part >= 0) {
        low = top - ask.lo + 0.5 - (ask.part + 1) * (1.0 / kRing) - kEdge;
        high = top - ask.lo + 0.5 - ask.part * (1.0 / kRing) + kEdge;
    }
    return {uniform((float)(low / per)), uniform((float)(high / per))};
}
__device__ __forceinline__ void answer_one(Scratch& sh, const Ask& ask, int top, double per,
                                           float v, uint32_t index) {
    const Binned b = binned(v, per);
    const int d = top - b.bin;
    if (d < ask.lo || d > ask.hi || (ask.joint && !sh.near[d])) return;
    const int part = part_of(b.r);
    if (ask.fine)
        atomicAdd((unsigned long long*)&sh.fine[part], (unsigned long long)b.word);
    if (ask.hold) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kHold) sh.held[at] = placed(v, index);
    }
    if (!ask.fine && (ask.part < 0 || part == ask.part)) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kFew) {
            sh.list[at] = placed(v, index);
        } else {
            atomicMin(&sh.least, key_of(v));
            atomicMax(&sh.most, key_of(v));
        }
    }
}
// A lane's logits x: those that are asked for.
template <typename F>
__device__ __forceinline__ void answer(Scratch& sh, const Ask& ask, int top, double per,
                                       const Range& range, const float (&x)[2 * kStrip], F index) {
    uint32_t some = 0;
#pragma unroll
    for (int e = 0; e < 2 * kStrip; e++)
        some |= x[e] >= range.low && x[e] <= range.high ? 1u << e : 0u;
    // one at a time, so that the code is there once
#pragma unroll 1
    while (some) {
        const int e = __builtin_ctz(some);
        some &= some - 1;
        float v = x[0];
#pragma unroll
        for (int i = 1; i < 2 * kStrip; i++) v = e == i ? x[i] : v;
        answer_one(sh, ask, top, per, v, index(e));
    }
}

// The same of those of 32 tiles that a lane's bits name, whose blocks [first, last)
// blocks_of(tile) gives.  A lane goes to the next that is its own.
template <int DT, typename F>
__device__ __forceinline__ void answer_tiles(Scratch& sh, const Ask& ask, int top, double per,
                                             const Range& range, const Blocks<DT>& row,
                                             uint32_t near, F blocks_of) {
#pragma unroll 1
    while (near) {
        const uint2 b = blocks_of(__builtin_ctz(near));
        near &= near - 1;
        float v[2 * kStrip];
        read_tile<DT>(row, b.x, b.y, 0, v);
        answer(sh, ask, top, per, range, v, [&](int e) { return index_in<DT>(row, b.x, 0, e); });
    }
}

// A wave's list in order, a lane a logit: its weight, its bin, and the sums up to it.
struct Listed {
    double weight, upto;
    uint32_t token, rank;              // rank: how many that is, itself among them
    int bin;
};
template <typename B>
__device__ __forceinline__ Listed in_order(Scratch& sh, uint32_t n, int top, double per,
                                           double one, B before) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t at = lane < n ? sh.list[lane] : ~0ull;
    uint32_t place = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < n; i++) {
        const uint64_t o =
            (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(at >> 32), i) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((uint32_t)at, i);
        place += o < at;
    }
    if (lane < n) sh.list[place] = at;
    // a lane reads what another has written
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (lane < n) at = sh.list[lane];
    const Binned b = binned(value_of(~(uint32_t)(at >> 32)), per);
    Listed l;
    l.token = (uint32_t)at;
    l.bin = lane < n ? top - b.bin : kRing;
    l.weight = lane < n ? (double)units_of(b) / one * two_to(l.bin) : 0.0;
    l.upto = l.weight;
    l.rank = 1;
#pragma unroll 1
    for (int x = 1; x < 64; x <<= 1) {
        const double m = __shfl_up(l.upto, x, 64);
        const uint32_t c = __shfl_up(l.rank, x, 64);
        const int o = __shfl_up(l.bin, x, 64);
        if ((int)lane >= x && o == l.bin) l.upto += m, l.rank += c;
    }
    before(l);
    return l;
}
__device__ __forceinline__ double lane_of(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(
        double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(b >> 32), lane) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((uint32_t)b, lane));
}

// What is left of a row: its sum and how many logits.
struct Left {
    double sum;
    uint32_t count;
};

// The token of a row, from each lane's bins, so many below the largest's.  look(ask) goes
// over the row's logits.  False where a border's bin holds too much.
template <int DT, typename L>
__device__ __forceinline__ bool finish(Scratch& sh, const Sampling& s, uint32_t row,
                                       const Rules& rules, double per, float top, const Bins& own,
                                       L look) {
    const int first = threadIdx.x * kPer;
    const bool leads = threadIdx.x == 0;
    const Binned big = binned(top, per);
    const int top_bin = __builtin_amdgcn_readfirstlane(big.bin);
    const uint64_t one_units = units_of(big);
    const double one = uniform((double)one_units);
    // units as weights, the largest's 1: whole ones and their rest, so that sums of
    // equal logits are whole
    const auto share = [&](uint64_t u) {
        const int q = (int)rint((double)u / one);
        return q + (double)((int64_t)u - (int64_t)q * (int64_t)one_units) / one;
    };
    Sums upto;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const bool some = first + j < kReach && own.count[j];
        upto.count[j] = some ? own.count[j] : 0u;
        upto.mass[j] = some ? share(units(own.count[j], own.rest[j])) * two_to(first + j) : 0.0;
    }
    // every lane has read the ring when its place is taken
    sums_upto(sh, upto);
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        sh.mass[first + j] = upto.mass[j];
        sh.count[first + j] = upto.count[j];
    }
    __syncthreads();
    const auto mass_before = [&](int b) { return b > 0 ? sh.mass[b - 1] : 0.0; };
    const auto count_before = [&](int b) { return b > 0 ? sh.count[b - 1] : 0u; };
    const double all = uniform(sh.mass[kRing - 1]);
    const uint32_t all_count = __builtin_amdgcn_readfirstlane(sh.count[kRing - 1]);
    // the least weight that a bin may hold, as a share of two_to
    const double edge = uniform(sixteenth_of(-0.5, 1.0) * sixteenth_of(-big.r, 1.0));
    const bool by_k = rules.top_k < all_count, by_p = rules.top_p < 1, by_m = rules.min_p > 0;
    int next = 0;
    const auto first_one = [&](auto holds, int none) {
        bool is[1][kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) is[0][j] = holds(j);
        int at[1];
        first_bins<1>(sh, next, is, none, at);
        return at[0];
    };
    struct Span {
        int lo, hi;
    };
    const auto first_two = [&](auto lo_holds, auto hi_holds, int none) {
        bool is[2][kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) is[0][j] = lo_holds(j), is[1][j] = hi_holds(j);
        int at[2];
        first_bins<2>(sh, next, is, none, at);
        return Span{at[0], at[1]};
    };

    // Where the borders may lie.  What one leaves of its bin is not known yet, so a sum
    // behind it is between two, and the next border's bin with it.
    Span k = {0, -1}, p = {0, -1}, m = {0, -1}, u;
    double lo = all, hi = all;
    u = first_two([&](int j) { return upto.count[j] >= rules.top_k; },
                  [&](int j) { return upto.count[j] >= all_count; }, kRing - 1);
    const int last = u.hi;              // the last that holds any
    int end = last;
    if (by_k) {
        end = u.lo;
        k = {end, end};
        lo = uniform(mass_before(end)), hi = uniform(sh.mass[end]);
    }
    if (by_p) {
        p = first_two([&](int j) { return upto.mass[j] >= rules.top_p * lo; },
                      [&](int j) { return upto.mass[j] >= rules.top_p * hi; }, end);
        lo = uniform(mass_before(p.lo)), hi = uniform(sh.mass[p.hi]);
        end = p.hi;
    }
    if (by_m) {
        const int at = first_one(
            [&](int j) { return two_to(first + j) * edge < rules.min_p; }, kRing);
        if (at <= end) {
            end = at;
            m = {end, end};
            lo = uniform(fmin(lo, mass_before(end))), hi = uniform(fmin(hi, sh.mass[end]));
        }
    }
    u = first_two([&](int j) { return upto.mass[j] > rules.u * lo; },
                  [&](int j) { return upto.mass[j] > rules.u * hi; }, end);
    const auto in = [](const Span& x, int b) { return b >= x.lo && b <= x.hi; };
    uint32_t planned = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const int b = first + j;
        const bool near = in(k, b) || in(p, b) || in(m, b) || in(u, b);
        sh.near[b] = near;
        planned += near ? sh.count[b] - count_before(b) : 0u;
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) planned += __shfl_xor(planned, x, 64);
    if ((threadIdx.x & 63) == 0) sh.wave_count[threadIdx.x >> 6] = planned;
    if (leads) sh.listed = 0, sh.least = ~0u, sh.most = 0;
    __syncthreads();
    planned = sh.wave_count[threadIdx.x & (kWaves - 1)];
#pragma unroll
    for (int x = kWaves / 2; x; x >>= 1) planned += __shfl_xor(planned, x, 64);
    Ask ask;
    ask.joint = (uint32_t)__builtin_amdgcn_readfirstlane(planned) <= kFew;
    ask.fine = ask.hold = false;
    ask.part = -1;
    ask.lo = 0;
    ask.hi = max(max(k.hi, p.hi), max(m.hi, u.hi));

    enum { kByK, kByP, kByM, kByU };
    Left left = {all, all_count};
    int stage = kByK;
    end = last;
    double base = 0;
    uint32_t base_count = 0;
    uint32_t held = 0;                 // logits of the border's bin that are in LDS
    for (;;) {
        const double border = uniform((stage == kByP ? rules.top_p : rules.u) * left.sum);
        // whether a sum, or the least weight there, is past the stage's border
        const auto past = [&](double mass, uint32_t count, double least) {
            return stage == kByK   ? count >= rules.top_k
                   : stage == kByP ? mass >= border
                   : stage == kByM ? least < rules.min_p
                                   : mass > border;
        };
        if (!ask.joint && ask.part < 0) {
            // the next border's bin
            if ((stage == kByK && !by_k) || (stage == kByP && !by_p) || (stage == kByM && !by_m)) {
                stage++;
                continue;
            }
            const int at = first_one(
                [&](int j) {
                    return past(sh.mass[first + j], sh.count[first + j], two_to(first + j) * edge);
                },
                stage == kByM ? kRing : end);
            if (stage == kByM && at > end) {
                stage++;
                continue;
            }
            ask.lo = ask.hi = at;
            base = uniform(mass_before(at));
            base_count = __builtin_amdgcn_readfirstlane(count_before(at));
            const uint32_t here = __builtin_amdgcn_readfirstlane(sh.count[at]) - base_count;
            if (here > kMostEach) return false;
            ask.fine = here > kFew;
            // a look that cuts a bin holds what it finds for the look that lists it (nearly
            // flat rows 56.3 -> 51.6 us; all that is near any border held by one look: 57.3)
            ask.hold = ask.fine && here <= kHold;
            held = ask.hold ? here : 0;
#pragma unroll
            for (int j = 0; j < kPer; j++) sh.fine[first + j] = 0;
            if (leads) sh.listed = 0, sh.least = ~0u, sh.most = 0;
            __syncthreads();
        }
        if (held && !ask.hold) {
#pragma unroll 1
            for (uint32_t i = threadIdx.x; i < held; i += kLanes) {
                const uint64_t x = sh.held[i];
                answer_one(sh, ask, top_bin, per, value_of(~(uint32_t)(x >> 32)), (uint32_t)x);
            }
        } else {
            look(ask);
        }
        __syncthreads();
        if (ask.fine) {
            // the 1024th that holds the border
            Sums x;
            uint32_t c[kPer];
            double w[kPer], least[kPer];
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                const uint64_t word = sh.fine[first + j];
                c[j] = x.count[j] = (uint32_t)(word >> kCount);
                w[j] = x.mass[j] =
                    c[j] ? share(units(c[j], word & kRest)) * two_to(ask.lo) : 0.0;
                least[j] = two_to(ask.lo) * sixteenth_of(-big.r, 1.0) *
                           sixteenth_of(0.5 - (first + j + 1) * (1.0 / kRing), 1.0);
            }
            sums_upto(sh, x);
#pragma unroll
            for (int j = 0; j < kPer; j++) x.mass[j] += base, x.count[j] += base_count;
            const uint32_t whole = __builtin_amdgcn_readfirstlane(sh.count[ask.lo]);
            const Span at = first_two(
                [&](int j) { return c[j] && past(x.mass[j], x.count[j], least[j]); },
                [&](int j) { return x.count[j] >= whole; }, kRing - 1);
            ask.part = at.lo < at.hi ? at.lo : at.hi;
#pragma unroll
            for (int j = 0; j < kPer; j++)
                if (first + j == ask.part) {
                    sh.kept = x.mass[j] - w[j], sh.kept_count = x.count[j] - c[j];
                    sh.listed = 0, sh.least = ~0u, sh.most = 0;
                }
            __syncthreads();
            base = uniform(sh.kept);
            base_count = __builtin_amdgcn_readfirstlane(sh.kept_count);
            ask.fine = ask.hold = false;
            continue;
        }
        const uint32_t n = __builtin_amdgcn_readfirstlane(sh.listed);
        if (ask.joint) {
            if (threadIdx.x < 64) {
                const Listed l = in_order(sh, n, top_bin, per, one, [&](Listed& x) {
                    const int b = x.bin < kRing ? x.bin : 0;
                    x.upto += mass_before(b);
                    x.rank += count_before(b);
                });
                const auto of = [&](const Span& x) { return l.bin >= x.lo && l.bin <= x.hi; };
                // the first listed logit of a span for which it holds, or the span's last
                const auto find = [&](const Span& x, bool is) {
                    const uint64_t some = __ballot(of(x)), hit = __ballot(of(x) && is);
                    return hit ? (int)__builtin_ctzll(hit)
                               : some ? 63 - (int)__builtin_clzll(some) : 0;
                };
                const auto cut = [&](int at) {
                    const uint32_t c = __builtin_amdgcn_readlane(l.rank, at);
                    if (c < left.count) left = {lane_of(l.upto, at), c};
                };
                if (by_k) cut(find(k, l.rank >= rules.top_k));
                if (by_p) cut(find(p, l.upto >= rules.top_p * left.sum));
                if (m.lo <= m.hi) {
                    // all of its bin that weigh as much, and all before it
                    const uint64_t ok = __ballot(of(m) && l.weight >= rules.min_p);
                    if (ok) cut(63 - (int)__builtin_clzll(ok));
                    else if (count_before(m.lo) < left.count)
                        left = {mass_before(m.lo), count_before(m.lo)};
                }
                int at = find(u, l.upto > rules.u * left.sum);
                // sums of bins and of their logits are rounded apart
                while (at && (uint32_t)__builtin_amdgcn_readlane(l.rank, at) > left.count) at--;
                if (leads) {
                    sh.token = __builtin_amdgcn_readlane(l.token, at);
                    sh.weight = lane_of(l.weight, at);
                    sh.kept = left.sum;
                }
            }
            break;
        }
        if (n <= kFew) {
            if (threadIdx.x < 64) {
                const Listed l = in_order(sh, n, top_bin, per, one, [&](Listed& x) {
                    x.upto += base;
                    x.rank += base_count;
                });
                const uint64_t hit = __ballot(
                    threadIdx.x < n && (past(l.upto, l.rank, l.weight) ||
                                        (stage == kByU && l.rank == left.count)));
                int at = hit ? (int)__builtin_ctzll(hit) : (int)n - 1;
                double upto = base;
                uint32_t rank = base_count;
                // the first that is too light goes with those behind it
                if (stage == kByM && hit) at--;
                if (at >= 0) upto = lane_of(l.upto, at), rank = __builtin_amdgcn_readlane(l.rank, at);
                if (leads) {
                    sh.kept = upto, sh.kept_count = rank;
                    sh.token = __builtin_amdgcn_readlane(l.token, at < 0 ? 0 : at);
                    sh.weight = lane_of(l.weight, at < 0 ? 0 : at);
                }
            }
        } else {
            // equal logits: so many of them
            const uint32_t most = __builtin_amdgcn_readfirstlane(sh.most);
            const bool odd = ~(uint32_t)(sh.list[threadIdx.x & (kFew - 1)] >> 32) != most;
            if (sh.least != most || first_one([&](int) { return odd; }, kRing) != kRing) return false;
            const Binned b = binned(value_of(most), per);
            const double w = (double)units_of(b) / one * two_to(top_bin - b.bin);
            uint32_t take = stage == kByK ? rules.top_k - base_count : 0;
            if (stage == kByP) take = (uint32_t)fmax(ceil((border - base) / w), 1.0);
            if (stage == kByM) take = w >= rules.min_p ? n : 0;
            if (stage == kByU) take = (uint32_t)fmax(floor((border - base) / w), 0.0) + 1;
            if (stage == kByU && base_count + take > left.count) take = left.count - base_count;
            if (take > n) take = n;
            __syncthreads();
            if (stage == kByU) {
                const void* at = static_cast<const char*>(s.logits) +
                                 (size_t)row * s.width * (DT == ACCEL_F32 ? 4 : 2);
                const uint32_t token = index_of<DT>(at, s.width, most, take ? take - 1 : 0, sh.slow);
                if (leads) sh.token = token;
            }
            if (leads) sh.kept = base + take * w, sh.kept_count = base_count + take, sh.weight = w;
        }
        if (stage == kByU) {
            if (leads) sh.kept = left.sum;
            break;
        }
        __syncthreads();
        const uint32_t c = __builtin_amdgcn_readfirstlane(sh.kept_count);
        if (c < left.count) {
            left = {uniform(sh.kept), c};
            end = ask.lo;
        }
        stage++;
        ask.part = -1;
        __syncthreads();
    }
    if (leads) {
        s.tokens[row] = sh.token;
        if (s.logprobs) s.logprobs[row] = (float)log(sh.weight / sh.kept);
    }
    return true;
}

// ---- the kernels ----------------------------------------------------------------

// A row that has no bins, or more than 64 logits of several values in a 1024th of one:
// borders digit by digit of the keys.
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
#pragma unroll 1
    for (int w = 1; w < kWaves; w++) v = sh.list[w] < v ? sh.list[w] : v;
    __syncthreads();
    return v;
}
template <int DT>
__device__ __forceinline__ uint64_t least_in(const Blocks<DT>& row, uint32_t first, uint32_t last) {
    float best = -INFINITY;
    uint32_t at = 0;
    for (uint32_t t = 0; t * kStripBlocks<DT> < last - first; t++) {
        float x[kStrip];
        read_strip<DT>(row, first, last, t, x);
        // a lane's logits are read in their order
#pragma unroll
        for (int e = 0; e < kStrip; e++)
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
// lane it is kept how far its largest logit is from the window's top, so a second look
// goes only to what may hold something near a border.
constexpr int kTiles = 30;             // what LDS holds beside another workgroup
constexpr int kTile = 2 * kStrip;
constexpr int kFar = 255;              // below the window; nearer ones are 253 at most
static_assert(kTiles * kTile * kLanes / kCopies <= kMostEach, "a word's count and sum");
static_assert(kTile * kLanes <= kMostEach, "the same, of a part's copies together");

template <int DT>
__global__ __launch_bounds__(kLanes, 4) void sample_whole_kernel(Sampling s, uint32_t first_row) {
    __shared__ Scratch sh;
    __shared__ uint8_t far[kTiles][kLanes];
    const uint32_t r = first_row + blockIdx.x;
    const Rules rules = rules_of(s, r);
    const Blocks<DT> row(s, r);
    if (rules.greedy) {
        give_first(s, r, least_of(sh, least_in<DT>(row, 0, row.count)));
        return;
    }
    const double per = bins_per(rules);
    float x[kStrip];
    read_strip<DT>(row, 0, row.count, 0, x);
    clear_scratch(sh);
    float most = largest(x), top = most;
    // the window is set by the first strip, with room for the rest to pass it by 2^16;
    // what passes it further is added afterwards
    const float first = top_of(sh, top);
    const bool bins = has_bins(first, per);
    Window w = {0, INFINITY, -INFINITY};
    if (bins) w.set(binned(first, per).bin + 256, per);
    const uint32_t strips = (row.count + kStripBlocks<DT> - 1) / kStripBlocks<DT>;
#pragma clang loop unroll(disable)
    for (uint32_t t = 0; t < strips; t++) {
        float ahead[kStrip];
        read_strip<DT>(row, 0, row.count, t + 1, ahead);
        if ((t & 1) || t + 1 == strips) {
            int code = kFar;
            if (most > w.high) code = 0;
            else if (most >= w.low) code = 1 + ((w.top - binned(most, per).bin) >> 2);
            far[t >> 1][threadIdx.x] = (uint8_t)code;
            most = -INFINITY;
        }
        add_to_ring(sh, x, per, [&](float v) { return v >= w.low && v <= w.high; });
#pragma unroll
        for (int e = 0; e < kStrip; e++) x[e] = ahead[e];
        const float m = largest(x);
        most = fmaxf(most, m);
        top = fmaxf(top, m);
    }
    top = top_of(sh, top);
    if (top == -INFINITY) {
        give_first(s, r, ~0ull);
        return;
    }
    bool done = has_bins(top, per);
    if (done) {
        const int bin = __builtin_amdgcn_readfirstlane(binned(top, per).bin);
        if (top > w.high) {
            const int past = bins ? bin - w.top : kRing;
            for (int i = threadIdx.x; i < past && i < kRing; i += kLanes) {
                uint64_t* p = &sh.ring[((bin - i) & (kRing - 1)) * kCopies];
#pragma unroll 1
                for (int c = 0; c < kCopies; c++) p[c] = 0;
            }
            __syncthreads();
            const float low = uniform((float)((bin - (kLow - 1)) / per));
#pragma clang loop unroll(disable)
            for (uint32_t t = 0; t < strips; t++) {
                if (far[t >> 1][threadIdx.x]) continue;
                read_strip<DT>(row, 0, row.count, t, x);
                add_to_ring(sh, x, per, [&](float v) { return v > w.high && v >= low; });
            }
            __syncthreads();
        }
        done = finish<DT>(sh, s, r, rules, per, top, read_ring(sh, bin), [&](const Ask& ask) {
            const int near = bins ? 1 + ((w.top - bin + ask.hi) >> 2) : 0;
            uint32_t tiles = 0;
#pragma unroll
            for (uint32_t t = 0; t < kTiles; t++) {
                const int code = 2 * t < strips ? far[t][threadIdx.x] : kFar;
                tiles |= !code || code <= near ? 1u << t : 0u;
            }
            answer_tiles<DT>(sh, ask, bin, per, range_of(ask, bin, per), row, tiles,
                             [&](uint32_t t) {
                                 return make_uint2(t * 2 * kStripBlocks<DT>, row.count);
                             });
        });
    }
    __syncthreads();
    if (!done) draw_slowly<DT>(sh.slow, s, r, rules, top);
}

// Longer rows, and too few rows to fill the chip: a workgroup a tile of a row.
// The last of a row's parts to end adds up their bins and goes on as above.
constexpr int kBatch = 8;             // parts whose words are asked for at once
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
__global__ __launch_bounds__(kLanes, 4) void sample_parts_kernel(Sampling s, Parts p) {
    __shared__ Scratch sh;
    // a row's parts' tops and their bins
    __shared__ union {
        float top;
        int bin;
    } parts[kMostParts];
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
    if (rules.greedy) {
        const uint64_t least = least_of(sh, least_in<DT>(row, begin, end));
        if (threadIdx.x == 0) put(p.least + slot, least);
    } else {
        float x[kStrip], y[kStrip];
        read_strip<DT>(row, begin, end, 0, x);
        read_strip<DT>(row, begin, end, 1, y);
        clear_scratch(sh);
        const float most = fmaxf(largest(x), largest(y));
        const float top = top_of(sh, most);
        if (threadIdx.x == 0) put(p.tops + slot, top);
        if (top > -INFINITY && has_bins(top, per)) {
            Window w;
            w.set(binned(top, per).bin, per);
            int code = kFar;
            if (most >= w.low) code = (w.top - binned(most, per).bin) >> 2;
            put(p.far + slot * kLanes + threadIdx.x, (uint8_t)code);
            const int strips = end - begin > kStripBlocks<DT> ? 2 : 1;
#pragma clang loop unroll(disable)
            for (int t = 0; t < strips; t++) {
                add_to_ring(sh, x, per, [&](float v) { return v >= w.low; });
#pragma unroll
                for (int e = 0; e < kStrip; e++) x[e] = y[e];
            }
            __syncthreads();
            const Bins b = read_ring(sh, w.top);
#pragma unroll
            for (int j = 0; j < kPer; j++)
                put(p.rings + slot * kRing +
                        ((w.top - (int)(threadIdx.x * kPer) - j) & (kRing - 1)),
                    (uint64_t)b.count[j] << kCount | b.rest[j]);
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
    // another workgroup's words come from far, 1.7 us, so they are asked for together
    constexpr int kNone = 1 << 30;
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < p.parts; i += kLanes) {
        const float t = get(p.tops + slot0 + i);
        top = fmaxf(top, t);
        parts[i].top = t;
    }
    top = top_of(sh, top);
    if (top == -INFINITY) {
        give_first(s, r, ~0ull);
        return;
    }
    for (uint32_t i = threadIdx.x; i < p.parts; i += kLanes) {
        const float t = parts[i].top;
        const bool some = t > -INFINITY, has = some && has_bins(t, per);
        parts[i].bin = has ? binned(t, per).bin : -kNone;
        // far from zero: far from the row's largest too, or the row has no bins
        if (some && !has && !(((double)top - (double)t) * per > 2 * kRing)) sh.listed = 1;
    }
    __syncthreads();
    bool done = has_bins(top, per) && !sh.listed;
    if (done) {
        const int big = __builtin_amdgcn_readfirstlane(binned(top, per).bin);
        Bins sum = {};
#pragma clang loop unroll(disable)
        for (uint32_t i = 0; i < p.parts; i += kBatch) {
            uint64_t v[kBatch][kPer];
            uint8_t code[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; x++)
                code[x] = get(p.far + (slot0 + (i + x < p.parts ? i + x : i)) * kLanes +
                              threadIdx.x);
#pragma unroll
            for (int x = 0; x < kBatch; x++)
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    // whatever a part holds, so that no load waits for another
                    const uint32_t at = i + x < p.parts ? i + x : i;
                    const int bin = big - (int)(threadIdx.x * kPer) - j;
                    v[x][j] = get(p.rings + (slot0 + at) * kRing + (bin & (kRing - 1)));
                }
            if (i < kHeld)
#pragma unroll
                for (int x = 0; x < kBatch; x++) sh.far[i + x][threadIdx.x] = code[x];
#pragma unroll
            for (int x = 0; x < kBatch; x++)
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const int bin = big - (int)(threadIdx.x * kPer) - j;
                    const int below = i + x < p.parts ? parts[i + x].bin - bin : -1;
                    const bool has = below >= 0 && below < kRing;
                    sum.count[j] += has ? (uint32_t)(v[x][j] >> kCount) : 0u;
                    sum.rest[j] += has ? v[x][j] & kRest : 0u;
                }
        }
        done = finish<DT>(sh, s, r, rules, per, top, sum, [&](const Ask& ask) {
            const int below = big - ask.hi;
            const Range range = range_of(ask, big, per);
#pragma clang loop unroll(disable)
            for (uint32_t i = 0; i < p.parts; i += 32) {
                uint32_t near = 0;
                for (uint32_t j = 0; j < 32 && i + j < p.parts; j += kBatch) {
                    uint8_t code[kBatch];
#pragma unroll
                    for (uint32_t x = 0; x < kBatch; x++) {
                        const uint32_t at = i + j + x < p.parts ? i + j + x : i;
                        code[x] = i < kHeld ? sh.far[at][threadIdx.x]
                                            : get(p.far + (slot0 + at) * kLanes + threadIdx.x);
                    }
#pragma unroll
                    for (uint32_t x = 0; x < kBatch; x++) {
                        const int b = i + j + x < p.parts ? parts[i + j + x].bin : -kNone;
                        near |= b - 4 * (int)code[x] >= below ? 1u << (j + x) : 0u;
                    }
                }
                answer_tiles<DT>(sh, ask, big, per, range, row, near, [&](uint32_t j) {
                    return make_uint2(begin_of(i + j), begin_of(i + j + 1));
                });
            }
        });
    }
    __syncthreads();
    if (!done) draw_slowly<DT>(sh.slow, s, r, rules, top);
}

template <int DT>
hipError_t launch(Device* d, hipStream_t st, const Sampling& s, int* status) {
    constexpr uint32_t E = Blocks<DT>::kEach;
    // a row's blocks, one of them for its start
    const uint32_t blocks = (s.width + E - 1) / E + 1;
    constexpr uint32_t kMost = kTile / E * kLanes;
    const uint32_t least = (blocks + kMost - 1) / kMost;
    // A row's workgroup takes 20 us and 1.45 a tile.  A workgroup a tile takes 24 to 27 us
    // whatever the width, as long as all run at once (rows of 16 tiles, us: one 43 whole
    // and 27 in parts, 16 46 and 32, 32 46 and 43, 64 48 and 71; of 8 tiles one 30 and 23;
    // of 4 one 24 and 24, 32 26 and 26).  Rows of more tiles than LDS has bytes for go in
    // parts however many they are (bf16: 300 of 262144 724 us, 300 of 245000 whole 125).
    if (least <= 4 ||
        (least <= kTiles && (uint64_t)s.rows * least > 2 * (uint32_t)d->cu_count)) {
        // a grid's lanes are counted in 32 bits
        constexpr uint32_t kRows = 1u << 22;
        for (uint32_t first = 0; first < s.rows; first += kRows) {
            const uint32_t n = s.rows - first < kRows ? s.rows - first : kRows;
            hipLaunchKernelGGL(sample_whole_kernel<DT>, dim3(n), dim3(kLanes), 0, st, s, first);
        }
        return hipGetLastError();
    }
    Parts p{};
    p.blocks = (blocks + least - 1) / least;
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
