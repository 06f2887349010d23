// A token of each row of logits, drawn from what its settings leave.
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
    r.temperature = t;
    const float p = s.top_p ? s.top_p[row] : 1.0f;
    r.top_p = p < 1 ? fmaxf(p, 0.0f) : 1.0f;
    const float m = s.min_p ? s.min_p[row] : 0.0f;
    r.min_p = m > 0 ? fminf(m, 1.0f) : 0.0f;
    const float u = s.u[row];
    r.u = u > 0 ? fminf(u, 1.0f - 0x1p-24f) : 0.0f;
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

template <int DT>
__global__ __launch_bounds__(kLanes) void sample_row_kernel(Sampling s) {
    __shared__ RowScratch sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
        const void* row = static_cast<const char*>(s.logits) +
                          (size_t)r * s.width * (DT == ACCEL_F32 ? 4 : 2);
        const Rules rules = rules_of(s, r);
        uint32_t top = 0;
        for (uint32_t i = threadIdx.x; i < s.width; i += kLanes) {
            const uint32_t key = key_of(logit<DT>(row, i));
            top = key > top ? key : top;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const uint32_t o = __shfl_xor(top, d, 64);
            top = o > top ? o : top;
        }
        __syncthreads();
        if (lane == 0) sh.wave_count[wave] = top;
        __syncthreads();
        for (int w = 0; w < kWaves; w++) top = sh.wave_count[w] > top ? sh.wave_count[w] : top;
        __syncthreads();
        if (top <= kNoKey) {
            if (threadIdx.x == 0) {
                s.tokens[r] = ACCEL_NO_TOKEN;
                if (s.logprobs) s.logprobs[r] = -INFINITY;
            }
            continue;
        }
        if (rules.greedy) {
            const uint32_t at = index_of<DT>(row, s.width, top, 0, sh);
            if (threadIdx.x == 0) {
                s.tokens[r] = at;
                if (s.logprobs) s.logprobs[r] = 0;
            }
            continue;
        }
        const Weigher weigh = {(double)value_of(top), rules.temperature,
                               (double)(1ull << (31 + __builtin_clz(s.width))),
                               value_of(top) == INFINITY};
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
    }
}

}  // namespace

hipError_t launch_sample(Device* d, hipStream_t st, const Sampling& s, int* status) {
    *status = ACCEL_OK;
    const dim3 grid(s.rows < (1u << 21) ? s.rows : 1u << 21);
    if (s.dtype == ACCEL_F32)
        hipLaunchKernelGGL(sample_row_kernel<ACCEL_F32>, grid, dim3(kLanes), 0, st, s);
    else if (s.dtype == ACCEL_F16)
        hipLaunchKernelGGL(sample_row_kernel<ACCEL_F16>, grid, dim3(kLanes), 0, st, s);
    else
        hipLaunchKernelGGL(sample_row_kernel<ACCEL_BF16>, grid, dim3(kLanes), 0, st, s);
    return hipGetLastError();
}

}  // namespace accel
