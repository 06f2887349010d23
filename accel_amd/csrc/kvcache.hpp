// Device helpers over the paged cache.  Included into one anonymous namespace
// per translation unit.
#pragma once

#include <hip/hip_runtime.h>

#include "internal.hpp"

namespace accel {
namespace {

__device__ __forceinline__ void report(uint32_t* fault, uint32_t bit) {
    __hip_atomic_fetch_or(fault, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Entry i's sequence: its index, or kNoSequence for a padded row and for an
// index outside the cache (reported where fault is not null).
constexpr uint32_t kNoSequence = ACCEL_KV_NONE;
__device__ __forceinline__ uint32_t sequence_of(const KvCache& c, const uint32_t* seqs, int i,
                                                uint32_t* fault) {
    const uint32_t s = seqs ? seqs[i] : (uint32_t)i;
    if (s < c.sequences) return s;
    if (s != ACCEL_KV_NONE && fault) report(fault, kFaultKvSequence);
    return kNoSequence;
}

// The positions a sequence holds, no more than its table has slots for.
__device__ __forceinline__ uint32_t length_of(const KvCache& c, uint32_t seq) {
    const uint32_t cap = c.slots << c.shift;
    const uint32_t n = c.lens[seq];
    return n < cap ? n : cap;
}

// A value of the cache's type.
__device__ __forceinline__ float widen(uint16_t h, bool bf16) {
    if (bf16) return __uint_as_float((uint32_t)h << 16);
    _Float16 v;
    __builtin_memcpy(&v, &h, 2);
    return (float)v;
}

// The entry of ascending offsets [n + 1] that row belongs to, or -1.
__device__ __forceinline__ int entry_of(const uint32_t* offsets, int n, uint32_t row) {
    int lo = 0, hi = n + 1;            // the first offset past row is in [lo, hi]
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);      // lo + hi may pass 31 bits
        if (offsets[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo > n ? -1 : lo - 1;
}

}  // namespace
}  // namespace accel
