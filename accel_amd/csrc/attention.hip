// Attention over the paged cache: for the query at position p of a sequence,
//
//   out = sum_j e_j v_j / sum_j e_j,   e_j = exp(scale q.k_j - m),
//
// m the largest score, over the keys j <= p with p - j < window or j < sinks
// (all j <= p without a window).
//
// One workgroup a query row and head; the softmax's running maximum and sum
// are carried over blocks of 256 keys, so the keys are read once.
#include <hip/hip_runtime.h>

#include "internal.hpp"
#include "kvcache.hpp"

namespace accel {
namespace {

__device__ __forceinline__ float widen(uint16_t h, bool bf16) {
    if (bf16) return __uint_as_float((uint32_t)h << 16);
    _Float16 v;
    __builtin_memcpy(&v, &h, 2);
    return (float)v;
}

__global__ __launch_bounds__(256) void paged_attention_kernel(KvCache c, Attention a,
                                                              uint32_t* fault) {
    __shared__ float q[256], e[256], red[4];
    __shared__ uint32_t at[256];
    const int tid = threadIdx.x;
    const uint32_t row = blockIdx.x / a.heads, head = blockIdx.x - row * a.heads;
    int entry = (int)row;
    uint32_t left = 1;
    if (a.offsets) {
        entry = entry_of(a.offsets, a.n, row);
        if (entry < 0) return;
        left = a.offsets[entry + 1] - row;
    }
    const uint32_t s = sequence_of(c, a.seqs, entry, fault);
    const uint32_t len = s == kNoSequence ? 0 : length_of(c, s);
    // keys [0, sinks) and [lo, n)
    const uint32_t n = left <= len ? len - left + 1 : 0;
    const uint32_t lo = a.window && n > a.window ? n - a.window : 0;
    const uint32_t first = a.sinks < lo ? a.sinks : lo;
    const uint32_t seen = first + n - lo;
    const size_t qrow = ((size_t)row * a.heads + head) * c.dim;
    if (tid < c.dim)
        q[tid] = a.scale * (a.q_f32 ? static_cast<const float*>(a.q)[qrow + tid]
                                    : widen(static_cast<const uint16_t*>(a.q)[qrow + tid], c.bf16));
    const uint32_t kvh = head / (a.heads / c.heads);
    const size_t base = (size_t)a.layer * c.pages * c.page_elems();
    float m = -INFINITY, sum = 0, acc = 0;
    for (uint32_t k0 = 0; k0 < seen; k0 += 256) {
        const uint32_t k = k0 + tid;
        float score = -INFINITY;
        uint32_t page = ACCEL_KV_NONE, pos = 0;
        if (k < seen) {
            pos = k < first ? k : lo + (k - first);
            page = c.tables[(size_t)s * c.slots + (pos >> c.shift)];
            if (page >= c.pages) report(fault, kFaultKvPage);
        }
        __syncthreads();
        at[tid] = page < c.pages ? page : ACCEL_KV_NONE;
        if (page < c.pages) {
            const uint16_t* kr = c.keys + base +
                ((((size_t)page * c.heads + kvh) << c.shift) + (pos & ((1u << c.shift) - 1))) * c.dim;
            score = 0;
            for (int d = 0; d < c.dim; d++) score += q[d] * widen(kr[d], c.bf16);
        }
        float top = score;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
        const float keep = top == -INFINITY ? 0.f : expf(m - top);
        const float mine = page < c.pages ? expf(score - top) : 0.f;
        e[tid] = mine;
        float part = mine;
        for (int x = 32; x; x >>= 1) part += __shfl_xor(part, x, 64);
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = part;
        __syncthreads();
        sum = sum * keep + (red[0] + red[1] + red[2] + red[3]);
        acc *= keep;
        m = top;
        if (tid < c.dim) {
            const uint32_t end = seen - k0 < 256 ? seen - k0 : 256;
            for (uint32_t j = 0; j < end; j++) {
                if (at[j] == ACCEL_KV_NONE) continue;
                const uint32_t pj = k0 + j < first ? k0 + j : lo + (k0 + j - first);
                const uint16_t* vr = c.values + base +
                    ((((size_t)at[j] * c.heads + kvh) << c.shift) + (pj & ((1u << c.shift) - 1))) *
                        c.dim;
                acc += e[j] * widen(vr[tid], c.bf16);
            }
        }
    }
    if (tid < c.dim) {
        const float o = sum > 0 || sum != sum ? acc / sum : 0.f;
        if (a.q_f32) static_cast<float*>(a.out)[qrow + tid] = o;
        else if (c.bf16) static_cast<__bf16*>(a.out)[qrow + tid] = (__bf16)o;
        else static_cast<_Float16*>(a.out)[qrow + tid] = (_Float16)o;
    }
}

}  // namespace

hipError_t launch_paged_attention(Device* d, hipStream_t st, const KvCache& c,
                                  const Attention& a, int* status) {
    *status = ACCEL_OK;
    hipLaunchKernelGGL(paged_attention_kernel, dim3((unsigned)(a.rows * a.heads)), dim3(256), 0,
                       st, c, a, d->fault_dev);
    return hipGetLastError();
}

}  // namespace accel
