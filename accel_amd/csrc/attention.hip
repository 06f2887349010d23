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

#include "attention.hpp"
#include "prompts.hpp"

namespace accel {
namespace {

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

// ---- one new token a sequence ---------------------------------------------------

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
            full ? go(paged_prefill_kernel<B, Q, P, 64, true, 64, Attention>)
                 : go(paged_prefill_kernel<B, Q, P, 64, false, 64, Attention>);
        else if (c.dim <= 128)
            full ? go(paged_prefill_kernel<B, Q, P, 128, true, 64, Attention>)
                 : go(paged_prefill_kernel<B, Q, P, 128, false, 64, Attention>);
        else
            full ? go(paged_prefill_kernel<B, Q, P, 256, true, 32, Attention>)
                 : go(paged_prefill_kernel<B, Q, P, 256, false, 32, Attention>);
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
