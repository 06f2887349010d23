// Attention of prompts over the paged cache: the kernel, for the translation units
// that launch it.  Included into one anonymous namespace per translation unit.
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
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "attention.hpp"

namespace accel {
namespace {

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

// Drafts: an entry's rows are the nodes of a tree behind its sequence's context.  A
// node sees the context and, of the nodes, those on its path to its root; it stands
// for the position of its depth behind the context.  All rows see the same keys up
// to the context's end, so only the tiles past it look at the paths: a bit for each
// of up to kDraft nodes, made by a lane a node that walks up its parents in LDS, two
// dependent reads an ancestor (after 500, bf16, one chain of 64 nodes 30.7 us and a tree
// of two to four children a node 22.6, of 256 nodes 67 and 29).
constexpr int kDraft = ACCEL_DRAFT_NODES;
struct Paths {
    // words of a node's bits, and as many past them as a tile reads; an odd stride,
    // for a wave's rows to meet in different banks
    uint32_t bits[kRows][kDraft / 32 + 3];
    int depth[kRows];                 // -1: a parent on the path is not before its child
    uint32_t parent[kDraft];
};
struct NoPaths {};

// A draft's work: its tiles of rows, and the tiles of keys of each, the sinks' and
// those from its roots' windows' start to its last node (a tile of rows that ends
// before has fewer).  One whose rows are zeros is a tile of keys.
struct DraftWork {
    uint32_t tiles, steps;
};
// Sums of them.  They stay below kTooMany for offsets that ascend; where entries share
// rows they may not, and no step is taken then.
constexpr uint32_t kTooMany = 0xffffffffu;
__device__ __forceinline__ uint32_t more_steps(uint32_t x, uint32_t y) {
    return x + y < x ? kTooMany : x + y;
}
template <int KT>
__device__ __forceinline__ DraftWork work_of(const Attention& a, uint32_t len, uint32_t nodes,
                                             int tokens) {
    DraftWork w = {(nodes + tokens - 1) / tokens, 1};
    if (nodes <= len && nodes <= (uint32_t)kDraft) {
        const uint32_t root = len - nodes;
        const uint32_t lo = a.window && root + 1 > a.window ? root + 1 - a.window : 0;
        const uint32_t near = a.window ? (a.sinks < lo ? a.sinks : lo) : 0;
        const uint32_t sink_tiles = (near + KT - 1) / KT;
        const uint32_t start = lo / KT > sink_tiles ? lo / KT : sink_tiles;
        const uint32_t last = len ? (len - 1) / KT + 1 : 0;
        w.steps = sink_tiles + (last > start ? last - start : 0);
    }
    return w;
}
// Of the line of all drafts' steps, a tile of rows after the other: where step x lies.
struct DraftPlace {
    int entry;
    Held held;
    uint32_t tile;                    // of the entry's rows
    uint32_t first, past;             // its steps' places in the line
};
template <int KT>
__device__ __forceinline__ DraftPlace place_of(const Cut& k, const KvCache& c, const Attention& a,
                                               int tokens, uint32_t x) {
    DraftPlace p;
    uint32_t start;
    p.entry = find_entry(k, x, &start);
    p.held = entry_held(k, c, a, p.entry);
    const DraftWork w = work_of<KT>(a, p.held.len, rows_of(a, p.entry).count, tokens);
    p.tile = (x - start) / w.steps;
    p.first = start + p.tile * w.steps;
    p.past = p.first + w.steps;
    return p;
}
// A cut this near to a tile of rows' first or last step moves there: a piece of it costs
// its queries' way in and its part's way out, some two steps.
constexpr uint32_t kNearDraft = 2;
// Steps that are worth a workgroup and a join, measured with 1, 2, 3, 4 and 8: 9 drafts of
// 1 to 100 nodes seen through a window of 333, f16, 30.1, 25.1, 25.1, 31.2 and 49.2 us; 8
// nodes after 500, bf16, 17.6, 17.1, 18.5, 16.9 and 20.7.
template <bool F32>
constexpr uint32_t kLeastDraft = F32 ? 1 : 2;
template <int KT>
__device__ __forceinline__ uint32_t draft_cut(const Cut& k, const KvCache& c, const Attention& a,
                                              int tokens, uint64_t w) {
    if (w * k.chunk >= k.tiles) return k.tiles;
    const uint32_t x = (uint32_t)(w * k.chunk);
    const DraftPlace p = place_of<KT>(k, c, a, tokens, x);
    return x - p.first <= kNearDraft ? p.first : p.past - x <= kNearDraft ? p.past : x;
}

// Two parts of a row, each scaled to the larger maximum.  Rounded by itself each, so
// that it is the same whichever of the two is at hand and which comes from memory.
__device__ __forceinline__ float joined(float x, float fx, float y, float fy) {
#pragma clang fp contract(off)
    const float a = x * fx, b = y * fy;
    return a + b;
}

template <bool BF16, int QT, int PT, int DIM, bool FULL, int KT, typename Call>
__global__ __launch_bounds__(256, QT == 1 && DIM <= 128 ? 2 : 1) void paged_prefill_kernel(
    KvCache c, Call a, const uint32_t* sums, uint32_t fold, uint32_t splits, uint32_t place0,
    uint32_t* tickets, uint32_t ticket_stride, float* parts, uint32_t* fault) {
    constexpr int NS = DIM / 16;            // MFMA steps of a score
    constexpr int NC = DIM / 8;             // 16-byte chunks of a key
    constexpr int SUB = KT / 32;            // 32-key parts of a tile
    constexpr int DT = DIM / 32;            // 32-dim parts of a row of values
    constexpr int BLOCKS = KT / 8;          // eight keys lie in one page
    constexpr int KL = KT * NC / 256;       // chunks of K, and of V, a lane stages
    constexpr bool F32 = QT > 1;
    constexpr bool TREE = std::is_same<Call, Drafts>::value;
    __shared__ typename std::conditional<TREE, Paths, NoPaths>::type paths;
    __shared__ __attribute__((aligned(256))) char k_sh[2][KT * NC * 16];
    __shared__ __attribute__((aligned(256))) char v_sh[2][KT * NC * 16];
    // keys of a tile with values that are not finite: tile t's in place t % 3,
    // which is cleared two steps before it is read, a barrier before it is set
    __shared__ uint32_t odd_sh[3][2];
    __shared__ uint32_t again_sh;
    // dims past the head's: K's chunks there are no load's target and stay 0
    const auto clear_keys = [&] {
        for (int i = threadIdx.x; i < 2 * KT * NC; i += 256)
            reinterpret_cast<u32x4*>(k_sh)[i] = (u32x4){0, 0, 0, 0};
    };
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
    const uint32_t split = TREE ? 0 : blockIdx.x / places;
    const uint32_t place = place0 + blockIdx.x - split * places;
    // (drafts: a stretch of the head's line of steps)
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
        if constexpr (TREE) {
            if (lane < a.n)
                v *= work_of<KT>(a, cut.lane_held.len, rows_of(a, lane).count, tokens).steps;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d, 64);
            if (lane >= d) v = TREE ? more_steps(v, up) : v + up;
        }
        cut.lane_sum = v;
        cut.tiles = lane_value(v, 63);
    } else {
        cut.tiles = __builtin_amdgcn_readfirstlane(sums[a.n - 1]);
    }
    uint32_t tile = 0;
    uint32_t u = 0, u_end = 0;           // drafts: the stretch's steps, to go and past
    if constexpr (TREE) {
        if (cut.tiles == kTooMany) {
            if (blockIdx.x == 0 && threadIdx.x == 0) report(fault, kFaultDraft);
            return;
        }
        const uint32_t even = (uint32_t)(((uint64_t)cut.tiles + splits - 1) / splits);
        cut.chunk = even > kLeastDraft<F32> ? even : kLeastDraft<F32>;
        u = draft_cut<KT>(cut, c, a, tokens, order);
        u_end = draft_cut<KT>(cut, c, a, tokens, order + 1);
        if constexpr (!FULL) clear_keys();
    } else {
        if (order >= cut.tiles) return;
        tile = cut.tiles <= 2 * fold && order >= fold ? order - fold : cut.tiles - 1 - order;
    }
    // a tile of rows; drafts: those of the stretch, one after the other (no lane goes on
    // to the next before the others: there are barriers on the way)
    do {
    int entry;
    Held held;
    uint32_t tok0;
    DraftPlace at = {};
    uint32_t u_next = 0;
    if constexpr (TREE) {
        if (u >= u_end) return;
        at = place_of<KT>(cut, c, a, tokens, u);
        entry = at.entry;
        held = at.held;
        tok0 = at.tile * tokens;
        u_next = at.past < u_end ? at.past : u_end;
        // LDS is the last tile's until all waves are here
        __syncthreads();
    } else {
        uint32_t item;
        entry = find_entry(cut, tile, &item);
        tok0 = (tile - item) * tokens;
        held = sums ? held_by(c, a, entry, threadIdx.x ? nullptr : fault)
                    : entry_held(cut, c, a, entry);
    }
    const Rows rows = rows_of(a, entry);
    if (tok0 >= rows.count) {            // offsets that do not ascend
        if constexpr (TREE) {
            u = u_next;
            continue;
        } else {
            return;
        }
    }
    const uint32_t toks = rows.count - tok0 < (uint32_t)tokens ? rows.count - tok0 : tokens;
    // the position of the tile's first token, or of a draft's roots; below 0 it sees
    // nothing
    const int base = (int)held.len - (int)rows.count + (TREE ? 0 : (int)tok0);
    // the tile's first place past base
    const int at0 = TREE ? (int)tok0 : 0;
    const bool drafted = !TREE || (base > -1 && rows.count <= (uint32_t)kDraft);
    if constexpr (TREE) {
        if (!drafted && held.seq != kNoSequence && threadIdx.x == 0)
            report(fault, base > -1 ? kFaultDraft : kFaultKvPage);
    }
    const int window = a.window ? (int)a.window : 0x7fffffff;
    const int sinks = a.window ? (int)a.sinks : 0;

    // this lane's row
    const int r = wave * 32 + col;
    const int tok = r / per, g = r - tok * per;
    const bool real = tok < (int)toks && g < gs;
    const size_t qrow = ((size_t)(rows.first + tok0 + (real ? tok : 0)) * a.heads + head * group +
                         g0 + (real ? g : 0)) * dim;
    // the wave's first and last position, and the workgroup's
    const int tok_a = wave * 32 / per, tok_b = (wave * 32 + 31) / per;
    const bool busy = tok_a < (int)toks;
    const int p_first = base + (TREE ? 0 : tok_a);
    const int p_a = p_first > -1 ? p_first : -1;
    const int p_last = base + at0 + (tok_b < (int)toks ? tok_b : (int)toks - 1);
    const int p_b = p_last > -1 ? p_last : -1;
    // past the workgroup's last
    const int p_end = drafted ? base + at0 + (int)toks : 0;

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
    if (!TREE && (int)split >= held_shares) return;

    // this lane's row's position, or -1 where it sees nothing
    int p = real && base + tok > -1 ? base + tok : -1;
    bool lost = false;      // some row of the wave's is such a draft
    if constexpr (TREE) {
        const int nodes = drafted ? at0 + (int)toks : 0;
        for (int i = threadIdx.x; i < nodes; i += 256)
            paths.parent[i] = a.parents[rows.first + i];
        for (int i = threadIdx.x; i < kRows * (int)(sizeof paths.bits[0] / 4); i += 256)
            (&paths.bits[0][0])[i] = 0;
        __syncthreads();
        if ((int)threadIdx.x < kRows) {
            const int x = threadIdx.x;
            int depth = -1;
            if (drafted && x < (int)toks) {
                const auto up = [&](uint32_t t) { return paths.parent[t]; };
                uint32_t t = at0 + x;
                for (depth = 0; up(t) < t; depth++) t = up(t);
                if (up(t) != ACCEL_KV_NONE) depth = -1;
                // the node k steps up stands k positions before this one
                t = at0 + x;
                for (int k = 0; k <= depth; k++, t = up(t))
                    if (k < window || base + depth - k < sinks)
                        paths.bits[x][t >> 5] |= 1u << (t & 31);
                if (depth < 0) report(fault, kFaultDraft);
            }
            paths.depth[x] = depth;
        }
        __syncthreads();
        const int depth = paths.depth[tok];
        p = real && depth > -1 ? base + depth : -1;
        lost = __any(real && depth < 0);
    }
    int t_begin = (int)split * share;
    int t_end = t_begin + share < count ? t_begin + share : count;
    if constexpr (TREE) {
        t_begin = (int)(u - at.first);
        t_end = (int)(u_next - at.first) < count ? (int)(u_next - at.first) : count;
    }
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
        return pos + KT <= base + (TREE ? 0 : 1) &&
               (pos > p_end - 1 - window || pos + KT <= sinks);
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

    if constexpr (!FULL && !TREE) clear_keys();
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
                if constexpr (TREE) {
                    if (pos + KT > base || lost) {
                        // a bit a key: those before the context's end, then the path's
                        const int past = pos - base;
                        uint64_t seen = past >= 0 ? 0 : past > -64 ? (1ull << -past) - 1 : ~0ull;
                        if (p < 0) seen = 0;
                        if (past > -64) {
                            const uint32_t* w = paths.bits[tok] + (past > 0 ? past >> 5 : 0);
                            const uint64_t low = w[0] | (uint64_t)w[1] << 32;
                            const int by = past & 31;
                            seen |= past <= 0 ? low << -past
                                    : by      ? low >> by | (uint64_t)w[2] << (64 - by)
                                              : low;
                        }
                        seen >>= half * 8;
                        hide([&](int x) { return (seen >> x & 1) != 0; });
                    }
                } else {
                    if (pos + KT > p_a + 1) hide([&](int x) { return x <= until; });
                }
                if (!(pos > p_b - window || pos + KT <= sinks)) {
                    // the first place the row's window holds; none where it is all past
                    const int from = until < window ? -KT : until - window + 1;
                    // a draft's nodes have been looked at by their depths
                    const int nodes = TREE ? base - here : KT;
                    if (pos >= sinks) {
                        hide([&](int x) { return (x >= from) | (TREE && x >= nodes); });
                    } else {
                        const int kept = sinks - here;
                        hide([&](int x) {
                            return (x >= from) | (x < kept) | (TREE && x >= nodes);
                        });
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
                    bool ok = (x <= p) & ((x > p - window) | (x < sinks));
                    if constexpr (TREE) {
                        const int t = x - base;
                        if (t >= 0) ok = (paths.bits[tok][t >> 5] >> (t & 31) & 1) != 0;
                    }
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
    if constexpr (TREE) {
        // The pieces of a tile of rows, of stretches w0 to w1 (the first and the last cut
        // of it that are farther than kNearDraft from its ends), join in pairs, then the
        // pairs: of two the one to arrive last adds the other's part to its own, lane by
        // lane, and goes on as the pair's first.  Two places a stretch: a tile's first
        // piece, and the others'.
        u = u_next;
        const bool whole = t_begin == 0 && u_next == at.past;
        if (!whole) {
            constexpr int kWords = DT * 16 + 2;
            const uint32_t w0 = (uint32_t)(((uint64_t)at.first + kNearDraft) / cut.chunk);
            const uint32_t w1 =
                (uint32_t)(((uint64_t)at.past - kNearDraft + cut.chunk - 1) / cut.chunk) - 1;
            const uint32_t pieces = w1 - w0 + 1;
            const auto part = [&](uint32_t i) {
                return reinterpret_cast<uint64_t*>(parts) +
                       (2 * ((size_t)(w0 + i) * heads + head_tile) + (i == 0 ? 1 : 0)) *
                           (kWords / 2 * 256) + threadIdx.x;
            };
            uint32_t mine = order - w0;
            bool last_one = true;
            for (uint32_t span = 1; span < pieces; span *= 2) {
                const uint32_t left = mine & ~(2 * span - 1), right = left + span;
                if (right >= pieces) continue;
                uint64_t* to = part(mine);
                if (real) {
                    __hip_atomic_store(to, __builtin_bit_cast(uint64_t, (f32x2){m, sum}),
                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                    for (int e = 0; e < DT; e++)
#pragma unroll
                        for (int x = 0; x < 8; x++)
                            __hip_atomic_store(
                                to + (1 + e * 8 + x) * 256,
                                __builtin_bit_cast(uint64_t,
                                                   (f32x2){o[e][2 * x], o[e][2 * x + 1]}),
                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __builtin_amdgcn_s_waitcnt(0);
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __syncthreads();
                uint32_t* ticket = tickets + ((size_t)(w0 + right) * heads + head_tile) *
                                                 ticket_stride;
                if (threadIdx.x == 0) {
                    const uint32_t before = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED,
                                                                   __HIP_MEMORY_SCOPE_AGENT);
                    if (before) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
                    odd_sh[0][0] = before;
                }
                __syncthreads();
                last_one = __builtin_amdgcn_readfirstlane(odd_sh[0][0]) != 0;
                if (!last_one) break;
                uint64_t* from = part(mine == left ? right : left);
                if (real) {
                    const auto get = [&](int i) {
                        return __builtin_bit_cast(
                            f32x2, __hip_atomic_load(from + i * 256, __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT));
                    };
                    const f32x2 ml = get(0);
                    f32x2 v[DT * 8];
#pragma unroll
                    for (int i = 0; i < DT * 8; i++) v[i] = get(1 + i);
                    const float top = fmaxf(m, ml[0]);
                    const float own = kept<true>(__builtin_amdgcn_exp2f(m - top));
                    const float its = kept<true>(__builtin_amdgcn_exp2f(ml[0] - top));
                    m = top;
                    sum = joined(sum, own, ml[1], its);
#pragma unroll
                    for (int i = 0; i < DT * 8; i++)
#pragma unroll
                        for (int x = 0; x < 2; x++)
                            o[i >> 3][2 * (i & 7) + x] =
                                joined(o[i >> 3][2 * (i & 7) + x], own, v[i][x], its);
                }
                mine = left;
            }
            if (!last_one) continue;
        }
    } else if (held_shares > 1) {
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
    if (!TREE && !real) return;
    sum += __shfl_xor(sum, 32, 64);
    const float scale = sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < DT; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = e * 32 + 8 * i + 4 * half;
            if ((TREE && !real) || (!FULL && d >= dim)) continue;
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
    } while (TREE);
}

}  // namespace
}  // namespace accel
