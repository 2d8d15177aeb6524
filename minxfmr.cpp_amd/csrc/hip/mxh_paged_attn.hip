// mxh_paged_attn.hip — attention of packed tokens over a paged K/V cache on
// the fp16 matrix cores, in flash form (include/minxfmr_hip.h:
// mxh_attention_paged).
//
// Reference op: the attention of transformer.cpp:529-629 per token (scores
// q.k / sqrt(hd), softmax softmax.cpp:4-18, weighted sum of V rows), here over
// the rows of a sequence's pages, for drafted trees only along a token's path.
//
// Work: a tile is T = R / group consecutive tokens of one sequence with the
// group = nh / nkv q heads of one kv head (row r: token r / group, head
// r % group), R = 16, 32 or 64 rows; an item is a tile and a split of its keys,
// a workgroup an item and a kv head.  The lengths are on the device, so every
// workgroup computes the same plan from them (paged_item): stages of 128 keys
// per split so that the batch makes about `target` items.  The grid has room
// for the most items that can come of it; the others leave at once.
//
// K and V rows go straight into LDS (16 rows of a page are evenly spaced, so
// their addresses are a scalar base and fixed lane offsets).  Per 32-key block
// and set of 32 rows, as in mxh_prefill_attn.hip:
//
//   S^T = K Q^T      v_mfma_f32_32x32x16_f16; q pre-scaled by log2(e) /
//                    sqrt(hd), fp16 hi + lo; K exact
//   O^T += V^T P^T   P = 64 2^(S - ref) as fp16 hi + lo; V exact, its
//                    transposed operand read from the rows by
//                    ds_read_b64_tr_b16
//
// Tiles of 16 rows use v_mfma_f32_16x16x32_f16 instead: block b of a 32-key
// block's two 16-key products takes the keys 8 (m / 4) + 4 b + m % 4 as its rows
// m, so that lane l ends with the scores of keys 8 (l / 16) .. +8, the very
// operand that the second product wants of it.
//
// Rows that a token does not attend must not reach it: their scores are
// replaced, not added to, and since 0 times an infinity is no zero, blocks with
// unattended rows look their V values over; an item that meets an infinity or a
// NaN there is computed again without products over such rows (redo_item).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "mxh_attn.h"
#include "mxh_internal.h"
#include "mxh_paged.h"

namespace mxh {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kThreads = 256, kWaves = 4;
constexpr int kStage = 128;                // keys that splits are made of

// floats a wave leaves for the merge: V sums [m][hd + 4], references, sums
__host__ __device__ constexpr int merge_floats(int hd, int m) { return m * (hd + 6); }
__host__ __device__ constexpr int lds_bytes(int hd, int rows) {
    const int ring = 2 * kStage * hd * 2,  // R = 16: a stage, R = 64: two of half its keys
               merge = kWaves * merge_floats(hd, rows == 16 ? 16 : 32) * 4;
    return ring > merge ? ring : merge;
}

// what absent rows read
__device__ __align__(256) uint32_t zero_row[64];

// One workgroup's share of the batch (all uniform)
struct Item {
    int s, first, n, cached;          // sequence: its first token row, new tokens, rows before them
    int tile, split, splits, stages;  // stages per split
    int slot;                         // of its part (splits > 1)
};

struct SeqPlan {
    uint32_t first, n, cached, tiles, stages, splits;  // stages: of a split
};

// x / d rounded up, for x < 2^21 and inv the rounded 1 / d (off by less than
// half a step of x / d)
__device__ __forceinline__ uint32_t div_up(uint32_t x, uint32_t d, float inv) {
    return (uint32_t)(((float)(x + d - 1) + 0.5f) * inv);
}

// (t: tokens of a tile; in one split)
__device__ __forceinline__ SeqPlan seq_plan(int start, int end, int cached, const PagedArgs& a, uint32_t t, float inv_t) {
    SeqPlan p;
    p.first = (uint32_t)max(start, 0);
    p.n = (uint32_t)max(min(end, a.n_tokens) - (int)p.first, 0);
    if (a.parent) p.n = min(p.n, (uint32_t)kTreeMax);
    p.cached = (uint32_t)min(max(cached, 0), 1 << 30);
    p.tiles = div_up(p.n, t, inv_t);
    p.stages = (p.cached + p.n + kStage - 1) / kStage;
    p.splits = 1;
    return p;
}
__device__ __forceinline__ void split_plan(SeqPlan& p, uint32_t per) {  // of `per` stages at most
    if (p.stages <= per) return;
    const uint32_t all = p.stages, eq = (all + per - 1) / per;
    p.stages = (all + eq - 1) / eq;  // (evenly)
    p.splits = (all + p.stages - 1) / p.stages;
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
    v += dpp_i<0x111>(v);       // row_shr:1
    v += dpp_i<0x112>(v);
    v += dpp_i<0x114>(v);
    v += dpp_i<0x118>(v);
    v += dpp_i<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp_i<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}

// Item `index` of the batch; false past the last.  With MERGE the items are the
// tiles in splits.  target: items wanted, 0: no splits.  Lane l sums up the
// plans of the sequences [l part, (l + 1) part); the one that holds the index
// is walked.  With per >= W / target stages a split, W = sum of tiles * stages,
// a sequence in splits makes less than twice its W / per items, so the parts of
// all of them fit 2 target slots, and the tiles in splits are target at most.
template <bool MERGE>
__device__ __forceinline__ bool paged_item(const PagedArgs& a, uint32_t t, int target, uint32_t index, Item& it) {
    const int lane = threadIdx.x & 63, part = (a.n_seq + 63) / 64;
    const int s0 = lane * part, s1 = min(s0 + part, a.n_seq);
    const float inv_t = 1.0f / (float)t;
    SeqPlan p{0, 0, 0, 0, 0, 1};
    float w = 0.f;
    for (int s = s0; s < s1; ++s) {
        p = seq_plan(a.start[s], a.start[s + 1], a.cached[s], a, t, inv_t);
        w += (float)p.tiles * (float)p.stages;
    }
    // (at least W / target: the sum is off by some 2^-23 a step)
    const uint32_t per = target > 0 ? (uint32_t)fminf(wave_sum_all(w) / (float)target * 1.001f, 1e9f) + 1 : UINT32_MAX;
    const auto items_of = [](const SeqPlan& q) { return MERGE ? (q.splits > 1 ? q.tiles : 0) : q.tiles * q.splits; };
    const auto slots_of = [](const SeqPlan& q) { return q.splits > 1 ? q.tiles * q.splits : 0; };
    uint32_t items = 0, slots = 0;
    if (part == 1) {  // (one sequence a lane: its plan is still there)
        split_plan(p, per);
        items = items_of(p), slots = slots_of(p);
    } else {
        for (int s = s0; s < s1; ++s) {
            p = seq_plan(a.start[s], a.start[s + 1], a.cached[s], a, t, inv_t);
            split_plan(p, per);
            items += items_of(p), slots += slots_of(p);
        }
    }
    const uint32_t upto = (uint32_t)wave_scan((int)items), slots_upto = (uint32_t)wave_scan((int)slots);
    const uint64_t past = __ballot(upto > index);
    if (!past) return false;
    const int l = __ffsll((unsigned long long)past) - 1;
    const auto lane_l = [l](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    uint32_t i = index - lane_l(upto - items), slot = lane_l(slots_upto - slots);
    it.s = l * part;
    if (part == 1) {
        p = SeqPlan{lane_l(p.first), lane_l(p.n), lane_l(p.cached), lane_l(p.tiles), lane_l(p.stages), lane_l(p.splits)};
    } else {
        for (;; ++it.s) {  // (ends within the lane's sequences: they hold the index)
            p = seq_plan(a.start[it.s], a.start[it.s + 1], a.cached[it.s], a, t, inv_t);
            split_plan(p, per);
            if (i < items_of(p) || it.s + 1 >= min((l + 1) * part, a.n_seq)) break;
            i -= items_of(p), slot += slots_of(p);
        }
    }
    it.first = p.first, it.n = p.n, it.cached = p.cached, it.splits = p.splits, it.stages = p.stages;
    it.split = MERGE ? 0 : i / p.tiles;
    // (tiles with the most keys first)
    it.tile = MERGE ? i : p.tiles - 1 - (i - it.split * p.tiles);
    it.slot = slot + it.tile * p.splits + it.split;
    return true;
}

struct AttnPagedArgs {
    PagedArgs pg;
    const float* q;
    float* att;
    float* part;  // [2 target][nkv][R][HD]: V sums of the splits
    float2* ml;   // [2 target][nkv][R]: references and sums
    int nh, target;
    float qscale;
};

// pairs of 16-byte pieces of a V row are rotated by the key, so that the four
// keys of a transposing read lie in different banks (the same for keys 16 apart)
template <int HD>
__device__ __forceinline__ int v_swz(int key) {
    return HD == 128 ? 2 * (key & 7) : HD == 64 ? 2 * ((key >> 1) & 3) : 2 * ((key >> 2) & 1);
}

// 8 halves of V's transposed operand.  One read turns 4 keys x 16 dims around
// in each 16 lanes.  M = 32: keys 16 t + 8 (l / 32) + 0..7 of the block, dim
// 32 d + l % 32.  M = 16: keys 8 (l / 16) + 0..7 (t = 0), dim 16 d + l % 16.
template <int HD, int M>
struct VRead {
    uint32_t at;  // byte offset of t, d = 0 in the block's V rows
    __device__ __forceinline__ VRead() {
        const int lane = threadIdx.x & 63, key = 8 * (M == 32 ? lane >> 5 : lane >> 4) + ((lane & 15) >> 2);
        const int piece = (M == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
        at = (uint32_t)(key * HD * 2 + 16 * (piece ^ v_swz<HD>(key)) + 8 * (lane & 1));
    }
    // v0: the rows' place, a multiple of 256 bytes.  Dims M d on are 2 M d bytes
    // on; keys 4 on are 4 rows on, rotated by another HD bytes
    __device__ __forceinline__ f16x8 operator()(uint32_t v0, int t, int d) const {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const uint32_t p = (v0 + at) ^ (uint32_t)(2 * M * d);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(p + t * 32 * HD));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((p ^ HD) + t * 32 * HD + 8 * HD));
        return __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

// whether any V value of the block is infinite or NaN
template <int HD>
__device__ __forceinline__ bool any_special(uint32_t v0) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const u32x4 x = *(lds_u32x4*)(uintptr_t)(v0 + 1024 * i + 16 * (threadIdx.x & 63));
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (x[e] & 0x7c00u) == 0x7c00u || (x[e] & 0x7c000000u) == 0x7c000000u;
    }
    return __any(bad);
}

// The item again with a wave a row and no product that meets a value its row
// does not attend: a key a lane for the scores, then a dim a lane (or two) for
// the sums.  For items that found such a value among rows that only some of
// their tokens attend; the rest of the kernel pays no register for it.
template <int HD, int R>
__device__ void redo_item(const AttnPagedArgs& a, const Item& it, int g, int key0, int key1, uint8_t* smem) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = a.nh / a.pg.nkv, T = R / group, i0 = it.tile * T, rows = min(T, it.n - i0) * group;
    float* qs = reinterpret_cast<float*>(smem + wave * 2048);                  // the row's q
    float* ps = reinterpret_cast<float*>(smem + wave * 2048 + 512);            // 64 keys' probabilities
    int64_t* at = reinterpret_cast<int64_t*>(smem + wave * 2048 + 1024);       // and pool rows
    const uint64_t paths = a.pg.parent ? tree_path(tree_parent(a.pg, it.first, it.n)) : 0;
    const auto settle = [] {  // what the wave's lanes wrote is there for the others
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    };
    for (int r = wave; r < rows; r += kWaves) {
        const int i = i0 + r / group, hq = g * group + r % group, tok = it.first + i;
        const uint64_t path = path_of(paths, i & 63);
        const float* q = a.q + ((size_t)tok * a.nh + hq) * HD;
        for (int d = lane; d < HD; d += 64) qs[d] = q[d] * a.qscale;
        settle();
        float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
        const int end = min(key1, it.cached + i + 1);
        for (int k0 = key0; k0 < end; k0 += 64) {
            const int key = k0 + lane;
            bool on = key < end && (key < it.cached || !a.pg.parent || (path >> ((key - it.cached) & 63) & 1));
            const int64_t row = on ? paged_row(a.pg, it.s, key) : -1;
            on = row >= 0;
            float sc = -INFINITY;
            if (on) {
                const __half* k = a.pg.k + (row * a.pg.nkv + g) * HD;
                sc = 0.f;
                for (int d = 0; d < HD; ++d) sc = fmaf(qs[d], __half2float(k[d]), sc);
            }
            const float mx = fmaxf(m, wave_max(sc));
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
            const float p = on ? kPaScale * __builtin_amdgcn_exp2f(sc - (mx == -INFINITY ? 0.f : mx)) : 0.f;
            m = mx;
            l = l * alpha + wave_sum(p);
            ps[lane] = p;
            at[lane] = row;
            settle();
            o[0] *= alpha, o[1] *= alpha;
            for (int j = 0; j < 64; ++j) {
                if (at[j] < 0) continue;
                const __half* v = a.pg.v + (at[j] * a.pg.nkv + g) * HD;
                for (int u = 0; u < 2; ++u)
                    if (lane + 64 * u < HD) o[u] = fmaf(ps[j], __half2float(v[lane + 64 * u]), o[u]);
            }
            settle();
        }
        float* out = a.att + ((size_t)tok * a.nh + hq) * HD;
        float inv = l == 0.f ? 0.f : 1.0f / l;
        if (it.splits > 1) {
            const size_t p = ((size_t)it.slot * a.pg.nkv + g) * R + r;
            out = a.part + p * HD;
            inv = 1.f;
            if (lane == 0) a.ml[p] = make_float2(m, l);
        }
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < HD) out[lane + 64 * u] = o[u] * inv;
    }
}

// The keys a lane's row attends, a bit each, of the block of 32 at key kb.
struct RowMask {
    int cached, lim;  // the row's sequence's rows; its first key past (causal)
    uint64_t path;    // its path (drafted trees)
    bool tree;
    __device__ __forceinline__ uint32_t operator()(int kb) const {
        if (!tree) {
            const int left = lim - kb;
            return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
        }
        const int sh = kb - cached;
        return sh >= kTreeMax ? 0u
               : sh >= 0      ? (uint32_t)(path >> sh)
               : sh > -32     ? (uint32_t)(path << -sh) | ((1u << -sh) - 1u)
                              : ~0u;
    }
};

// a product of the matrix cores with M rows of the first operand and M columns
template <int M>
struct Mfma {
    typedef f32x16 acc;
    static __device__ __forceinline__ acc mul(f16x8 a, f16x8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mfma<16> {
    typedef f32x4 acc;
    static __device__ __forceinline__ acc mul(f16x8 a, f16x8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// the larger / the sum over the lanes that hold one row (l % M)
template <int M>
__device__ __forceinline__ float row_max(float v) {
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return pa_pair_max(v);
}
template <int M>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (M == 16) v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// R = 16: every wave takes 32 keys of a stage of 128 for all rows of the tile
// and reads only what it loaded: no barrier before the merge.  K and V have one
// place each; the next K comes while V is used, the next V while K is.
// R = 64: two waves, one a set of 32 rows, take the same 32 keys of a stage of
// 64, which all four waves load, a barrier a stage.  The scores run a stage
// ahead, so that a wave's products of the next scores and its vector work on
// these can overlap: at stage st there are V(st), K(st + 1), and on their way
// V(st + 1), K(st + 2).
template <int HD, int R>
__global__ __launch_bounds__(kThreads, 2) void attention_paged_kernel(AttnPagedArgs a) {
    constexpr int M = R == 16 ? 16 : 32, RS = R / M;  // rows of a wave; waves to a key group
    constexpr int KS = HD * M / 512, DB = HD / M;     // products of a score and of a sum
    constexpr int SB = 32 / M, NA = M * M / 64;       // score blocks of 32 keys, accumulators of one
    constexpr int NP = SB * NA, TT = NP / 8;          // a lane's scores; operands they make
    constexpr int NCH = HD / 8, KG = kWaves / RS, STAGE = 32 * KG;  // 16-byte pieces of a row; keys of a stage
    constexpr int GROUPS = STAGE / 16, OWN = GROUPS / kWaves;       // page groups of a stage; of them a wave loads
    constexpr int RPI = 64 / NCH, LPG = 16 / RPI;     // rows a load brings; loads of 16 rows (K or V)
    constexpr bool PRIVATE = RS == 1;
    // LDS: K places, then V places, of a stage each; q's rows before R = 64 needs the second ones
    constexpr int PLACE = STAGE * HD * 2, V0 = (PRIVATE ? 1 : 2) * PLACE;
    using MM = Mfma<M>;
    using acc_t = typename MM::acc;
    extern __shared__ __align__(256) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane % M, h = lane / M;
    const int set = wave % RS, kg = wave / RS;
    const uint32_t nkv = (uint32_t)a.pg.nkv, group = (uint32_t)a.nh / nkv, T = R / group;
    const uint32_t index = blockIdx.x / nkv, g = blockIdx.x - index * nkv;
    Item it;
    if (!paged_item<false>(a.pg, T, a.target, index, it)) return;

    const int i0 = it.tile * (int)T, ntok = min((int)T, it.n - i0);
    const int kend = it.cached + i0 + ntok;  // keys [0, kend) for the tile
    const int lim_min = a.pg.parent ? it.cached : it.cached + i0 + 1;  // every row attends the keys below
    const int key0 = kStage * it.stages * it.split;
    const int key1 = min(key0 + kStage * it.stages, kend);
    const int nst = max((key1 - key0 + STAGE - 1) / STAGE, 0);

    // this lane's query row
    const uint32_t row = 32 * set + n, tl = row / group;
    const bool valid = (int)tl < ntok;  // (the others: zeros at the tile's first token)
    const int i = i0 + (valid ? (int)tl : 0);
    const size_t qd = (size_t)a.nh * HD;
    const float* q0 = a.q + (size_t)(it.first + i0) * qd + g * group * HD;  // the tile's rows
    float4 qv[KS][2];
    if constexpr (PRIVATE) {  // (few rows: their loads go first, those of K and V come back after them)
        const float* qp = q0 + (i - i0) * qd + (row - tl * group) * HD + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                qv[ks][e] = valid ? *reinterpret_cast<const float4*>(qp + HD / KS * ks + 4 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int parent = a.pg.parent ? tree_parent(a.pg, it.first, it.n) : -1;

    // Where the stages' rows are: lane l holds the byte offset in the pool of
    // 16-row group l of a window of 64 groups (a page holds whole groups), the
    // high word negative where there is none, and that of the next window
    const uint32_t row_b = 2u * nkv * HD;
    const int* table = a.pg.table + (size_t)it.s * a.pg.table_ld;
    constexpr int WIN = 64 / GROUPS;  // stages of a window
    int2 win, win_next{0, -1};
    const auto window = [&](int w) __attribute__((always_inline)) {
        const int r = key0 + STAGE * WIN * w + 16 * lane, p = r >> a.pg.page_shift;
        int id = -1;
        if (r < kend && r >= 0 && p < a.pg.table_ld) id = table[p];
        const uint64_t row = ((uint64_t)(uint32_t)id << a.pg.page_shift) + (r & ((1 << a.pg.page_shift) - 1));
        const uint64_t off = (unsigned)id < (unsigned)a.pg.n_pages ? row * row_b : ~0ull;
        return make_int2((int)(uint32_t)off, (int)(uint32_t)(off >> 32));
    };
    win = window(0);
    if (nst > WIN) win_next = window(1);
    uint64_t gone_win = __ballot(win.y < 0);
    // the wave's groups of a stage, and which of all its groups are absent (a bit each)
    struct Place {
        int lo[OWN], hi[OWN];
        int r0;  // key of the first row
        uint32_t gone;
    };
    const auto look_up = [&](int st) __attribute__((always_inline)) {  // stages in their order
        if (st % WIN == 0 && st > 0) {
            win = win_next;
            gone_win = __ballot(win.y < 0);
            if (st + WIN < nst) win_next = window(st / WIN + 1);
        }
        Place p;
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            p.lo[u] = __builtin_amdgcn_readlane(win.x, (GROUPS * st + OWN * wave + u) & 63);
            p.hi[u] = __builtin_amdgcn_readlane(win.y, (GROUPS * st + OWN * wave + u) & 63);
        }
        p.r0 = key0 + STAGE * st + 16 * OWN * wave;
        p.gone = (uint32_t)(gone_win >> (GROUPS * st & 63)) & ((1u << GROUPS) - 1);
        return p;
    };
    const uint64_t kbase = scalar_addr(a.pg.k + g * HD), vbase = scalar_addr(a.pg.v + g * HD);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const auto k_place = [&](int st) { return lds0 + (PRIVATE ? 0 : (uint32_t)(st & 1) * PLACE); };
    const auto v_place = [&](int st) { return lds0 + V0 + (PRIVATE ? 0 : (uint32_t)(st & 1) * PLACE); };
    // lane offsets of the loads of 16 rows: row, and the row's piece that belongs
    // in the lane's place of the LDS row
    const uint32_t lr = (uint32_t)(lane / NCH);
    uint32_t koff[LPG], voff[LPG];
#pragma unroll
    for (int x = 0; x < LPG; ++x) {
        const uint32_t r = x * RPI + lr;
        koff[x] = r * row_b + 16 * (uint32_t)(lane % NCH ^ pa_swz<HD>((int)r));
        voff[x] = r * row_b + 16 * (uint32_t)(lane % NCH ^ v_swz<HD>((int)r));
    }
    // the wave's rows of a stage into K's or V's place
    const auto issue = [&](const Place& p, uint32_t place, bool is_v) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            const uint32_t to = place + 32 * (OWN * wave + u) * HD;
            const uint32_t(&off)[LPG] = is_v ? voff : koff;
            const uint64_t from = (is_v ? vbase : kbase) + (((uint64_t)(uint32_t)p.hi[u] << 32) | (uint32_t)p.lo[u]);
            if (p.hi[u] >= 0 && p.r0 + 16 * u + 15 < kend) {
#pragma unroll
                for (int x = 0; x < LPG; ++x) g2l_s(from, off[x], to + 1024 * x);
            } else {
                // rows past the last repeat it (their scores are replaced); an absent
                // group reads the row of zeros
                const bool none = p.hi[u] < 0;
                const uint32_t last = none ? 0 : (uint32_t)(kend - 1 - p.r0 - 16 * u);
                const uint64_t at = none ? scalar_addr(zero_row) : from;
#pragma unroll
                for (int x = 0; x < LPG; ++x) {
                    const uint32_t r = x * RPI + lr;
                    g2l_s(at, off[x] - (r - min(r, last)) * row_b, to + 1024 * x);
                }
            }
        }
    };
    Place ahead;  // of the next rows to come
    f16x8 qh[KS], ql[KS];
    uint32_t gone = 0, gone_next = 0;  // of the current stage, and of the next
    if (nst > 0) ahead = look_up(0), gone = ahead.gone;
    if constexpr (PRIVATE) {
        if (nst > 0) issue(ahead, k_place(0), false), issue(ahead, v_place(0), true);
    } else {
        // q's rows through LDS, in the places of K(1) and V(1), 16-byte pieces
        // rotated by the row (a lane reads its row, not its load's neighbour's)
        constexpr int QP = HD / 4, QR = 64 / QP;  // pieces of a row, rows a load brings
        const uint64_t from = scalar_addr(q0);
#pragma unroll
        for (int x = 0; x < R / QR / kWaves; ++x) {
            const uint32_t r0 = (uint32_t)(R / kWaves * wave + QR * x), r = r0 + lane / QP;
            const uint32_t t = min(r / group, (uint32_t)ntok - 1);
            const uint32_t off = 4 * (t * (uint32_t)qd + (r - r / group * group) * HD) + 16 * ((lane % QP) ^ (r & 7));
            const uint32_t at = r0 * 4 * HD;
            g2l_s(from, off, lds0 + (at < PLACE ? PLACE + at : V0 + at));
        }
        if (nst > 0) issue(ahead, k_place(0), false), issue(ahead, v_place(0), true);
        if (nst > 0) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LPG * OWN) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
        const uint32_t at = row * 4 * HD, q = lds0 + (at < PLACE ? PLACE + at : V0 + at);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const f32x4 x = *(lds_f32x4*)(uintptr_t)(q + 16 * ((4 * ks + 2 * h + e) ^ (row & 7)));
                qv[ks][e] = valid ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (nst > 1) {
            ahead = look_up(1), gone_next = ahead.gone;
            issue(ahead, k_place(1), false);
        }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const float v[8] = {qv[ks][0].x, qv[ks][0].y, qv[ks][0].z, qv[ks][0].w,
                            qv[ks][1].x, qv[ks][1].y, qv[ks][1].z, qv[ks][1].w};
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            f16x2 hi, lo;
            pa_split(v[e] * a.qscale, v[e + 1] * a.qscale, hi, lo);
            qh[ks][e] = hi[0], qh[ks][e + 1] = hi[1], ql[ks][e] = lo[0], ql[ks][e + 1] = lo[1];
        }
    }
    RowMask mask{it.cached, it.cached + i + 1, 0, a.pg.parent != nullptr};
    if (a.pg.parent) mask.path = path_of(tree_path(parent), i);

    bool redo = false;  // (uniform)
    float mref = -INFINITY, lrun = 0.f;
    acc_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < NA; ++v) o[d][v] = 0.f;
    const VRead<HD, M> vr;
    // this lane's first piece of its K row; the next products' are 1024 / M bytes on
    const int key_row = M == 32 ? pa_pi(n) : 8 * (n >> 2) + (n & 3);
    const uint32_t krow = (uint32_t)(key_row * HD * 2 + 16 * (h ^ pa_swz<HD>(key_row)));

    // scores of the wave's keys with K's rows at k0
    const auto score = [&](uint32_t k0, acc_t (&s)[SB]) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < SB; ++b) {
            typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
#pragma unroll
            for (int v = 0; v < NA; ++v) s[b][v] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                // (4 keys on: 4 rows on, rotated by another HD / 2 bytes)
                const uint32_t at = ((k0 + krow) ^ (uint32_t)(1024 / M * ks) ^ (uint32_t)(b * HD / 2)) + 8 * HD * b;
                const f16x8 k = *(lds_f16x8*)(uintptr_t)at;
                s[b] = MM::mul(k, qh[ks], s[b]);
                s[b] = MM::mul(k, ql[ks], s[b]);
            }
        }
    };
    // masks, and the reference moved where a score exceeds it by far
    const auto settle = [&](int kb, uint32_t v0, acc_t (&s)[SB], auto&& v_there) __attribute__((always_inline)) {
        if (kb + 32 > lim_min || gone) {
            uint32_t w = mask(kb);
            if (gone >> (2 * kg) & 1) w &= 0xffff0000u;
            if (gone >> (2 * kg) & 2) w &= 0xffffu;
            w >>= 8 * h;  // value v: key 8 h + 16 (v / 8) + v % 8
#pragma unroll
            for (int v = 0; v < NP; ++v)
                if (!((w >> (16 * (v >> 3) + (v & 7))) & 1)) s[v / NA][v % NA] = -INFINITY;
            v_there();
            redo |= any_special<HD>(v0);
        }
        float mx = s[0][0];
#pragma unroll
        for (int v = 1; v < NP; ++v) mx = fmaxf(mx, s[v / NA][v % NA]);
        mx = row_max<M>(mx);
        if (__any(mx > mref + kPaSlack)) {  // also the first block with an attended key
            const float mnew = fmaxf(mref, mx);
            // (nothing attended so far: the sums are zero)
            const float alpha = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - mnew);
            mref = mnew;
            lrun *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < NA; ++v) o[d][v] *= alpha;
        }
    };
    f16x8 bh[TT], bl[TT];
    const auto weigh = [&](const acc_t (&s)[SB]) __attribute__((always_inline)) {
        const float ref0 = mref == -INFINITY ? 0.f : mref;
        float p[NP], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NP; ++v) {
            p[v] = kPaScale * __builtin_amdgcn_exp2f(s[v / NA][v % NA] - ref0);
            ps[v & 3] += p[v];
        }
        lrun += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int u = 0; u < 8; u += 2) {
                f16x2 hi, lo;
                pa_split(p[8 * t + u], p[8 * t + u + 1], hi, lo);
                bh[t][u] = hi[0], bh[t][u + 1] = hi[1], bl[t][u] = lo[0], bl[t][u + 1] = lo[1];
            }
    };
    const auto sum = [&](uint32_t v0) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const f16x8 v = vr(v0, t, d);
                o[d] = MM::mul(v, bh[t], o[d]);
                o[d] = MM::mul(v, bl[t], o[d]);
            }
    };

    // R = 64: weigh, the next score and sum with the first two's work interleaved
    // as written (a product keeps the matrix cores busy for 32 cycles, in which a
    // wave can issue seven vector instructions; left to itself the scheduler puts
    // one behind the other)
    const auto weigh_and_score = [&](uint32_t k0, uint32_t v0, const acc_t (&s)[SB], acc_t (&next)[SB]) __attribute__((always_inline)) {
        if constexpr (!PRIVATE) {
            constexpr int VALS = NP / (2 * KS), AHEAD = KS < 3 ? KS : 3;  // scores of a product; operands on their way
            typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
            const float ref0 = mref == -INFINITY ? 0.f : mref;
            f16x8 kf[KS], vf[TT * DB];
            const auto k_read = [&](int ks) { kf[ks] = *(lds_f16x8*)(uintptr_t)((k0 + krow) ^ (uint32_t)(32 * ks)); };
#pragma unroll
            for (int ks = 0; ks < AHEAD; ++ks) k_read(ks);
#pragma unroll
            for (int v = 0; v < NA; ++v) next[0][v] = 0.f;
            float ps[4] = {0.f, 0.f, 0.f, 0.f};
            __builtin_amdgcn_sched_barrier(0);
            float p[NP];
            const auto halves = [&](int u) {  // of values u and u + 1
                f16x2 hi, lo;
                pa_split(p[u], p[u + 1], hi, lo);
                bh[u / 8][u % 8] = hi[0], bh[u / 8][u % 8 + 1] = hi[1];
                bl[u / 8][u % 8] = lo[0], bl[u / 8][u % 8 + 1] = lo[1];
            };
#pragma unroll
            for (int j = 0; j < 2 * KS; ++j) {
                const int ks = j / 2;
                next[0] = MM::mul(kf[ks], j & 1 ? ql[ks] : qh[ks], next[0]);
                if (j & 1) {
                    if (ks + AHEAD < KS) k_read(ks + AHEAD);
                    else if (ks + AHEAD - KS < TT * DB) vf[ks + AHEAD - KS] = vr(v0, (ks + AHEAD - KS) / DB, (ks + AHEAD - KS) % DB);
                }
#pragma unroll
                for (int u = VALS * j; u < VALS * (j + 1); ++u) {
                    p[u] = kPaScale * __builtin_amdgcn_exp2f(s[0][u] - ref0);
                    ps[u & 3] += p[u];
                    if (u & 1) halves(u - 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            lrun += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
            for (int y = 0; y < TT * DB; ++y) {
                o[y % DB] = MM::mul(vf[y], bh[y / DB], o[y % DB]);
                o[y % DB] = MM::mul(vf[y], bl[y / DB], o[y % DB]);
                if (y + AHEAD < TT * DB) vf[y + AHEAD] = vr(v0, (y + AHEAD) / DB, (y + AHEAD) % DB);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    if constexpr (PRIVATE) {
        for (int st = 0; st < nst; ++st) {
            const uint32_t k0 = k_place(st) + 64 * kg * HD, v0 = v_place(st) + 64 * kg * HD;
            const int kb = key0 + STAGE * st + 32 * kg;  // first key of this wave's block
            const auto v_there = [&] {  // (the next K's loads may be out)
                if (st + 1 < nst) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPG * OWN) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            };
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPG * OWN) : "memory");  // K, not yet V
            acc_t s[SB];
            score(k0, s);
            // K's rows have been read: the next ones may come
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (st + 1 < nst) {
                ahead = look_up(st + 1);
                issue(ahead, k_place(0), false);
            }
            if (kb < key1) {
                settle(kb, v0, s, v_there);
                weigh(s);
                v_there();
                sum(v0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (st + 1 < nst) issue(ahead, v_place(0), true), gone = ahead.gone;
        }
    } else {
        acc_t s[SB], next[SB];
        if (nst > 0) {
            // K(0) has landed for every wave (V(0) with it; K(1) may be out)
            if (nst > 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LPG * OWN) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            score(k_place(0) + 64 * kg * HD, s);
        }
        for (int st = 0; st < nst; ++st) {
            // V(st) and K(st + 1) have landed for every wave, and every wave is done
            // with V(st - 1) and K(st)
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (st + 1 < nst) issue(ahead, v_place(st + 1), true);
            if (st + 2 < nst) {
                ahead = look_up(st + 2);
                issue(ahead, k_place(st), false);
            }
            const int kb = key0 + STAGE * st + 32 * kg;  // first key of this wave's block
            const uint32_t v0 = v_place(st) + 64 * kg * HD;
            // (a block behind the last key has every score replaced)
            settle(kb, v0, s, [] {});
            // (past the last stage the scores of whatever lies there, unused)
            weigh_and_score(k_place(st + 1) + 64 * kg * HD, v0, s, next);
#pragma unroll
            for (int b = 0; b < SB; ++b) s[b] = next[b];
            gone = gone_next, gone_next = ahead.gone;
        }
    }

    // the waves' parts meet, where no load is to come any more
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (__syncthreads_or(redo)) {
        redo_item<HD, R>(a, it, (int)g, key0, key1, smem);
        return;
    }
    float* ms = reinterpret_cast<float*>(smem);
    {
        float* mb = ms + wave * merge_floats(HD, M);  // V sums [M rows][HD + 4], references, sums
        const float lsum = row_sum<M>(lrun);
        if (valid) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < NA; v += 4)
                    *reinterpret_cast<float4*>(mb + n * (HD + 4) + M * d + 2 * v + 4 * h) =
                        make_float4(o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]);
            if (h == 0) {
                mb[M * (HD + 4) + n] = mref;
                mb[M * (HD + 5) + n] = lsum;
            }
        }
    }
    __syncthreads();
    // a thread takes four dims of a row
    for (int u = tid; u < ntok * (int)group * (HD / 4); u += kThreads) {
        const int rr = u / (HD / 4), d = 4 * (u % (HD / 4)), rn = rr % M;
        const float* mb = ms + rr / M * merge_floats(HD, M);
        constexpr int NEXT = RS * merge_floats(HD, M);  // (the next key group's part)
        float wt[KG], mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int k = 0; k < KG; ++k) mm = fmaxf(mm, mb[k * NEXT + M * (HD + 4) + rn]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const float mk = mb[k * NEXT + M * (HD + 4) + rn];
            wt[k] = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - mm);  // (nothing attended there)
            ll += wt[k] * mb[k * NEXT + M * (HD + 5) + rn];
            const float4 v = *reinterpret_cast<const float4*>(mb + k * NEXT + rn * (HD + 4) + d);
            x.x += wt[k] * v.x, x.y += wt[k] * v.y, x.z += wt[k] * v.z, x.w += wt[k] * v.w;
        }
        if (it.splits > 1) {
            const size_t p = ((size_t)it.slot * nkv + g) * R + rr;
            if (d == 0) a.ml[p] = make_float2(mm, ll);
            *reinterpret_cast<float4*>(a.part + p * HD + d) = x;
        } else {
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;  // (no row exists: zeros)
            const int rt = rr / (int)group;
            *reinterpret_cast<float4*>(a.att + ((size_t)(it.first + i0 + rt) * a.nh + g * group + (rr - rt * (int)group)) * HD + d) =
                make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
}

// att from the splits' parts: a workgroup takes 16 rows of a tile and kv head,
// a thread four dims of a row, and where there are fewer rows every LANES-th
// split
constexpr int kMergeRows = 16, kMergeThreads = 512;
template <int HD, int R>
__global__ __launch_bounds__(kMergeThreads) void attention_paged_merge_kernel(AttnPagedArgs a) {
    constexpr int AHEAD = 8, RB = R / kMergeRows;
    __shared__ float4 acc[kMergeThreads];
    __shared__ float2 st[kMergeThreads];
    const int nkv = a.pg.nkv, group = a.nh / nkv, T = R / group;
    const uint32_t rb = blockIdx.x % RB, index = blockIdx.x / RB / (uint32_t)nkv, g = blockIdx.x / RB - index * nkv;
    Item it;
    if (!paged_item<true>(a.pg, T, a.target, index, it)) return;
    const int rows = min(min(T, it.n - it.tile * T) * group - (int)rb * kMergeRows, kMergeRows);
    if (rows <= 0) return;
    const int tid = threadIdx.x, per = rows * (HD / 4), lanes = kMergeThreads / per;
    const int z0 = tid / per, u = tid % per, d = 4 * (u % (HD / 4)), row = rb * kMergeRows + u / (HD / 4);
    float M = -INFINITY, L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto join = [&](float2 t, float4 v) __attribute__((always_inline)) {
        if (t.x == -INFINITY) return;  // (nothing attended there)
        const float m1 = fmaxf(M, t.x), a0 = __builtin_amdgcn_exp2f(M - m1), a1 = __builtin_amdgcn_exp2f(t.x - m1);
        M = m1;
        L = L * a0 + t.y * a1;
        s.x = s.x * a0 + v.x * a1, s.y = s.y * a0 + v.y * a1, s.z = s.z * a0 + v.z * a1, s.w = s.w * a0 + v.w * a1;
    };
    if (z0 < lanes)
        for (int z = z0; z < it.splits; z += lanes * AHEAD) {
            float2 t[AHEAD];
            float4 v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const size_t p = ((size_t)(it.slot + min(z + i * lanes, it.splits - 1)) * nkv + g) * R + row;
                t[i] = a.ml[p];
                v[i] = *reinterpret_cast<const float4*>(a.part + p * HD + d);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (z + i * lanes < it.splits) join(t[i], v[i]);
        }
    if (lanes > 1) {
        acc[tid] = s;
        st[tid] = make_float2(M, L);
        __syncthreads();
    }
    if (z0) return;
    for (int i = 1; i < lanes; ++i) join(st[tid + i * per], acc[tid + i * per]);
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const size_t tok = (size_t)it.first + it.tile * T + row / group;
    *reinterpret_cast<float4*>(a.att + (tok * a.nh + g * group + row % group) * HD + d) =
        make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
}

// What the host can choose without the lengths: rows of a tile by the average
// sequence, and the number of items that the splits aim at.
struct Shape {
    int rows, target;
    int64_t items;  // at most
};
Shape attention_shape(const PagedArgs& a, int nh, int hd) {
    Shape s;
    const int group = nh / a.nkv;
    const int64_t want = (int64_t)((a.n_tokens + a.n_seq - 1) / a.n_seq) * group;
    s.rows = want > 16 ? 64 : 16;
    const int64_t tiles = a.n_tokens / (s.rows / group) + a.n_seq;
    const int64_t stages = (((int64_t)a.table_ld << a.page_shift) + kStage - 1) / kStage;  // of a tile, at most
    const int resident = (hd == 128 ? 2 : hd == 64 ? 3 : 4) * device_cus();
    static const double mult = getenv("MXH_MULT") ? atof(getenv("MXH_MULT")) : 1.0;
    s.target = stages > 1 ? std::max(2, (int)(mult * resident / a.nkv)) : 0;
    s.items = std::min(s.target + tiles, tiles * stages);
    return s;
}

template <int HD, int R>
int launch(const AttnPagedArgs& a, const Shape& sh, hipStream_t st) {
    static bool attr_set = false;  // above 64 KiB of LDS needs the opt-in, once per kernel
    if (!attr_set && lds_bytes(HD, R) > 65536) {
        if (hipFuncSetAttribute((const void*)attention_paged_kernel<HD, R>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds_bytes(HD, R)) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const int64_t items = sh.items * a.pg.nkv, merges = (int64_t)sh.target * a.pg.nkv * (R / kMergeRows);
    if (items * kThreads > UINT32_MAX || merges * kMergeThreads > UINT32_MAX) return MXH_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((attention_paged_kernel<HD, R>), dim3((unsigned)items), dim3(kThreads), lds_bytes(HD, R), st, a);
    if (sh.target > 0)
        hipLaunchKernelGGL((attention_paged_merge_kernel<HD, R>), dim3((unsigned)merges), dim3(kMergeThreads), 0, st, a);
    return MXH_OK;
}

template <int HD>
int launch_hd(const AttnPagedArgs& a, const Shape& sh, hipStream_t st) {
    return sh.rows == 64 ? launch<HD, 64>(a, sh, st) : launch<HD, 16>(a, sh, st);
}

}  // namespace

size_t attention_paged_work_bytes(const PagedArgs& a, int nh, int hd) {
    const Shape s = attention_shape(a, nh, hd);
    return (size_t)2 * s.target * a.nkv * s.rows * (hd + 2) * sizeof(float);
}

int attention_paged_launch(const PagedArgs& a, const float* q, int nh, int hd, float* att, void* work, hipStream_t st) {
    const Shape s = attention_shape(a, nh, hd);
    float* part = static_cast<float*>(work);
    float2* ml = reinterpret_cast<float2*>(part + (size_t)2 * s.target * a.nkv * s.rows * hd);
    const AttnPagedArgs args{a, q, att, part, ml, nh, s.target, 1.4426950408889634f / sqrtf((float)hd)};
    return hd == 32 ? launch_hd<32>(args, s, st) : hd == 64 ? launch_hd<64>(args, s, st) : launch_hd<128>(args, s, st);
}

}  // namespace mxh
