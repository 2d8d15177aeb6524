// mxh_paged_attn.hip — attention of packed tokens over a paged K/V cache on
// the fp16 matrix cores, in flash form (include/minxfmr_hip.h:
// mxh_attention_paged).
//
// Reference op: the attention of transformer.cpp:529-629 per token (scores
// q.k / sqrt(hd), softmax softmax.cpp:4-18, weighted sum of V rows), here over
// the rows of a sequence's pages, for drafted trees only along a token's path.
//
// Work: a tile is T = 32 RS / group consecutive tokens of one sequence with
// the group = nh / nkv q heads of one kv head (row r: token r / group, head
// r % group); an item is a tile and a split of its keys, a workgroup an item
// and a kv head.  The lengths are on the device, so every workgroup computes
// the same plan from them (paged_item): stages of 128 keys per split so that
// the batch makes about `target` items.  The grid has room for the most items
// that can come of it; the others leave at once.
//
// Inside a workgroup nothing is shared: wave w of four walks the 32-key blocks
// 4 st + w of its split, whose K and V rows it loads itself, straight into its
// own two LDS slots (a block's 16 rows of a page are contiguous, so the
// addresses are a scalar base a page and fixed lane offsets).  So there is no
// barrier before the end, where the waves' (reference, sum, V sum) meet in LDS.
// Per block and set of 32 rows, as in mxh_prefill_attn.hip:
//
//   S^T = K Q^T      v_mfma_f32_32x32x16_f16; q pre-scaled by log2(e) /
//                    sqrt(hd), fp16 hi + lo; K exact
//   O^T += V^T P^T   P = 64 2^(S - ref) as fp16 hi + lo; V exact, its
//                    transposed operand read from the rows by
//                    ds_read_b64_tr_b16
//
// Rows that a token does not attend must not reach it: their scores are
// replaced, not added to, and since 0 times an infinity is no zero, blocks with
// unattended rows look their V values over; an item that meets an infinity or a
// NaN there is computed again without products over such rows (redo_item).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mxh_attn.h"
#include "mxh_internal.h"
#include "mxh_paged.h"

namespace mxh {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kThreads = 256, kWaves = 4;
constexpr int kStage = 128;                // keys that splits are made of
constexpr int kSlots = 2;                  // stages in LDS

// floats a wave leaves for the merge: V sums [hd][32], references, sums
__host__ __device__ constexpr int merge_floats(int hd) { return hd * 32 + 64; }
__host__ __device__ constexpr int lds_bytes(int hd, int rs) {
    const int ring = kSlots * 2 * (kStage / rs) * hd * 2, merge = kWaves * merge_floats(hd) * 4;
    return ring > merge ? ring : merge;
}

// what absent rows read
__device__ __align__(256) uint32_t zero_row[64];

// One workgroup's share of the batch (all uniform)
struct Item {
    int s, first, n, cached;  // sequence: its first token row, new tokens, rows before them
    int tile, split, splits, stages;  // stages per split
    int slot;                 // of its part (splits > 1)
};

struct SeqPlan {
    int first, n, cached, tiles, stages, splits;
};

// tokens, tiles, and splits of `per` stages at most (0: one split) of sequence s
__device__ __forceinline__ SeqPlan seq_plan(const PagedArgs& a, int s, int T, int per) {
    SeqPlan p;
    p.first = max(a.start[s], 0);
    p.n = max(min(a.start[s + 1], a.n_tokens) - p.first, 0);
    if (a.parent) p.n = min(p.n, kTreeMax);
    p.cached = min(max(a.cached[s], 0), 1 << 30);
    p.tiles = (p.n + T - 1) / T;
    p.stages = (p.cached + p.n + kStage - 1) / kStage;
    p.splits = 1;
    if (per > 0 && p.stages > per) {
        const int eq = (p.stages + per - 1) / per;
        p.stages = (p.stages + eq - 1) / eq;  // (evenly)
        p.splits = ((p.cached + p.n + kStage - 1) / kStage + p.stages - 1) / p.stages;
    }
    return p;
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

// Item `index` of the batch (of its tiles alone with TILES); false past the
// last.  target: items wanted, 0: no splits.  Lane l sums up the plans of the
// sequences [l part, (l + 1) part); the one that holds the index is walked.
// With per = ceil(W / target) stages a split, W = sum of tiles * stages, a
// sequence in splits makes less than twice W_s / per items, so the parts of
// all of them fit 2 target slots.
template <bool TILES>
__device__ bool paged_item(const PagedArgs& a, int T, int target, int index, Item& it) {
    const int lane = threadIdx.x & 63, part = (a.n_seq + 63) / 64;
    const int s0 = lane * part, s1 = min(s0 + part, a.n_seq);
    int per = 0;
    if (target > 0) {
        double w = 0.0;
        for (int s = s0; s < s1; ++s) {
            const SeqPlan p = seq_plan(a, s, T, 0);
            w += (double)p.tiles * p.stages;
        }
        per = (int)fmin(ceil(wave_sum_d_all(w) / target), 1e9);
    }
    int items = 0, slots = 0;
    for (int s = s0; s < s1; ++s) {
        const SeqPlan p = seq_plan(a, s, T, per);
        items += p.tiles * (TILES ? 1 : p.splits);
        slots += p.splits > 1 ? p.tiles * p.splits : 0;
    }
    const int upto = wave_scan(items), slots_upto = wave_scan(slots);
    const uint64_t past = __ballot(upto > index);
    if (!past) return false;
    const int l = __ffsll((unsigned long long)past) - 1;
    int at = __builtin_amdgcn_readlane(upto - items, l), slot = __builtin_amdgcn_readlane(slots_upto - slots, l);
    for (int s = l * part;; ++s) {
        const SeqPlan p = seq_plan(a, s, T, per);
        const int here = p.tiles * (TILES ? 1 : p.splits);
        if (index < at + here || s + 1 >= min((l + 1) * part, a.n_seq)) {
            const int i = index - at;
            it.s = s, it.first = p.first, it.n = p.n, it.cached = p.cached;
            // (tiles with the most keys first)
            it.tile = TILES ? i : p.tiles - 1 - i % p.tiles;
            it.split = TILES ? 0 : i / p.tiles;
            it.splits = p.splits, it.stages = p.stages;
            it.slot = slot + it.tile * p.splits + it.split;
            return index < at + here;
        }
        at += here;
        slot += p.splits > 1 ? p.tiles * p.splits : 0;
    }
}

struct AttnPagedArgs {
    PagedArgs pg;
    const float* q;
    float* att;
    float* part;  // [2 target][nkv][32 RS][HD]: V sums of the splits
    float2* ml;   // [2 target][nkv][32 RS]: references and sums
    int nh, target;
    float qscale;
};

// 8 halves of V's transposed operand: keys 16 t + 8 h + 0..7 of the block (h:
// the lane's upper half), dim 32 d + lane % 32.  One read turns 4 keys x 16
// dims around in each 16 lanes.
template <int HD>
struct VRead {
    uint32_t at;  // byte offset of t, d = 0 in the block's V rows
    __device__ __forceinline__ VRead() {
        const int lane = threadIdx.x & 63, key = 8 * (lane >> 5) + ((lane & 15) >> 2);
        const int piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        at = (uint32_t)(key * HD * 2 + 16 * (piece ^ v_swz(key)) + 8 * (lane & 1));
    }
    // pairs of 16-byte pieces rotated by the key, so that the four keys of a
    // read lie in different banks (the same for keys 16 apart)
    static __device__ __forceinline__ int v_swz(int key) {
        return HD == 128 ? 2 * (key & 7) : HD == 64 ? 2 * ((key >> 1) & 3) : 2 * ((key >> 2) & 1);
    }
    // v0: the rows' place, a multiple of 256 bytes.  Dims 32 d on are 64 d bytes
    // on; keys 4 on are 4 rows on, rotated by another HD bytes
    __device__ __forceinline__ f16x8 operator()(uint32_t v0, int t, int d) const {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const uint32_t p = v0 + at;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((p ^ (64 * d)) + t * 32 * HD));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4*)(uintptr_t)(((p ^ (64 * d)) ^ HD) + t * 32 * HD + 8 * HD));
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
template <int HD, int RS>
__device__ void redo_item(const AttnPagedArgs& a, const Item& it, int g, int key0, int key1, uint8_t* smem) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = a.nh / a.pg.nkv, T = 32 * RS / group, i0 = it.tile * T, rows = min(T, it.n - i0) * group;
    float* qs = reinterpret_cast<float*>(smem + wave * 2048);                  // the row's q
    float* ps = reinterpret_cast<float*>(smem + wave * 2048 + 512);            // 64 keys' probabilities
    int64_t* at = reinterpret_cast<int64_t*>(smem + wave * 2048 + 1024);       // and pool rows
    const uint64_t paths = a.pg.parent ? tree_path(a.pg, it.first, it.n) : 0;
    const auto settle = [] {  // what the wave's lanes wrote is there for the others
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    };
    for (int r = wave; r < rows; r += kWaves) {
        const int i = i0 + r / group, hq = g * group + r % group, tok = it.first + i;
        const uint64_t path = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(paths >> 32), i & 63) << 32) |
                              (uint32_t)__shfl((int)(uint32_t)paths, i & 63);
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
            const size_t p = ((size_t)it.slot * a.pg.nkv + g) * (32 * RS) + r;
            out = a.part + p * HD;
            inv = 1.f;
            if (lane == 0) a.ml[p] = make_float2(m, l);
        }
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < HD) out[lane + 64 * u] = o[u] * inv;
    }
}

// The keys a lane's row of a block attends, bit 16 t + u for key 16 t + 8 h + u
// of the block at key kb (h: the lane's upper half).
struct RowMask {
    int cached, lim;  // the row's sequence's rows; its first key past (causal)
    uint64_t path;    // its path (drafted trees)
    bool tree;
    __device__ __forceinline__ uint32_t operator()(int kb, int h) const {
        uint32_t w;
        if (tree) {
            const int sh = kb - cached;
            w = sh >= kTreeMax ? 0u
                : sh >= 0      ? (uint32_t)(path >> sh)
                : sh > -32     ? (uint32_t)(path << -sh) | ((1u << -sh) - 1u)
                               : ~0u;
        } else {
            const int left = lim - kb;
            w = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
        }
        return w >> (8 * h);
    }
};

// KG key groups: waves that take the same 32 keys of a stage share the rows
// RS sets: 32-row sets, each a wave of every key group
template <int HD, int RS>
__global__ __launch_bounds__(kThreads, HD == 128 && RS == 1 ? 1 : 2) void attention_paged_kernel(AttnPagedArgs a) {
    constexpr int KS = HD / 16, DB = HD / 32, NCH = HD / 8;
    constexpr int KG = kWaves / RS, STAGE = 32 * KG;  // keys of a stage
    constexpr int GROUPS = STAGE / 16;     // page groups of a stage
    constexpr int OWN = GROUPS / kWaves;   // of them a wave loads
    constexpr int RPI = 64 / NCH;          // rows a load instruction brings
    constexpr int LPG = 16 / RPI;          // load instructions per 16 rows (K or V)
    constexpr int SLOT = 2 * STAGE * HD * 2;
    constexpr bool PRIVATE = RS == 1;      // a wave reads the rows it loaded itself
    extern __shared__ __align__(256) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int set = RS == 1 ? 0 : wave % RS, kg = wave / RS;
    const int nkv = a.pg.nkv, group = a.nh / nkv, T = 32 * RS / group;
    const int g = blockIdx.x % nkv;
    Item it;
    if (!paged_item<false>(a.pg, T, a.target, blockIdx.x / nkv, it)) return;

    const int i0 = it.tile * T, ntok = min(T, it.n - i0);
    const int kend = it.cached + i0 + ntok;  // keys [0, kend) for the tile
    const int lim_min = a.pg.parent ? it.cached : it.cached + i0 + 1;  // every row attends the keys below
    const int key0 = kStage * it.stages * it.split;
    const int key1 = min(key0 + kStage * it.stages, kend);
    const int nst = max((key1 - key0 + STAGE - 1) / STAGE, 0);

    // Lane l holds the page of 16-row group l of a window of 64 groups
    const uint32_t row_b = 2u * (uint32_t)(nkv * HD), page_b = row_b << a.pg.page_shift;
    const int* table = a.pg.table + (size_t)it.s * a.pg.table_ld;
    constexpr int WIN = 64 / GROUPS;  // stages of a window
    const auto page_ids = [&](int st) __attribute__((always_inline)) {
        const int row = key0 + STAGE * st + 16 * lane, p = row >> a.pg.page_shift;
        int id = -1;
        if (row < kend && row >= 0 && p < a.pg.table_ld) id = table[p];
        return (unsigned)id < (unsigned)a.pg.n_pages ? id : -1;
    };
    // (absent groups of the current stage's window, and of the one issued from)
    int ids = page_ids(0), ids_next = ids;
    uint64_t gone_win = __ballot(ids < 0), gone_next = gone_win;
    constexpr int AHEAD = PRIVATE ? 2 : 1;  // stages from a slot's issue to its use
    const auto turn_window = [&](int st) __attribute__((always_inline)) {  // before st + AHEAD is issued
        if (st % WIN == 0 && st > 0) gone_win = gone_next;
        if ((st + AHEAD) % WIN == 0) ids = ids_next, gone_next = __ballot(ids < 0);
        if (st % WIN == 0 && st + WIN < nst) ids_next = page_ids(st + WIN);
    };
    const uint64_t kbase = scalar_addr(a.pg.k + g * HD), vbase = scalar_addr(a.pg.v + g * HD);
    const uint64_t zero = scalar_addr(zero_row);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const int lr = lane / NCH;
    uint32_t kx = 16 * (uint32_t)(lane % NCH ^ pa_swz<HD>(lr)), vx = 16 * (uint32_t)(lane % NCH ^ VRead<HD>::v_swz(lr));
    // the wave's groups of stage st (16 rows of a page each)
    const auto issue = [&](int st) __attribute__((always_inline)) {
        const uint32_t slot = lds0 + (uint32_t)(st % kSlots) * SLOT;
        asm volatile("" : "+v"(kx), "+v"(vx));  // (else every offset below is kept in registers)
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            const int gr = OWN * wave + u, row = key0 + STAGE * st + 16 * gr;
            const int id = __builtin_amdgcn_readlane(ids, (GROUPS * st + gr) & 63);
            const uint32_t in = (uint32_t)(row & ((1 << a.pg.page_shift) - 1)) * row_b;
            const uint64_t off = (uint64_t)(uint32_t)id * page_b + in;
            const uint64_t kb = id < 0 ? zero : kbase + off, vb = id < 0 ? zero : vbase + off;
            // rows past the last repeat it (their scores are replaced); an absent
            // group reads the row of zeros
            const int last = id < 0 ? 0 : kend - 1 - row;
#pragma unroll
            for (int x = 0; x < LPG; ++x) {
                // (the rotation of row x RPI + lr is that of row lr and a constant)
                const uint32_t ro = __umul24((uint32_t)min(x * RPI + lr, last), row_b);
                const uint32_t to = slot + (uint32_t)(16 * gr + x * RPI) * (2 * HD);
                g2l_s(kb, ro + (kx ^ (64 * x)), to);
                g2l_s(vb, ro + (HD == 128 ? vx ^ (128 * (x & 1)) : vx), to + STAGE * HD * 2);
            }
        }
    };
    if (nst > 0) issue(0);
    if (PRIVATE && nst > 1) issue(1);

    // this lane's query row, split, and what it attends
    f16x8 qh[KS], ql[KS];
    RowMask mask;
    {
        const int row = 32 * set + n, tl = row / group, hh = row % group;
        const bool valid = tl < ntok;  // (the others: zeros at the tile's first token)
        const int i = i0 + (valid ? tl : 0);
        mask = RowMask{it.cached, it.cached + i + 1, 0, a.pg.parent != nullptr};
        if (a.pg.parent) {
            const uint64_t paths = tree_path(a.pg, it.first, it.n);
            mask.path = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(paths >> 32), i) << 32) |
                        (uint32_t)__shfl((int)(uint32_t)paths, i);
        }
        const float* qp = a.q + ((size_t)(it.first + i) * a.nh + g * group + hh) * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (valid) {
                const float4 x = *reinterpret_cast<const float4*>(qp + 16 * ks + 8 * h);
                const float4 y = *reinterpret_cast<const float4*>(qp + 16 * ks + 8 * h + 4);
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                f16x2 hi, lo;
                pa_split(v[e] * a.qscale, v[e + 1] * a.qscale, hi, lo);
                qh[ks][e] = hi[0], qh[ks][e + 1] = hi[1], ql[ks][e] = lo[0], ql[ks][e + 1] = lo[1];
            }
        }
    }

    bool redo = false;  // (uniform)
    float mref = -INFINITY, lrun = 0.f;
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
    const VRead<HD> vr;
    // this lane's piece 0 of its K row (every second piece from there: XOR 32 ks)
    const uint32_t krow = (uint32_t)(pa_pi(n) * HD * 2 + 16 * (h ^ pa_swz<HD>(pa_pi(n))));

    for (int st = 0; st < nst; ++st) {
        if constexpr (PRIVATE) {
            if (st + 1 < nst) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LPG * OWN) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
            // this stage has landed for every wave, and every wave is done with the
            // slot that the next one goes to
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        turn_window(st);
        if (!PRIVATE && st + 1 < nst) issue(st + 1);
        const int kb = key0 + STAGE * st + 32 * kg;  // first key of this wave's block
        if (kb < key1) {
            const uint32_t k0 = lds0 + (uint32_t)(st % kSlots) * SLOT + 32 * kg * HD * 2, v0 = k0 + STAGE * HD * 2;
            f32x16 s;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
                const f16x8 k = *(lds_f16x8*)(uintptr_t)((k0 + krow) ^ (32 * ks));
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[ks], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[ks], s, 0, 0, 0);
            }
            const uint32_t gone = (uint32_t)(gone_win >> (GROUPS * (st % WIN) + 2 * kg)) & 3;
            if (kb + 32 > lim_min || gone) {
                uint32_t w = mask(kb, h);
                if (gone & 1) w &= 0xffff0000u;
                if (gone & 2) w &= 0xffffu;
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (!((w >> (16 * (v >> 3) + (v & 7))) & 1)) s[v] = -INFINITY;
                redo |= any_special<HD>(v0);
            }
            float mx = s[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) mx = fmaxf(mx, s[v]);
            mx = pa_pair_max(mx);
            if (__any(mx > mref + kPaSlack)) {  // also the first block with an attended key
                const float mnew = fmaxf(mref, mx);
                // (nothing attended so far: the sums are zero)
                const float alpha = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - mnew);
                mref = mnew;
                lrun *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
            }
            const float ref0 = mref == -INFINITY ? 0.f : mref;
            float p[16], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                p[v] = kPaScale * __builtin_amdgcn_exp2f(s[v] - ref0);
                ps[v & 3] += p[v];
            }
            lrun += (ps[0] + ps[1]) + (ps[2] + ps[3]);
            f16x8 bh[2], bl[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int u = 0; u < 8; u += 2) {
                    f16x2 hi, lo;
                    pa_split(p[8 * t + u], p[8 * t + u + 1], hi, lo);
                    bh[t][u] = hi[0], bh[t][u + 1] = hi[1], bl[t][u] = lo[0], bl[t][u + 1] = lo[1];
                }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 v = vr(v0, t, d);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, bh[t], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, bl[t], o[d], 0, 0, 0);
                }
        }
        if constexpr (PRIVATE) {
            // the slot's last reads are done before its next rows are requested
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (st + 2 < nst) issue(st + 2);
        }
    }

    // the waves' parts meet (every load into the slots has been waited for)
    if (__syncthreads_or(redo)) {
        redo_item<HD, RS>(a, it, g, key0, key1, smem);
        return;
    }
    float* ms = reinterpret_cast<float*>(smem);
    {
        float* mb = ms + wave * merge_floats(HD);
        const float lsum = lrun + __shfl_xor(lrun, 32, 64);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) mb[(32 * d + 8 * (v >> 2) + 4 * h + (v & 3)) * 32 + n] = o[d][v];
        if (h == 0) {
            mb[HD * 32 + n] = mref;
            mb[HD * 32 + 32 + n] = lsum;
        }
    }
    __syncthreads();
    // thread: row 32 mr + mn, dims d0 .. d0 + ND
    constexpr int ND = HD * RS / 8;
    const int mr = RS == 2 ? (tid >> 5) & 1 : 0, mn = tid & 31, d0 = (tid >> (RS == 2 ? 6 : 5)) * ND;
    const float* mb[KG];
    float wt[KG], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < KG; ++i) {
        mb[i] = ms + (i * RS + mr) * merge_floats(HD);
        M = fmaxf(M, mb[i][HD * 32 + mn]);
    }
#pragma unroll
    for (int i = 0; i < KG; ++i) {
        const float mi = mb[i][HD * 32 + mn];
        wt[i] = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - M);  // (nothing attended there)
        L += wt[i] * mb[i][HD * 32 + 32 + mn];
    }
    const int row = 32 * mr + mn, tl = row / group;
    if (tl >= ntok) return;
    float* op;
    float inv = 1.f;
    if (it.splits > 1) {
        const size_t p = ((size_t)it.slot * nkv + g) * (32 * RS) + row;
        op = a.part + p * HD;
        if (d0 == 0) a.ml[p] = make_float2(M, L);
    } else {
        op = a.att + ((size_t)(it.first + i0 + tl) * a.nh + g * group + row % group) * HD;
        inv = L == 0.f ? 0.f : 1.0f / L;  // (no row exists: zeros)
    }
#pragma unroll
    for (int d = 0; d < ND; d += 4) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = 0.f;
#pragma unroll
            for (int i = 0; i < KG; ++i) x[e] += wt[i] * mb[i][(d0 + d + e) * 32 + mn];
        }
        *reinterpret_cast<float4*>(op + d0 + d) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
}

// att from the splits' parts: a workgroup takes 4 rows of one tile and kv
// head, a thread four dims of a row and every (256 / HD)-th... split
constexpr int kMergeRows = 4, kMergeThreads = 512;
template <int HD, int RS>
__global__ __launch_bounds__(kMergeThreads) void attention_paged_merge_kernel(AttnPagedArgs a) {
    constexpr int PER = kMergeRows * HD / 4, LANES = kMergeThreads / PER, AHEAD = 4;
    __shared__ float4 acc[kMergeThreads];
    __shared__ float2 st[kMergeThreads];
    constexpr int RB = 32 * RS / kMergeRows;
    const int nkv = a.pg.nkv, group = a.nh / nkv, T = 32 * RS / group;
    const int rb = blockIdx.x % RB, g = blockIdx.x / RB % nkv;
    Item it;
    if (!paged_item<true>(a.pg, T, a.target, blockIdx.x / RB / nkv, it) || it.splits < 2) return;
    const int ntok = min(T, it.n - it.tile * T);
    if (rb * kMergeRows >= ntok * group) return;
    const int tid = threadIdx.x, d = 4 * (tid % (HD / 4)), row = rb * kMergeRows + tid / (HD / 4) % kMergeRows;
    const int z0 = tid / PER;
    const bool valid = row < ntok * group;
    float M = -INFINITY, L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z = z0; valid && z < it.splits; z += LANES * AHEAD) {
        float2 t[AHEAD];
        float4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const size_t p = ((size_t)(it.slot + min(z + i * LANES, it.splits - 1)) * nkv + g) * (32 * RS) + row;
            t[i] = a.ml[p];
            v[i] = *reinterpret_cast<const float4*>(a.part + p * HD + d);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (z + i * LANES >= it.splits || t[i].x == -INFINITY) continue;  // (nothing attended there)
            const float m1 = fmaxf(M, t[i].x), a0 = __builtin_amdgcn_exp2f(M - m1), a1 = __builtin_amdgcn_exp2f(t[i].x - m1);
            M = m1;
            L = L * a0 + t[i].y * a1;
            s.x = s.x * a0 + v[i].x * a1, s.y = s.y * a0 + v[i].y * a1;
            s.z = s.z * a0 + v[i].z * a1, s.w = s.w * a0 + v[i].w * a1;
        }
    }
    acc[tid] = s;
    st[tid] = make_float2(M, L);
    __syncthreads();
    if (!valid || z0) return;
    for (int i = 1; i < LANES; ++i) {
        const float2 t = st[tid + i * PER];
        const float4 v = acc[tid + i * PER];
        if (t.x == -INFINITY) continue;
        const float m1 = fmaxf(M, t.x), a0 = __builtin_amdgcn_exp2f(M - m1), a1 = __builtin_amdgcn_exp2f(t.x - m1);
        M = m1;
        L = L * a0 + t.y * a1;
        s.x = s.x * a0 + v.x * a1, s.y = s.y * a0 + v.y * a1, s.z = s.z * a0 + v.z * a1, s.w = s.w * a0 + v.w * a1;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<float4*>(a.att + ((size_t)(it.first + it.tile * T + row / group) * a.nh + g * group + row % group) * HD + d) =
        make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
}

// What the host can choose without the lengths: rows of a tile by the average
// sequence, and the number of items that the splits aim at.
struct Shape {
    int rs, target;
    int64_t tiles;  // at most
};
Shape attention_shape(const PagedArgs& a, int nh, int hd) {
    Shape s;
    const int group = nh / a.nkv;
    s.rs = (int64_t)((a.n_tokens + a.n_seq - 1) / a.n_seq) * group > 32 ? 2 : 1;
    const int T = 32 * s.rs / group;
    s.tiles = a.n_tokens / T + a.n_seq;
    const int resident = (hd == 128 ? 1 : 2) * device_cus();
    s.target = ((int64_t)a.table_ld << a.page_shift) > kStage ? std::max(2, resident / a.nkv) : 0;
    return s;
}

template <int HD, int RS>
int launch(const AttnPagedArgs& a, const Shape& sh, hipStream_t st) {
    static bool attr_set = false;  // above 64 KiB of LDS needs the opt-in, once per kernel
    if (!attr_set && lds_bytes(HD, RS) > 65536) {
        if (hipFuncSetAttribute((const void*)attention_paged_kernel<HD, RS>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds_bytes(HD, RS)) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const int64_t items = (sh.target + sh.tiles) * a.pg.nkv, merges = sh.tiles * a.pg.nkv * (32 * RS / kMergeRows);
    if (items * kThreads > UINT32_MAX || merges * kMergeThreads > UINT32_MAX) return MXH_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((attention_paged_kernel<HD, RS>), dim3((unsigned)items), dim3(kThreads), lds_bytes(HD, RS), st, a);
    if (sh.target > 0)
        hipLaunchKernelGGL((attention_paged_merge_kernel<HD, RS>), dim3((unsigned)merges), dim3(kMergeThreads), 0, st, a);
    return MXH_OK;
}

}  // namespace

size_t attention_paged_work_bytes(const PagedArgs& a, int nh, int hd) {
    const Shape s = attention_shape(a, nh, hd);
    return (size_t)2 * s.target * a.nkv * 32 * s.rs * (hd + 2) * sizeof(float);
}

int attention_paged_launch(const PagedArgs& a, const float* q, int nh, int hd, float* att, void* work, hipStream_t st) {
    const Shape s = attention_shape(a, nh, hd);
    float* part = static_cast<float*>(work);
    float2* ml = reinterpret_cast<float2*>(part + (size_t)2 * s.target * a.nkv * 32 * s.rs * hd);
    const AttnPagedArgs args{a, q, att, part, ml, nh, s.target, 1.4426950408889634f / sqrtf((float)hd)};
    switch (hd) {
    case 32: return s.rs == 2 ? launch<32, 2>(args, s, st) : launch<32, 1>(args, s, st);
    case 64: return s.rs == 2 ? launch<64, 2>(args, s, st) : launch<64, 1>(args, s, st);
    default: return s.rs == 2 ? launch<128, 2>(args, s, st) : launch<128, 1>(args, s, st);
    }
}

}  // namespace mxh
