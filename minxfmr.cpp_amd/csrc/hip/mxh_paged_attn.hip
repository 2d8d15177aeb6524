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
// replaced, not added to, and since 0 times an infinity is none, blocks with
// unattended rows look their V values over; where one is infinite or NaN the
// products take the finite values alone, and two more products of 0 / 1
// matrices tell which sums have an infinity or a NaN coming (blend_special).
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
constexpr int kBlock = 32;                 // keys a wave takes at a time
constexpr int kStage = kWaves * kBlock;    // keys a workgroup takes at a time
constexpr int kSlots = 2;                  // blocks of a wave in LDS

__host__ __device__ constexpr int slot_bytes(int hd) { return 2 * kBlock * hd * 2; }  // K and V rows
// floats a wave leaves for the merge of one set: V sums [hd][32], references, sums
__host__ __device__ constexpr int merge_floats(int hd) { return hd * 32 + 64; }
__host__ __device__ constexpr int lds_bytes(int hd, int rs) {
    const int ring = kWaves * kSlots * slot_bytes(hd), merge = kWaves * rs * merge_floats(hd) * 4;
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
    uint32_t at[2][HD / 32];  // byte offsets in the V rows of a slot
    __device__ __forceinline__ VRead() {
        const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                const int key = 8 * h + 4 * r + ((lane & 15) >> 2);
                const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                at[r][d] = (uint32_t)(key * HD * 2 + 16 * (piece ^ v_swz(key)) + 8 * (lane & 1));
            }
    }
    // pairs of 16-byte pieces rotated by the key, so that the four keys of a
    // read lie in different banks (the same for keys 16 apart)
    static __device__ __forceinline__ int v_swz(int key) {
        return HD == 128 ? 2 * (key & 7) : HD == 64 ? 2 * ((key >> 1) & 3) : 2 * ((key >> 2) & 1);
    }
    __device__ __forceinline__ f16x8 operator()(uint32_t v0, int t, int d) const {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(v0 + at[0][d] + t * 16 * HD * 2));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(v0 + at[1][d] + t * 16 * HD * 2));
        return __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// whether any V value of the block is infinite or NaN
template <int HD>
__device__ __forceinline__ bool any_special(uint32_t v0) {
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    const int lane = threadIdx.x & 63;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const u32x4 x = *(lds_u32x4*)(uintptr_t)(v0 + 1024 * i + 16 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (x[e] & 0x7c00u) == 0x7c00u || (x[e] & 0x7c000000u) == 0x7c000000u;
    }
    return __any(bad);
}

// O^T += V^T P^T for one set where V has infinities or NaN: the finite values'
// products, and +-inf / NaN into the sums of rows that attend such a value.  w:
// this lane's row's attended keys, bit 16 t + u for key 16 t + 8 h + u.
template <int HD>
__device__ __forceinline__ void blend_special(const VRead<HD>& vr, uint32_t v0, uint32_t w, const f16x8 (&bh)[2],
                                              const f16x8 (&bl)[2], f32x16 (&o)[HD / 32]) {
    f16x8 on[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 8; ++u) on[t][u] = (w >> (16 * t + u)) & 1 ? (_Float16)1 : (_Float16)0;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) {
        f32x16 up, dn;
#pragma unroll
        for (int v = 0; v < 16; ++v) up[v] = dn[v] = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f16x8 a = vr(v0, t, d), pos, neg;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)a[u]);
                const bool odd = (b & 0x7c00u) == 0x7c00u, nan = odd && (b & 0x3ffu);
                pos[u] = nan || b == 0x7c00u ? (_Float16)1 : (_Float16)0;
                neg[u] = nan || b == 0xfc00u ? (_Float16)1 : (_Float16)0;
                if (odd) a[u] = (_Float16)0;
            }
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, bh[t], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, bl[t], o[d], 0, 0, 0);
            up = __builtin_amdgcn_mfma_f32_32x32x16_f16(pos, on[t], up, 0, 0, 0);
            dn = __builtin_amdgcn_mfma_f32_32x32x16_f16(neg, on[t], dn, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            if (up[v] > 0.f) o[d][v] += INFINITY;
            if (dn[v] > 0.f) o[d][v] -= INFINITY;
        }
    }
}

template <int HD, int RS>
__global__ __launch_bounds__(kThreads, HD == 128 || (HD == 64 && RS == 2) ? 1 : 2) void attention_paged_kernel(AttnPagedArgs a) {
    constexpr int KS = HD / 16, DB = HD / 32, NCH = HD / 8;
    constexpr int RPI = 64 / NCH;          // rows a load instruction brings
    constexpr int LPG = 16 / RPI;          // load instructions per 16 rows
    constexpr int LPB = 4 * LPG;           // per block, K and V
    extern __shared__ __align__(256) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int nkv = a.pg.nkv, group = a.nh / nkv, T = 32 * RS / group;
    const int g = blockIdx.x % nkv;
    Item it;
    if (!paged_item<false>(a.pg, T, a.target, blockIdx.x / nkv, it)) return;

    const int i0 = it.tile * T, ntok = min(T, it.n - i0);
    const int kend = it.cached + i0 + ntok;  // keys [0, kend) for the tile
    const int lim_min = a.pg.parent ? it.cached : it.cached + i0 + 1;  // every row attends the keys below
    const int st0 = it.split * it.stages, st1 = min(st0 + it.stages, (kend + kStage - 1) / kStage);
    // this wave's blocks
    const int nb = max(min(st1, (kend - kBlock * wave + kStage - 1) / kStage) - st0, 0);

    // Rows of K and V for block b, 16 of one page at a time.  Lane l holds the
    // page of the wave's 16-row group l of a window of 32 blocks.
    const uint32_t row_b = 2u * (uint32_t)(nkv * HD), page_b = row_b << a.pg.page_shift;
    const int* table = a.pg.table + (size_t)it.s * a.pg.table_ld;
    const auto page_ids = [&](int b0) __attribute__((always_inline)) {
        const int row = kStage * (st0 + b0 + (lane >> 1)) + kBlock * wave + 16 * (lane & 1), p = row >> a.pg.page_shift;
        int id = -1;
        if (row < kend && row >= 0 && p < a.pg.table_ld) id = table[p];
        return (unsigned)id < (unsigned)a.pg.n_pages ? id : -1;
    };
    int ids = page_ids(0), ids_next = ids;
    const uint64_t kbase = scalar_addr(a.pg.k + g * HD), vbase = scalar_addr(a.pg.v + g * HD);
    const uint64_t zero = scalar_addr(zero_row);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem +
                          (uint32_t)(wave * kSlots * slot_bytes(HD));
    const int lr = lane / NCH, lc = lane % NCH;
    const auto issue = [&](int b) __attribute__((always_inline)) {
        const uint32_t slot = lds0 + (uint32_t)(b % kSlots) * slot_bytes(HD);
        const int r0 = kStage * (st0 + b) + kBlock * wave;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int id = __builtin_amdgcn_readlane(ids, (2 * b + u) & 63), row = r0 + 16 * u;
            const uint32_t in = (uint32_t)(row & ((1 << a.pg.page_shift) - 1)) * row_b;
            const uint64_t off = (uint64_t)(uint32_t)id * page_b + in;
            const uint64_t kb = id < 0 ? zero : kbase + off, vb = id < 0 ? zero : vbase + off;
            // rows past the last repeat it (their scores are replaced); an absent
            // group reads the row of zeros
            const int last = id < 0 ? 0 : kend - 1 - row;
#pragma unroll
            for (int x = 0; x < LPG; ++x) {
                const int r = x * RPI + lr, key = 16 * u + r;
                const uint32_t ro = (uint32_t)min(r, last) * row_b;
                const uint32_t to = slot + (uint32_t)(16 * u + x * RPI) * (2 * HD);
                g2l_s(kb, ro + 16 * (lc ^ pa_swz<HD>(key)), to);
                g2l_s(vb, ro + 16 * (lc ^ VRead<HD>::v_swz(key)), to + kBlock * HD * 2);
            }
        }
    };
    if (nb > 0) issue(0);
    if (nb > 1) issue(1);

    // this lane's query row of each set, split; its last key (causal) or path
    f16x8 qh[RS][KS], ql[RS][KS];
    int lim[RS];
    uint64_t path[RS];
    uint64_t paths = 0;
    if (a.pg.parent) paths = tree_path(a.pg, it.first, it.n);
#pragma unroll
    for (int r = 0; r < RS; ++r) {
        const int row = 32 * r + n, tl = row / group, hh = row % group;
        const bool valid = tl < ntok;  // (the others: zeros at the tile's first token)
        const int i = i0 + (valid ? tl : 0);
        lim[r] = it.cached + i + 1;
        path[r] = 0;
        if (a.pg.parent)
            path[r] = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(paths >> 32), i) << 32) |
                      (uint32_t)__shfl((int)(uint32_t)paths, i);
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
                qh[r][ks][e] = hi[0], qh[r][ks][e + 1] = hi[1], ql[r][ks][e] = lo[0], ql[r][ks][e + 1] = lo[1];
            }
        }
    }

    float mref[RS], lrun[RS];
    f32x16 o[RS][DB];
#pragma unroll
    for (int r = 0; r < RS; ++r) {
        mref[r] = -INFINITY, lrun[r] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[r][d][v] = 0.f;
    }
    const VRead<HD> vr;
    const int krow = pa_pi(n);

    for (int b = 0; b < nb; ++b) {
        if (b + 1 < nb) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPB) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint32_t k0 = lds0 + (uint32_t)(b % kSlots) * slot_bytes(HD), v0 = k0 + kBlock * HD * 2;
        const int kb = kStage * (st0 + b) + kBlock * wave;
        f32x16 s[RS];
#pragma unroll
        for (int r = 0; r < RS; ++r)
#pragma unroll
            for (int v = 0; v < 16; ++v) s[r][v] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
            const f16x8 k = *(lds_f16x8*)(uintptr_t)(k0 + krow * HD * 2 + 16 * ((2 * ks + h) ^ pa_swz<HD>(krow)));
#pragma unroll
            for (int r = 0; r < RS; ++r) {
                s[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[r][ks], s[r], 0, 0, 0);
                s[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[r][ks], s[r], 0, 0, 0);
            }
        }
        const bool gone0 = __builtin_amdgcn_readlane(ids, (2 * b) & 63) < 0;
        const bool gone1 = __builtin_amdgcn_readlane(ids, (2 * b + 1) & 63) < 0;
        uint32_t w[RS];  // attended keys: bit 16 t + u for key 16 t + 8 h + u
        bool special = false;
        if (kb + kBlock > lim_min || gone0 || gone1) {
#pragma unroll
            for (int r = 0; r < RS; ++r) {
                if (a.pg.parent) {
                    const int sh = kb - it.cached;
                    w[r] = sh >= kTreeMax ? 0u
                           : sh >= 0      ? (uint32_t)(path[r] >> sh)
                           : sh > -32     ? (uint32_t)(path[r] << -sh) | ((1u << -sh) - 1u)
                                          : ~0u;
                } else {
                    const int left = lim[r] - kb;
                    w[r] = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
                }
                if (gone0) w[r] &= 0xffff0000u;
                if (gone1) w[r] &= 0xffffu;
                w[r] >>= 8 * h;
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (!((w[r] >> (16 * (v >> 3) + (v & 7))) & 1)) s[r][v] = -INFINITY;
            }
            special = any_special<HD>(v0);
        }
        float mx[RS];
        bool up = false;
#pragma unroll
        for (int r = 0; r < RS; ++r) {
            mx[r] = s[r][0];
#pragma unroll
            for (int v = 1; v < 16; ++v) mx[r] = fmaxf(mx[r], s[r][v]);
            mx[r] = pa_pair_max(mx[r]);
            up |= mx[r] > mref[r] + kPaSlack;  // also the first block with an attended key
        }
        if (__any(up)) {
#pragma unroll
            for (int r = 0; r < RS; ++r) {
                const float mnew = fmaxf(mref[r], mx[r]);
                // (nothing attended so far: the sums are zero)
                const float alpha = mref[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref[r] - mnew);
                mref[r] = mnew;
                lrun[r] *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[r][d][v] *= alpha;
            }
        }
        f16x8 bh[RS][2], bl[RS][2];
#pragma unroll
        for (int r = 0; r < RS; ++r) {
            const float ref0 = mref[r] == -INFINITY ? 0.f : mref[r];
            float p[16], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                p[v] = kPaScale * __builtin_amdgcn_exp2f(s[r][v] - ref0);
                ps[v & 3] += p[v];
            }
            lrun[r] += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int u = 0; u < 8; u += 2) {
                    f16x2 hi, lo;
                    pa_split(p[8 * t + u], p[8 * t + u + 1], hi, lo);
                    bh[r][t][u] = hi[0], bh[r][t][u + 1] = hi[1], bl[r][t][u] = lo[0], bl[r][t][u + 1] = lo[1];
                }
        }
        if (special) {
#pragma unroll
            for (int r = 0; r < RS; ++r) blend_special<HD>(vr, v0, w[r], bh[r], bl[r], o[r]);
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 v = vr(v0, t, d);
#pragma unroll
                    for (int r = 0; r < RS; ++r) {
                        o[r][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, bh[r][t], o[r][d], 0, 0, 0);
                        o[r][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, bl[r][t], o[r][d], 0, 0, 0);
                    }
                }
        }
        // the slot's last reads are done before its next rows are requested
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        // a window's pages are requested 30 blocks ahead of their use
        if ((b & 31) == 0 && b + 32 < nb) ids_next = page_ids(b + 32);
        if (((b + kSlots) & 31) == 0) ids = ids_next;
        if (b + kSlots < nb) issue(b + kSlots);
    }

    // the waves' parts meet (every load into the slots has been waited for)
    __syncthreads();
    float* ms = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int r = 0; r < RS; ++r) {
        float* mb = ms + (wave * RS + r) * merge_floats(HD);
        const float lsum = lrun[r] + __shfl_xor(lrun[r], 32, 64);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) mb[(32 * d + 8 * (v >> 2) + 4 * h + (v & 3)) * 32 + n] = o[r][d][v];
        if (h == 0) {
            mb[HD * 32 + n] = mref[r];
            mb[HD * 32 + 32 + n] = lsum;
        }
    }
    __syncthreads();
    // thread: row 32 mr + mn, dims d0 .. d0 + ND
    constexpr int ND = HD * RS / 8;
    const int mr = RS == 2 ? (tid >> 5) & 1 : 0, mn = tid & 31, d0 = (tid >> (RS == 2 ? 6 : 5)) * ND;
    const float* mb[kWaves];
    float wt[kWaves], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        mb[i] = ms + (i * RS + mr) * merge_floats(HD);
        M = fmaxf(M, mb[i][HD * 32 + mn]);
    }
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
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
            const int at = (d0 + d + e) * 32 + mn;
            x[e] = ((wt[0] * mb[0][at] + wt[1] * mb[1][at]) + (wt[2] * mb[2][at] + wt[3] * mb[3][at])) * inv;
        }
        *reinterpret_cast<float4*>(op + d0 + d) = make_float4(x[0], x[1], x[2], x[3]);
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
