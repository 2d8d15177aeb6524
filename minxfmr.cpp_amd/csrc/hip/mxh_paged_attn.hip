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
// r % group), R = 16 or 64 rows.  Where the batch has tiles enough of like
// length, an item is a tile, those with the most keys of a sequence first.
// Elsewhere the stages (128 or 64 keys) of all tiles are laid end to end and cut
// into items of equal length, whatever tiles they cross: the workgroups, all
// resident, end together.  A tile that is cut leaves its parts in the workspace,
// two at most an item, and a second kernel joins them.  The lengths are on the
// device, so every workgroup makes the plan for itself (Plan; its integers are in
// mxh_paged_plan.h); the grid is as wide as the plan can be, and what is past its
// end leaves at once.
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
// replaced, not added to, and since 0 times an infinity is no zero, an item whose
// sums met an infinity or a NaN is computed again in fp32, without products over
// rows that a token does not attend (redo_item).  That takes in infinite scores.
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

// floats a wave leaves for the merge: V sums [m][hd + 4], references, sums (and a flag, behind all of theirs)
__host__ __device__ constexpr int merge_floats(int hd, int m) { return m * (hd + 6); }
__host__ __device__ constexpr int lds_bytes(int hd, int rows) {
    const int ring = 2 * 128 * hd * 2,  // R = 16: a stage, R = 64: two
               merge = kWaves * (merge_floats(hd, rows == 16 ? 16 : 32) + 1) * 4;
    return ring > merge ? ring : merge;
}

// what absent rows read
__device__ __align__(256) uint32_t zero_row[64];

// A tile, or some of its stages
struct Segment {
    int s;
    uint32_t first, n, cached;
    uint32_t tile, st0, st1;  // stages [st0, st1)
    int slot;                 // of the part in the workspace; -1: the whole tile
};

__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {  // inclusive
    int v = (int)x;
    v += dpp_i<0x111>(v);       // row_shr:1
    v += dpp_i<0x112>(v);
    v += dpp_i<0x114>(v);
    v += dpp_i<0x118>(v);
    v += dpp_i<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp_i<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return (uint32_t)v;
}

// The line of the batch's units (mxh_paged_plan.h), made by a wave from the
// lengths.  All uniform but what a lane says of its sequences.
struct Plan : PagedLine {
    const PagedArgs& a;

    __device__ __forceinline__ PagedSeq seq(int s) const {
        return PagedLine::seq(a.start[s], a.start[s + 1], a.cached[s], a.n_tokens, (uint64_t)a.table_ld << a.page_shift);
    }

    // Lane l's sequences are [l part, (l + 1) part), units `upto - sum` to `upto`
    int part;
    uint32_t sum, upto;
    PagedSeq mine;  // (part == 1: the lane's sequence)

    __device__ __forceinline__ Plan(const PagedArgs& args, int rows, uint32_t tokens, int target)
        : PagedLine(rows, tokens, args.parent != nullptr, target), a(args) {
        const int lane = threadIdx.x & 63;
        part = (a.n_seq + 63) / 64;
        sum = 0;
        mine = PagedSeq{0, 0, 0, 0, 0};
        uint32_t tiles = 0, longest = 0;
        bool falls = false;
        for (int s = lane * part; s < min((lane + 1) * part, a.n_seq); ++s) {
            mine = seq(s);
            falls |= a.start[s + 1] < a.start[s];
            tiles += mine.tiles;
            if (cut && mine.tiles > 0) sum += units(mine), longest = max(longest, lead + mine.stages);
        }
        if (cut) {
            upto = wave_scan(sum);
            const uint32_t units = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
            settle_cut(units, __any(cut_pays(rows, (float)longest, (float)units, (float)target)), rows, target);
        }
        if (!cut) {
            sum = tiles;
            upto = wave_scan(sum);
            settle_whole((uint32_t)__builtin_amdgcn_readlane((int)upto, 63));
        }
        if (__any(falls)) total = 0;  // (sequences that overlap: their units need not fit 32 bits)
    }
    // the sequence of unit x (< total), and x from its first unit on
    __device__ __forceinline__ int find(uint32_t& x, PagedSeq& q) const {
        const int l = __ffsll((unsigned long long)__ballot(upto > x)) - 1;
        const auto lane_l = [l](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
        x -= lane_l(upto - sum);
        if (part == 1) {
            q = PagedSeq{lane_l(mine.first), lane_l(mine.n), lane_l(mine.cached), lane_l(mine.tiles),
                         lane_l(mine.stages)};
            return l;
        }
        int s = l * part;
        for (;; ++s) {  // (ends within the lane's sequences: they hold x)
            q = seq(s);
            const uint32_t here = units(q);
            if (x < here || s + 1 >= min((l + 1) * part, a.n_seq)) return s;
            x -= here;
        }
    }
};

// N loads of g2l_s, to lds, lds + 1024, ...: an instruction's offset counts for both
// of its addresses, so off[i] is 1024 i less than where lane i's bytes are.  (One M0
// for all: as LDS addresses of their own they filled the scalar registers and were
// read back from spilled lanes at every load.)
#define MXH_G2L_ROWS(HINT)                                                                                             \
    if constexpr (N == 4)                                                                                              \
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %4" HINT                                                  \
                     "\n\tglobal_load_lds_dwordx4 %1, %4 offset:%6" HINT                                               \
                     "\n\tglobal_load_lds_dwordx4 %2, %4 offset:%7" HINT                                               \
                     "\n\tglobal_load_lds_dwordx4 %3, %4 offset:%8" HINT ::"v"(off[0]),                                \
                     "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "{m0}"(lds), "n"(1024), "n"(2 * 1024),          \
                     "n"(3 * 1024)                                                                                     \
                     : "memory");                                                                                      \
    else if constexpr (N == 2)                                                                                         \
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %2" HINT                                                  \
                     "\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4" HINT ::"v"(off[0]),                                \
                     "v"(off[1]), "s"(base), "{m0}"(lds), "n"(1024)                                                    \
                     : "memory");                                                                                      \
    else                                                                                                               \
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" HINT ::"v"(off[0]), "s"(base), "{m0}"(lds) : "memory")
template <int N>
__device__ __forceinline__ void g2l_rows(uint64_t base, const uint32_t (&off)[N], uint32_t lds) {
    static_assert(N == 1 || N == 2 || N == 4, "");
    MXH_G2L_ROWS("");
}
// of rows that nothing else will read: their lines are the next to leave the caches
template <int N>
__device__ __forceinline__ void g2l_rows_once(uint64_t base, const uint32_t (&off)[N], uint32_t lds) {
    MXH_G2L_ROWS(" nt");
}
#undef MXH_G2L_ROWS

struct AttnPagedArgs {
    PagedArgs pg;
    const float* q;
    float* att;
    float* part;  // [2 target][nkv][R][HD]: V sums of the parts of tiles
    float2* ml;   // [2 target][nkv][R]: references and sums
    int4* cuts;   // [target]: of the tile that is cut first where item i starts, its first token, rows, parts (0: none)
    int nh, target;  // target: items that stages are cut into, at most; 0: an item is a tile
    float qscale;
    uint32_t group, tokens;  // q heads of a kv head; tokens of a tile, R / group
    uint32_t group_inv;      // 2^16 / group rounded up
    // r / group for r up to 64
    __device__ __forceinline__ uint32_t over_group(uint32_t r) const { return (r * group_inv) >> 16; }
};
// the workgroup's item: the grid is (kv heads, items, more of them)
__device__ __forceinline__ uint32_t item_index() { return blockIdx.y + gridDim.y * blockIdx.z; }

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
    __device__ __forceinline__ explicit VRead(int lane) {
        const int key = 8 * (M == 32 ? lane >> 5 : lane >> 4) + ((lane & 15) >> 2);
        const int piece = (M == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
        at = (uint32_t)(key * HD * 2 + 16 * (piece ^ v_swz<HD>(key)) + 8 * (lane & 1));
    }
    // v0: the rows' place, a multiple of 256 bytes.  Dims M d on are 2 M d bytes
    // on; keys 4 on are 4 rows on, rotated by another HD bytes
    __device__ __forceinline__ f16x8 operator()(uint32_t v0, int t, int d) const {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const uint32_t p = (v0 + at) ^ (uint32_t)(2 * M * d);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(p + t * 32 * HD));
        const uint32_t p1 = (p ^ HD) + t * 32 * HD + 8 * HD;
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)p1);
        return __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// The item again with a wave a row and no product that meets a value its row
// does not attend: a key a lane for the scores, then a dim a lane (or two) for
// the sums.  For items whose sums met an infinity or a NaN; the rest of the
// kernel pays no register for it.
template <int HD, int R>
__device__ void redo_item(const AttnPagedArgs& a, const Segment& it, int g, int key0, int key1, uint8_t* smem) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = (int)a.group, T = (int)a.tokens, i0 = (int)it.tile * T, rows = min(T, (int)it.n - i0) * group;
    float* qs = reinterpret_cast<float*>(smem + wave * 2048);                  // the row's q
    float* ps = reinterpret_cast<float*>(smem + wave * 2048 + 512);            // 64 keys' probabilities
    int64_t* at = reinterpret_cast<int64_t*>(smem + wave * 2048 + 1024);       // and pool rows
    const uint64_t paths = a.pg.parent ? tree_path(tree_parent(a.pg, (int)it.first, (int)it.n)) : 0;
    const auto settle = [] {  // what the wave's lanes wrote is there for the others
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    };
    for (int r = wave; r < rows; r += kWaves) {
        const int tl = (int)a.over_group((uint32_t)r), i = i0 + tl, hq = g * group + r - tl * group;
        const int tok = (int)it.first + i, cached = (int)it.cached;
        const uint64_t path = path_of(paths, i & 63);
        const float* q = a.q + ((size_t)tok * a.nh + hq) * HD;
        for (int d = lane; d < HD; d += 64) qs[d] = q[d] * a.qscale;
        settle();
        float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
        const int end = min(key1, cached + i + 1);
        for (int k0 = key0; k0 < end; k0 += 64) {
            const int key = k0 + lane;
            bool on = key < end && (key < cached || !a.pg.parent || (path >> ((key - cached) & 63) & 1));
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
        if (it.slot >= 0) {
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

// q enters as fp16 hi + lo, which say 22 bits of a value from 2^-3 up to 65504 and
// steps of 2^-24 below.  A row whose largest |q| (with log2(e) / sqrt(hd)) lies
// outside [2^-3, 2^15) is multiplied by the 2^f that brings it to [2^13, 2^14), and
// its scores are multiplied by 2^-f, which is what this returns (1: neither; none
// for zeros and infinities).  Every q is then within 2^-22 of the row's largest.
// Ordinary q stay in the range and pay a branch a stage and the search for the
// largest: packed prompts 270 us (267 without either), the tree of 27 24.3 (23.9).
// Where all rows are scaled the prompts take 270 us too (flat scores, q a fiftieth
// as large; 261 without); with the blocks of scaled rows sent the way of those that
// need a mask, 290.
__device__ __forceinline__ float q_unscale(float largest) {
    const int f = min(14 - __builtin_amdgcn_frexp_expf(largest), 120);  // (down to 2^-107; scores of less are zero)
    const bool as_it_is = (largest >= 0.125f && largest < 32768.f) || !(largest > 0.f) || largest == INFINITY;
    return as_it_is ? 1.f : __uint_as_float((uint32_t)(127 - f) << 23);
}
// the largest of x, |a|, |b| (as fmaxf every operand costs an instruction of its own)
__device__ __forceinline__ float larger_of(float x, float a, float b) {
    float m;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(m) : "v"(x), "v"(a), "v"(b));
    return m;
}
// 1 / x of a power of two
__device__ __forceinline__ float inverse_power(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// R = 16: every wave takes 32 keys of a stage of 128 for all rows of the tile
// and reads only what it loaded: no barrier before the merge.  K and V have one
// place each; the next K comes while V is used, the next V while K is.
// R = 64: two waves, one a set of 32 rows, take the same 32 keys of a stage of
// 64, which all four waves load, a barrier a stage.  The scores run a stage
// ahead, so that a wave's products of the next scores and its vector work on
// these can overlap: at stage st there are V(st), K(st + 1), and on their way
// V(st + 1), K(st + 2).
//
// Measured with 32/8 heads of 128:
//   R = 16: 48 single tokens at up to 16,000 rows 229 us = 6.3 TB/s of K and V (a
//   large read 6.7), bound by those; one at 8,192 14 us.  One token of 16/8 heads
//   at 700 10.0 us: two launches, and in the first the plan's, the pages' and the
//   rows' loads one after the other.
//   R = 64: six packed prompts of 29 to 2,100 tokens behind up to 1,500 rows 267
//   us (263 to 270 card to card) = 464 TFLOP/s of the formula's, 930 of the products
//   made (a large fp16 product 1,184); matrix cores and vector units half busy
//   each, and neither fewer reads nor fewer exponentials made it faster by more
//   than 4%.  27 drafted tokens at 8,192 rows 24.2 us: 8 stages an item 12 of them
//   (a stage's loads are one stage ahead and HBM is 1.4 us away), what comes before
//   and after an item's stages 8, the second kernel 4.
// Many sequences: every workgroup plans for itself, so 1,024 single tokens at up to
// 300 rows take 282 us (their rows 78) and 4,096 2,980 (304); 256 take 41 (19).
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
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int set = wave % RS, kg = wave / RS;
    const uint32_t nkv = (uint32_t)a.pg.nkv, group = a.group, T = a.tokens;
    const uint32_t index = item_index(), g = blockIdx.x;
    const Plan plan(a.pg, R, T, a.target);
    static_assert(STAGE == stage_keys(R), "");
    uint32_t x = plan.first_unit(index);
    const bool tells = g == 0 && threadIdx.x == 0 && index < (uint32_t)a.target;  // (for the second kernel)
    if (x >= plan.total) {
        if (tells) a.cuts[index] = make_int4(0, 0, 0, 0);
        return;
    }
    const uint32_t x0 = x, x1 = min(x + plan.per, plan.total);
    PagedSeq seq;
    uint32_t r_unit = x;
    Segment it;
    it.s = plan.find(r_unit, seq);
    for (;;) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // (else what follows from it is kept in registers from tile to tile)
        const int lane = tid & 63, n = lane % M, h = lane / M;
        {
            const Plan::Spot spot = plan.spot(seq, r_unit);
            const PagedPiece p = plan.piece(seq, spot, x1 - x, index);
            it.first = seq.first, it.n = seq.n, it.cached = seq.cached;
            it.tile = p.tile, it.st0 = p.st0, it.st1 = p.st1, it.slot = p.slot;
            if (tells && x == x0) {
                const int i0 = (int)(spot.tile * T), rows = min((int)T, (int)seq.n - i0) * (int)group;
                a.cuts[index] = make_int4((int)seq.first + i0, rows, (int)plan.parts(spot), 0);
            }
            x += p.len, r_unit += p.len;
        }
        if (it.st0 < it.st1 || it.slot < 0) {  // (else only units of the lead)
        const int i0 = (int)(it.tile * T), ntok = min((int)T, (int)it.n - i0), cached = (int)it.cached;
        // keys [0, kend) for the tile
        const int kend = (int)min((int64_t)(cached + i0 + ntok), (int64_t)a.pg.table_ld << a.pg.page_shift);
        const int lim_min = a.pg.parent ? cached : cached + i0 + 1;  // every row attends the keys below
        const int key0 = STAGE * (int)it.st0, key1 = min(STAGE * (int)it.st1, kend);
        const int nst = max((key1 - key0 + STAGE - 1) / STAGE, 0);

        // this lane's query row
        const uint32_t row = 32 * set + n, tl = a.over_group(row);
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
                    qv[ks][e] = valid ? *reinterpret_cast<const float4*>(qp + HD / KS * ks + 4 * e)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const int parent = a.pg.parent ? tree_parent(a.pg, (int)it.first, (int)it.n) : -1;

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
        // Whether the rows are read once: the batch's are more than the 256 MB that the
        // last cache holds, so none stay for the next call, the sequence has no other
        // tile, and none of the 63 sequences around it has the first row's page in the
        // same place, as forks would.  Then the loads say so, and the caches do not fill
        // with them: 48 single tokens at up to 16,000 rows 255 us without, 228 with;
        // 64 at up to 9,000 rows, 8,000 of them shared, 158 and 205.
        bool once = false;
        if constexpr (PRIVATE) {
            if (nst > 0 && seq.tiles == 1 && (float)plan.all * (float)(STAGE * 4 * HD) * (float)nkv > 256e6f) {
                const int page = key0 >> a.pg.page_shift, s = max(min(it.s - 32, a.pg.n_seq - 64), 0) + lane;
                int other = -2;
                if (s < a.pg.n_seq && s != it.s) other = a.pg.table[(size_t)s * a.pg.table_ld + page];
                once = !__any(other == table[page]);
            }
        }
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
            const uint32_t at = r * row_b - 1024 * x;  // (not below zero: x * RPI rows have 1024 x bytes of one head)
            koff[x] = at + 16 * (uint32_t)(lane % NCH ^ pa_swz<HD>((int)r));
            voff[x] = at + 16 * (uint32_t)(lane % NCH ^ v_swz<HD>((int)r));
        }
        // the wave's rows of a stage into K's or V's place
        const auto issue = [&](const Place& p, uint32_t place, bool is_v) __attribute__((always_inline)) {
            const uint32_t(&off)[LPG] = is_v ? voff : koff;
            const auto from = [&](int u) {
                return (is_v ? vbase : kbase) + (((uint64_t)(uint32_t)p.hi[u] << 32) | (uint32_t)p.lo[u]);
            };
            const auto to = [&](int u) { return place + 32 * (OWN * wave + u) * HD; };
            bool all = p.r0 + 16 * OWN - 1 < kend;
#pragma unroll
            for (int u = 0; u < OWN; ++u) all &= p.hi[u] >= 0;
            if (all && PRIVATE && once) {
#pragma unroll
                for (int u = 0; u < OWN; ++u) g2l_rows_once(from(u), off, to(u));
            } else if (all) {
#pragma unroll
                for (int u = 0; u < OWN; ++u) g2l_rows(from(u), off, to(u));
            } else {
                // rows past the last repeat it (their scores are replaced); an absent
                // group reads the row of zeros
#pragma unroll
                for (int u = 0; u < OWN; ++u) {
                    const bool none = p.hi[u] < 0;
                    const uint32_t last = none ? 0 : (uint32_t)max(min(kend - 1 - p.r0 - 16 * u, 15), 0);
                    const uint64_t at = none ? scalar_addr(zero_row) : from(u);
#pragma unroll
                    for (int x = 0; x < LPG; ++x) {
                        const uint32_t r = x * RPI + lr;
                        g2l_s(at, off[x] + 1024 * x - (r - min(r, last)) * row_b, to(u) + 1024 * x);
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
                const uint32_t t = a.over_group(r);
                const uint32_t off = 4 * (min(t, (uint32_t)ntok - 1) * (uint32_t)qd + (r - t * group) * HD) +
                                     16 * ((lane % QP) ^ (r & 7));
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
        // The row's q by a power of two where fp16 halves would lose it: unscale is
        // 2^-f, what turns its scores back (q_unscale)
        float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                big[e] = larger_of(big[e], qv[ks][e].x, qv[ks][e].y);
                big[e + 2] = larger_of(big[e + 2], qv[ks][e].z, qv[ks][e].w);
            }
        const float unscale = q_unscale(row_max<M>(larger_of(fmaxf(big[0], big[1]), big[2], big[3])) * a.qscale);
        const float qscale = a.qscale * inverse_power(unscale);
        const bool scaled = __any(unscale != 1.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const float v[8] = {qv[ks][0].x, qv[ks][0].y, qv[ks][0].z, qv[ks][0].w,
                                qv[ks][1].x, qv[ks][1].y, qv[ks][1].z, qv[ks][1].w};
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                f16x2 hi, lo;
                pa_split(v[e] * qscale, v[e + 1] * qscale, hi, lo);
                qh[ks][e] = hi[0], qh[ks][e + 1] = hi[1], ql[ks][e] = lo[0], ql[ks][e + 1] = lo[1];
            }
        }
        RowMask mask{cached, cached + i + 1, 0, a.pg.parent != nullptr};
        if (a.pg.parent) mask.path = path_of(tree_path(parent), i);

        float mref = -INFINITY, lrun = 0.f;
        acc_t o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < NA; ++v) o[d][v] = 0.f;
        const VRead<HD, M> vr(lane);
        // this lane's first piece of its K row; the next products' are 1024 / M bytes on
        const int key_row = M == 32 ? pa_pi(n) : 8 * (n >> 2) + (n & 3);
        const uint32_t krow = (uint32_t)(key_row * HD * 2 + 16 * (h ^ pa_swz<HD>(key_row)));

        // what the rows do not attend, out of the scores of the block at key kb
        const auto unmask = [&](int kb, acc_t (&s)[SB]) __attribute__((always_inline)) {
            uint32_t w = mask(kb);
            if (gone >> (2 * kg) & 1) w &= 0xffff0000u;
            if (gone >> (2 * kg) & 2) w &= 0xffffu;
            w >>= 8 * h;  // value v: key 8 h + 16 (v / 8) + v % 8
#pragma unroll
            for (int v = 0; v < NP; ++v)
                if (!((w >> (16 * (v >> 3) + (v & 7))) & 1)) s[v / NA][v % NA] = -INFINITY;
        };
        const auto largest = [&](const acc_t (&s)[SB]) __attribute__((always_inline)) {
            float mx = s[0][0];
#pragma unroll
            for (int v = 1; v < NP; ++v) mx = fmaxf(mx, s[v / NA][v % NA]);
            return row_max<M>(mx);
        };
        // The scores come as S - ref: the products start at minus the reference (0
        // while there is none).  mx: the row's largest.  The reference moves only
        // where a score exceeds it by 2^kPaSlack, and at the first attended key.
        acc_t start;
#pragma unroll
        for (int v = 0; v < NA; ++v) start[v] = 0.f;
        // scores of the wave's keys with K's rows at k0
        const auto score = [&](uint32_t k0, acc_t (&s)[SB]) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
                s[b] = start;
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
        const auto move_reference = [&](float mx, acc_t (&s)[SB]) __attribute__((always_inline)) {
            const bool first = mref == -INFINITY;
            if (!__any(mx > (first ? -INFINITY : kPaSlack))) return;
            const float up = first ? (mx == -INFINITY ? 0.f : mx) : fmaxf(mx, 0.f);
            const float alpha = first ? 0.f : __builtin_amdgcn_exp2f(-up);  // (first: the sums are zero)
            if (!first) mref += up;
            else if (mx > -INFINITY) mref = mx;
            lrun *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < NA; ++v) o[d][v] *= alpha;
#pragma unroll
            for (int v = 0; v < NP; ++v) s[v / NA][v % NA] -= up;
#pragma unroll
            for (int v = 0; v < NA; ++v) start[v] = mref == -INFINITY ? 0.f : -mref * inverse_power(unscale);
        };
        // scores of scaled rows as they are without the scale
        const auto turn_back = [&](acc_t (&s)[SB]) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < NP; ++v) s[v / NA][v % NA] *= unscale;
        };
        f16x8 bh[TT], bl[TT];
        const auto weigh = [&](const acc_t (&s)[SB]) __attribute__((always_inline)) {
            float p[NP], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < NP; ++v) {
                p[v] = kPaScale * __builtin_amdgcn_exp2f(s[v / NA][v % NA]);
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

        // R = 64: weigh, the next score and sum, interleaved as written (left to
        // itself the scheduler puts one behind the other).  A product keeps the matrix
        // cores busy for 32 cycles, time for some seven other instructions of a wave,
        // so what they wait for is spread: beside a score's products the vector work
        // of two values for two of them, every instruction a product away from what it
        // needs; beside the sums' products the next scores' largest.  Returns that.
        const auto weigh_and_score = [&](uint32_t k0, uint32_t v0, const acc_t (&s)[SB],
                                         acc_t (&next)[SB]) __attribute__((always_inline)) {
            float mx = -INFINITY;
            if constexpr (!PRIVATE) {
                constexpr int STEPS = 2 * KS, VALS = NP / STEPS;  // products; scores beside one
                constexpr int AHEAD = KS < 3 ? KS : 3;            // operands on their way
                constexpr int Y = TT * DB;
                typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
                f16x8 kf[KS], vf[Y];
                const auto k_read = [&](int ks) {
                    kf[ks] = *(lds_f16x8*)(uintptr_t)((k0 + krow) ^ (uint32_t)(32 * ks));
                };
#pragma unroll
                for (int ks = 0; ks < AHEAD; ++ks) k_read(ks);
                float p[NP], ps[4] = {0.f, 0.f, 0.f, 0.f};
                f16x2 hi[NP / 2];
                float e[NP], rest[NP];
                // a value's steps: exponential; scaled and summed; (pairs) high half; rests; low half
                // (work(u): the u-th value's exponential and what follows from earlier ones)
                const auto work = [&](int u) __attribute__((always_inline)) {
                    const int pr = (u - 5) / 2;
                    if (u >= 5 && (u - 5) % 2 == 0 && pr < NP / 2) {
                        rest[2 * pr] = pa_rest<0>(p[2 * pr], hi[pr]);
                        rest[2 * pr + 1] = pa_rest<1>(p[2 * pr + 1], hi[pr]);
                    }
                    if (u < NP) e[u] = __builtin_amdgcn_exp2f(s[0][u]);
                    if (u >= 1 && u - 1 < NP) {
                        p[u - 1] = kPaScale * e[u - 1];
                        ps[(u - 1) & 3] += p[u - 1];
                    }
                    if (u >= 3 && (u - 3) % 2 == 0 && (u - 3) / 2 < NP / 2) {
                        const int q = (u - 3) / 2;
                        hi[q] = __builtin_convertvector((f32x2{p[2 * q], p[2 * q + 1]}), f16x2);
                        asm("" : "+v"(hi[q]));
                        bh[q / 4][2 * q % 8] = hi[q][0], bh[q / 4][2 * q % 8 + 1] = hi[q][1];
                    }
                    if (u >= 6 && (u - 6) % 2 == 0 && (u - 6) / 2 < NP / 2) {
                        const int q = (u - 6) / 2;
                        const f16x2 lo = __builtin_convertvector((f32x2{rest[2 * q], rest[2 * q + 1]}), f16x2);
                        bl[q / 4][2 * q % 8] = lo[0], bl[q / 4][2 * q % 8 + 1] = lo[1];
                    }
                };
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < STEPS; ++j) {
                    const int ks = j / 2;
                    next[0] = MM::mul(kf[ks], j & 1 ? ql[ks] : qh[ks], j ? next[0] : start);
                    if (j & 1) {
                        if (ks + AHEAD < KS) k_read(ks + AHEAD);
                        else if (ks + AHEAD - KS < Y)
                            vf[ks + AHEAD - KS] = vr(v0, (ks + AHEAD - KS) / DB, (ks + AHEAD - KS) % DB);
                    }
#pragma unroll
                    for (int u = VALS * j; u < VALS * (j + 1); ++u) work(u);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int u = NP; u < NP + 6; ++u) work(u);
                lrun += (ps[0] + ps[1]) + (ps[2] + ps[3]);
                mx = -INFINITY;
#pragma unroll
                for (int y = 0; y < Y; ++y) {
                    o[y % DB] = MM::mul(vf[y], bh[y / DB], o[y % DB]);
                    o[y % DB] = MM::mul(vf[y], bl[y / DB], o[y % DB]);
                    if (y + AHEAD < Y) vf[y + AHEAD] = vr(v0, (y + AHEAD) / DB, (y + AHEAD) % DB);
                    // (from Y0 on: the scores are done by then)
                    constexpr int Y0 = Y / 4 > 1 ? Y / 4 : 1, PER = (NP + Y - Y0 - 1) / (Y - Y0);
#pragma unroll
                    for (int v = PER * (y - Y0); y >= Y0 && v < PER * (y - Y0 + 1) && v < NP; ++v)
                        mx = fmaxf(mx, next[0][v]);
                    asm volatile("" : "+v"(mx));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            return mx;
        };

        if constexpr (PRIVATE) {
            for (int st = 0; st < nst; ++st) {
                const uint32_t k0 = k_place(st) + 64 * kg * HD, v0 = v_place(st) + 64 * kg * HD;
                const int kb = key0 + STAGE * st + 32 * kg;  // first key of this wave's block
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
                    if (__builtin_expect(scaled, 0)) turn_back(s);
                    if (kb + 32 > lim_min || gone) unmask(kb, s);
                    move_reference(largest(s), s);
                    weigh(s);
                    // V, not the next K
                    if (st + 1 < nst) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPG * OWN) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    sum(v0);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (st + 1 < nst) issue(ahead, v_place(0), true), gone = ahead.gone;
            }
        } else {
            acc_t s[SB], next[SB];
            float mx = -INFINITY;
            if (nst > 0) {
                // K(0) has landed for every wave (V(0) with it; K(1) may be out)
                if (nst > 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LPG * OWN) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
                score(k_place(0) + 64 * kg * HD, s);
                mx = largest(s);
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
                if (__builtin_expect(scaled, 0)) turn_back(s), mx *= unscale;
                if (kb + 32 > lim_min || gone) {  // (a block behind the last key has every score replaced)
                    unmask(kb, s);
                    mx = largest(s);
                }
                move_reference(mx, s);
                // (past the last stage the scores of whatever lies there, unused)
                mx = row_max<M>(weigh_and_score(k_place(st + 1) + 64 * kg * HD, v0, s, next));
                s[0] = next[0];
                gone = gone_next, gone_next = ahead.gone;
            }
        }

        // the waves' parts meet, where no load is to come any more
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        float* ms = reinterpret_cast<float*>(smem);
        uint32_t* flags = reinterpret_cast<uint32_t*>(ms + kWaves * merge_floats(HD, M));
        {
            float* mb = ms + wave * merge_floats(HD, M);  // V sums [M rows][HD + 4], references, sums
            const float lsum = row_sum<M>(lrun);
            float bad = 0.f;
            if (valid) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int v = 0; v < NA; v += 4) {
                        *reinterpret_cast<float4*>(mb + n * (HD + 4) + M * d + 2 * v + 4 * h) =
                            make_float4(o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) bad = fmaf(o[d][v + e], 0.f, bad);
                    }
                if (h == 0) {
                    mb[M * (HD + 4) + n] = mref;
                    mb[M * (HD + 5) + n] = lsum;
                }
            }
            // An infinity or a NaN in a V row makes sums of infinities and NaN, of rows
            // that attend it and, as 0 times it, of rows that do not; one in K a NaN of
            // what may be an infinite score (its products with q's halves meet).  Nothing
            // helps a row whose q is not finite.
            bool redo = valid && !(bad == 0.f);
            if (redo && !(lsum == lsum)) {
                const float* qp = q0 + (i - i0) * qd + (row - tl * group) * HD;
                float rest = 0.f;
#pragma unroll 1
                for (int d = 0; d < HD; ++d) rest = fmaf(qp[d], 0.f, rest);
                redo = rest == 0.f;
            }
            const uint64_t any = __ballot(redo);
            if (lane == 0) flags[wave] = any != 0;
        }
        __syncthreads();
        const bool again = flags[0] | flags[1] | flags[2] | flags[3];
        if (again) {  // (uniform)
            __syncthreads();
            redo_item<HD, R>(a, it, (int)g, key0, key1, smem);
        }
        // a thread takes four dims of every PASS-th row (past the tile's last: whatever lies there, not stored)
        constexpr int PASS = kThreads / (HD / 4);
        const int d = 4 * (tid % (HD / 4)), rows = again ? 0 : ntok * (int)group;
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += PASS) {
            const int rr = r0 + tid / (HD / 4), rn = rr % M;
            const float* mb = ms + (rr / M % RS) * merge_floats(HD, M);
            constexpr int NEXT = RS * merge_floats(HD, M);  // (the next key group's part)
            float wt[KG], mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int k = 0; k < KG; ++k) mm = fmaxf(mm, mb[k * NEXT + M * (HD + 4) + rn]);
            float4 x4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KG; ++k) {
                const float mk = mb[k * NEXT + M * (HD + 4) + rn], lk = mb[k * NEXT + M * (HD + 5) + rn];
                wt[k] = lk == 0.f ? 0.f : __builtin_amdgcn_exp2f(mk - mm);  // (0: nothing attended there)
                ll += wt[k] * lk;
                const float4 v = *reinterpret_cast<const float4*>(mb + k * NEXT + rn * (HD + 4) + d);
                x4.x += wt[k] * v.x, x4.y += wt[k] * v.y, x4.z += wt[k] * v.z, x4.w += wt[k] * v.w;
            }
            if (rr >= rows) continue;
            if (it.slot >= 0) {
                const size_t p = ((size_t)it.slot * nkv + g) * R + rr;
                if (d == 0) a.ml[p] = make_float2(mm, ll);
                *reinterpret_cast<float4*>(a.part + p * HD + d) = x4;
            } else {
                const float inv = ll == 0.f ? 0.f : 1.0f / ll;  // (no row exists: zeros)
                const int rt = (int)a.over_group((uint32_t)rr);
                const size_t head = (size_t)(it.first + i0 + rt) * a.nh + g * group + (rr - rt * (int)group);
                *reinterpret_cast<float4*>(a.att + head * HD + d) =
                    make_float4(x4.x * inv, x4.y * inv, x4.z * inv, x4.w * inv);
            }
        }
        }
        if (x >= x1) return;
        // the item's next tile
        while (r_unit >= plan.units(seq)) {
            r_unit = 0;
            if (++it.s >= a.pg.n_seq) return;  // (the line ends with the last sequence)
            seq = plan.seq(it.s);
        }
        __syncthreads();
    }
}

// att from the parts of the tiles that were cut: a workgroup takes 8 rows of a
// tile and kv head, a thread four dims of a row, and where there are fewer rows
// every `lanes`-th part.  A tile is found at its first cut, the start of item i,
// where that item left word of it (the plan made again here took 0.3 to 0.9 us
// more).  Bound by its launch and two loads in a row: 3.8 us after one token at
// 700 rows, 4.4 us after 27 drafted ones at 8,192 (8 MB of parts).
constexpr int kMergeRows = 8, kMergeThreads = 256;
template <int HD, int R>
__global__ __launch_bounds__(kMergeThreads) void attention_paged_merge_kernel(AttnPagedArgs a) {
    constexpr int AHEAD = 8;
    __shared__ float4 acc[kMergeThreads];
    __shared__ float2 st[kMergeThreads];
    const uint32_t nkv = (uint32_t)a.pg.nkv, group = a.group;
    const uint32_t rb = blockIdx.y, g = blockIdx.x, item = blockIdx.z + 1;
    const int4 cut = a.cuts[item];
    const int rows = min(cut.y - (int)rb * kMergeRows, kMergeRows), parts = cut.z;  // of items item - 1, item, ...
    if (parts == 0 || rows <= 0) return;
    const auto slot = [&](int z) { return PagedLine::part_slot(item, (uint32_t)z); };
    const int tid = threadIdx.x, per = rows * (HD / 4), lanes = kMergeThreads / per;
    const int z0 = tid / per, u = tid - z0 * per, d = 4 * (u % (HD / 4)), row = (int)rb * kMergeRows + u / (HD / 4);
    float M = -INFINITY, L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto join = [&](float2 t, float4 v) __attribute__((always_inline)) {
        if (t.y == 0.f) return;  // (nothing attended there)
        const float m1 = fmaxf(M, t.x), a0 = __builtin_amdgcn_exp2f(M - m1), a1 = __builtin_amdgcn_exp2f(t.x - m1);
        M = m1;
        L = L * a0 + t.y * a1;
        s.x = s.x * a0 + v.x * a1, s.y = s.y * a0 + v.y * a1, s.z = s.z * a0 + v.z * a1, s.w = s.w * a0 + v.w * a1;
    };
    if (z0 < lanes)
        for (int z = z0; z < parts; z += lanes * AHEAD) {
            float2 t[AHEAD];
            float4 v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const size_t p = ((size_t)slot(min(z + i * lanes, parts - 1)) * nkv + g) * R + row;
                t[i] = a.ml[p];
                v[i] = *reinterpret_cast<const float4*>(a.part + p * HD + d);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (z + i * lanes < parts) join(t[i], v[i]);
        }
    if (lanes > 1) {
        acc[tid] = s;
        st[tid] = make_float2(M, L);
        __syncthreads();
    }
    if (z0) return;
    for (int i = 1; i < lanes; ++i) join(st[tid + i * per], acc[tid + i * per]);
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const uint32_t tl = a.over_group((uint32_t)row);
    const size_t tok = (size_t)cut.x + tl;
    *reinterpret_cast<float4*>(a.att + (tok * a.nh + g * group + ((uint32_t)row - tl * group)) * HD + d) =
        make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
}

PagedSize paged_size(const PagedArgs& a, int nh) {
    return PagedSize{a.n_seq, a.n_tokens, (int64_t)a.table_ld << a.page_shift, a.nkv, nh / a.nkv, device_cus()};
}

template <int HD, int R>
int launch(const AttnPagedArgs& a, const PagedShape& sh, hipStream_t st) {
    static bool attr_set = false;  // above 64 KiB of LDS needs the opt-in, once per kernel
    if (!attr_set && lds_bytes(HD, R) > 65536) {
        if (hipFuncSetAttribute((const void*)attention_paged_kernel<HD, R>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds_bytes(HD, R)) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const unsigned nkv = (unsigned)a.pg.nkv, items = (unsigned)sh.items, y = std::min(items, 32768u);
    hipLaunchKernelGGL((attention_paged_kernel<HD, R>), dim3(nkv, y, (items + y - 1) / y), dim3(kThreads),
                       lds_bytes(HD, R), st, a);
    if (sh.target > 0)
        hipLaunchKernelGGL((attention_paged_merge_kernel<HD, R>), dim3(nkv, R / kMergeRows, (unsigned)sh.target - 1),
                           dim3(kMergeThreads), 0, st, a);
    return MXH_OK;
}

template <int HD>
int launch_hd(const AttnPagedArgs& a, const PagedShape& sh, hipStream_t st) {
    return sh.rows == 64 ? launch<HD, 64>(a, sh, st) : launch<HD, 16>(a, sh, st);
}

}  // namespace

size_t attention_paged_work_bytes(const PagedArgs& a, int nh, int hd) {
    const PagedShape s = paged_shape(paged_size(a, nh));
    return paged_work_bytes(s.rows, s.target, a.nkv, hd);
}

size_t attention_paged_work_bound(const PagedArgs& a, int nh, int hd) { return paged_work_bound(paged_size(a, nh), hd); }

int attention_paged_launch(const PagedArgs& a, const float* q, int nh, int hd, float* att, void* work, hipStream_t st) {
    const PagedShape s = paged_shape(paged_size(a, nh));
    float* part = static_cast<float*>(work);
    float2* ml = reinterpret_cast<float2*>(part + (size_t)2 * s.target * a.nkv * s.rows * hd);
    const uint32_t group = (uint32_t)(nh / a.nkv);
    int4* cuts = reinterpret_cast<int4*>(ml + (size_t)2 * s.target * a.nkv * s.rows);
    const AttnPagedArgs args{a, q, att, part, ml, cuts, nh, s.target, 1.4426950408889634f / sqrtf((float)hd),
                             group, (uint32_t)s.rows / group, (65536 + group - 1) / group};
    return hd == 32 ? launch_hd<32>(args, s, st) : hd == 64 ? launch_hd<64>(args, s, st) : launch_hd<128>(args, s, st);
}

}  // namespace mxh
