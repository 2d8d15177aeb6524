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
// end leaves at once.  What a workgroup does of a tile is in mxh_paged_tile.h.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "mxh_attn.h"
#include "mxh_internal.h"
#include "mxh_paged.h"
#include "mxh_paged_tile.h"

namespace mxh {

namespace {

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

struct AttnPagedArgs : TileArgs {  // (slots: 2 target)
    int4* cuts;  // [target]: of the tile that is cut first where item i starts, its first token, rows, parts (0: none)
    int target;  // items that stages are cut into, at most; 0: an item is a tile
};
// the workgroup's item: the grid is (kv heads, items, more of them)
__device__ __forceinline__ uint32_t item_index() { return blockIdx.y + gridDim.y * blockIdx.z; }

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
    extern __shared__ __align__(256) uint8_t smem[];
    const uint32_t nkv = (uint32_t)a.pg.nkv, group = a.group, T = a.tokens;
    const uint32_t index = item_index(), g = blockIdx.x;
    const Plan plan(a.pg, R, T, a.target);
    uint32_t x = plan.first_unit(index);
    const bool tells = g == 0 && index < (uint32_t)a.target;  // (the second kernel; thread 0)
    if (x >= plan.total) {
        if (tells && threadIdx.x == 0) a.cuts[index] = make_int4(0, 0, 0, 0);
        return;
    }
    const uint32_t x0 = x, x1 = min(x + plan.per, plan.total);
    PagedSeq seq;
    uint32_t r_unit = x;
    Segment it;
    it.s = plan.find(r_unit, seq);
    for (;;) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // (as in attend_tile)
        {
            const Plan::Spot spot = plan.spot(seq, r_unit);
            const PagedPiece p = plan.piece(seq, spot, x1 - x, index);
            it.first = seq.first, it.n = seq.n, it.cached = seq.cached;
            it.tile = p.tile, it.st0 = p.st0, it.st1 = p.st1, it.slot = p.slot;
            if (tells && tid == 0 && x == x0) {
                const int i0 = (int)(spot.tile * T), rows = min((int)T, (int)seq.n - i0) * (int)group;
                a.cuts[index] = make_int4((int)seq.first + i0, rows, (int)plan.parts(spot), 0);
            }
            x += p.len, r_unit += p.len;
        }
        if (it.st0 < it.st1 || it.slot < 0) {  // (else only units of the lead)
            const bool unshared =
                seq.tiles == 1 && (float)plan.all * (float)(stage_keys(R) * 4 * HD) * (float)nkv > 256e6f;
            attend_tile<HD, R, kSequence>(a, it, g, unshared, smem);
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
    *reinterpret_cast<float4*>(a.att + (tok * a.nh() + g * group + ((uint32_t)row - tl * group)) * HD + d) =
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
    const AttnPagedArgs args{{a, q, att, part, ml, 1.4426950408889634f / sqrtf((float)hd), group,
                              (uint32_t)s.rows / group, (65536 + group - 1) / group},
                             cuts,
                             s.target};
    return hd == 32 ? launch_hd<32>(args, s, st) : hd == 64 ? launch_hd<64>(args, s, st) : launch_hd<128>(args, s, st);
}

}  // namespace mxh
