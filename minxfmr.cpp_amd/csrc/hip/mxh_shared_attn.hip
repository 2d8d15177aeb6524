// mxh_shared_attn.hip — attention of packed tokens over a paged K/V cache where
// sequences begin, group by group, with the same rows (include/minxfmr_hip.h:
// mxh_attention_shared).
//
// Softmax over two sets of keys is joined from each set's largest score m, sum l
// of 2^(score - m) and weighted sum o of V rows: with M = max(m1, m2) the result is
// (2^(m1 - M) o1 + 2^(m2 - M) o2) / (2^(m1 - M) l1 + 2^(m2 - M) l2).  So the rows of a
// group's prefix are attended by the tokens of all its sequences together, in
// tiles of up to 64 rows that read K and V once for all of them, and each
// sequence's own rows by its own tokens.
//
// Three kernels: one workgroup cuts the tiles of both kinds into items of about as
// many stages (the lengths are on the device), a workgroup an item and kv head
// leaves its part in the workspace, and the last joins each token's parts.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "mxh_internal.h"
#include "mxh_paged.h"
#include "mxh_paged_tile.h"
#include "mxh_shared_plan.h"

namespace mxh {

namespace {

struct SharedPlanArgs {
    PagedArgs pg;
    const int *group_start, *group_shared;
    int n_groups;
    SharedShape sh;
    uint32_t tokens_p, tokens_s;  // of a tile
    int2* counts;
    SharedItem* items;
    int4* records;  // [n_tokens][2]
};

// What the plan keeps in LDS: starts and lengths of the sequences, the groups' starts,
// rows in common and first sequences with tokens, tiles and stages of the runs, the
// sequences' groups
__host__ __device__ constexpr size_t plan_lds(int n_seq, int n_groups) {
    return sizeof(int) * ((size_t)4 * n_seq + (size_t)5 * n_groups + 3) + sizeof(int16_t) * n_seq;
}
constexpr int kPlanWaves = 16;

// Workgroup 0 writes the items, the others the records of tokens that no sequence
// may have.  A group's rows in common are whole pages, no more than any of its
// sequences with tokens has cached (group_start that falls or leaves the batch:
// no rows in common).  The lengths are read once, all at a time, and little code is
// written twice: it comes from memory as the one workgroup gets to it.  64 sequences
// 8 us, 9 before that.
__global__ __launch_bounds__(64 * kPlanWaves) void shared_plan_kernel(SharedPlanArgs a) {
    extern __shared__ int lds[];
    __shared__ unsigned long long sums[2][kPlanWaves];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
    if (blockIdx.x > 0) {
        const int t = (int)(blockIdx.x - 1) * threads + tid;
        if (t < a.pg.n_tokens) a.records[2 * t] = make_int4(0, 0, -1, 0);
        return;
    }
    const int ng = a.n_groups, ns = a.pg.n_seq, runs = ng + ns;
    int *start = lds, *cached = start + ns + 1, *gstart = cached + ns, *common = gstart + ng + 1,
        *lead = common + ng;
    uint32_t *base = (uint32_t*)(lead + ng), *stages = base + runs + 1;  // base: tiles, then items before the run's
    int16_t* group = (int16_t*)(stages + runs);
    const int64_t table_rows = (int64_t)a.pg.table_ld << a.pg.page_shift;
    const int page = ~((1 << a.pg.page_shift) - 1);
#pragma unroll 1
    for (int i = tid; i <= ns; i += threads) {
        start[i] = a.pg.start[i];
        if (i < ns) cached[i] = min(max(a.pg.cached[i], 0), 1 << 30);
        if (i <= ng && ng > 0) gstart[i] = a.group_start[i];  // (no more groups than sequences)
        if (i < ng) common[i] = (int)min((int64_t)max(a.group_shared[i], 0), table_rows) & page, lead[i] = INT_MAX;
    }
    __syncthreads();
    int wrong = 0;  // 1: groups that make no sense, 2: starts that fall
#pragma unroll 1
    for (int i = tid; i < ns; i += threads) {
        if (i < ng && (gstart[i] < 0 || gstart[i + 1] > ns || gstart[i + 1] < gstart[i])) wrong |= 1;
        if (start[i + 1] < start[i]) wrong |= 2;
    }
    if (__syncthreads_or(wrong & 2)) {
        if (tid == 0) *a.counts = make_int2(0, 0);
        return;
    }
    const bool grouped = !__syncthreads_or(wrong) && ng > 0;
    const auto tokens_of = [&](int s) {
        const int n = start[s] < 0 ? 0 : max(min(start[s + 1], a.pg.n_tokens) - start[s], 0);
        return a.pg.parent ? min(n, kTreeMax) : n;
    };
#pragma unroll 1
    for (int s = tid; s < ns; s += threads) {
        int g = -1;
        if (grouped && s >= gstart[0] && s < gstart[ng]) {
            int hi = ng;  // gstart[g] <= s < gstart[hi]
            for (g = 0; hi - g > 1;) {
                const int mid = (g + hi) >> 1;
                if (gstart[mid] <= s) g = mid;
                else hi = mid;
            }
        }
        group[s] = (int16_t)g;
        if (g >= 0 && tokens_of(s) > 0) {
            atomicMin(&common[g], cached[s] & page);
            atomicMin(&lead[g], s);
        }
    }
    __syncthreads();
    unsigned long long units[2] = {0, 0};  // of prefixes, of own rows
#pragma unroll 1
    for (int r = tid; r < runs; r += threads) {
        int n = 0, keys = 0;
        if (r >= ng) {
            const int s = r - ng, g = group[s];
            n = tokens_of(s);
            keys = (int)min((int64_t)cached[s] + n, table_rows) - (g >= 0 && n > 0 ? common[g] : 0);
        } else if (grouped && lead[r] != INT_MAX && common[r] > 0) {  // the tokens of all the group's sequences
            n = max(min(start[gstart[r + 1]], a.pg.n_tokens) - max(start[gstart[r]], 0), 0);
            keys = common[r];
        }
        const SharedRun x = shared_run((uint32_t)n, (uint32_t)keys, r < ng ? a.sh.rows_p : a.sh.rows_s,
                                       r < ng ? a.tokens_p : a.tokens_s);
        base[r] = x.tiles, stages[r] = x.stages;
        units[r >= ng] += x.units();
    }
#pragma unroll 1
    for (int off = 32; off > 0; off >>= 1) {
        units[0] += __shfl_xor(units[0], off);
        units[1] += __shfl_xor(units[1], off);
    }
    if (lane == 0) sums[0][wave] = units[0], sums[1][wave] = units[1];
    __syncthreads();
    units[0] = units[1] = 0;
#pragma unroll 1
    for (int w = 0; w < waves; ++w) units[0] += sums[0][w], units[1] += sums[1][w];
    const uint32_t per_p = shared_per(units[0], a.sh.target_p), per_s = shared_per(units[1], a.sh.target_s);
    __syncthreads();
    // items before each run's: a thread has the runs [tid part, (tid + 1) part)
    const int part = (runs + threads - 1) / threads, r0 = min(tid * part, runs), r1 = min(r0 + part, runs);
    const auto count = [&](int r) { return base[r] * SharedRun{base[r], stages[r]}.parts(r < ng ? per_p : per_s); };
    uint32_t mine = 0;
#pragma unroll 1
    for (int r = r0; r < r1; ++r) mine += count(r);
    uint32_t at = wave_scan(mine);
    if (lane == 63) sums[0][wave] = at;
    at -= mine;
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < wave; ++w) at += (uint32_t)sums[0][w];
#pragma unroll 1
    for (int r = r0; r < r1; ++r) {
        const uint32_t n = count(r);
        base[r] = at;
        at += n;
    }
    if (r0 < runs && r1 == runs) base[runs] = at;
    __syncthreads();
    const uint32_t total_p = base[ng], total = base[runs];
    if (tid == 0) *a.counts = make_int2((int)total_p, (int)total);
#pragma unroll 1
    for (uint32_t i = (uint32_t)tid; i < total; i += threads) {
        int r = 0, hi = runs;  // base[r] <= i < base[hi]
#pragma unroll 1
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if (base[mid] <= i) r = mid;
            else hi = mid;
        }
        const bool own = r >= ng;
        SharedItem it;
        it.begin = 0;
        if (own) {
            const int s = r - ng, g = group[s];
            it.s = s, it.first = start[s], it.n = tokens_of(s), it.cached = cached[s];
            if (g >= 0) it.begin = common[g];
        } else {
            it.s = lead[r], it.first = max(start[gstart[r]], 0), it.cached = common[r];
            it.n = max(min(start[gstart[r + 1]], a.pg.n_tokens) - it.first, 0);
        }
        const uint32_t t = own ? a.tokens_s : a.tokens_p, per = own ? per_s : per_p;
        const SharedRun x{((uint32_t)it.n + t - 1) / t, stages[r]};
        const uint32_t len = x.length(per), local = i - base[r];
        // (the tiles of a part next to one another: they read the same rows)
        const uint32_t z = local / x.tiles, tile = local - z * x.tiles;
        it.tile = (int)tile, it.parts = (int)x.parts(per), it.stride = (int)x.tiles;
        it.st0 = (int)(z * len), it.st1 = (int)min((z + 1) * len, x.stages);
        const uint32_t kind = own ? total_p : 0;
        it.slot0 = (int)(base[r] + tile - kind), it.slot = (int)(i - kind);
        if (own && it.begin == 0 && it.parts == 1) it.slot = -1;  // (nothing to join)
        a.items[i] = it;
    }
}

struct SharedArgs {
    TileArgs t;  // (part and ml: the prefixes')
    float* part_s;
    float2* ml_s;
    const int2* counts;
    const SharedItem* items;
    int4* records;
};

template <int HD, int RP, int RS>
__global__ __launch_bounds__(kThreads, 2) void attention_shared_kernel(SharedArgs a) {
    extern __shared__ __align__(256) uint8_t smem[];
    const int tid = threadIdx.x;
    const uint32_t index = blockIdx.y + gridDim.y * blockIdx.z, g = blockIdx.x;
    const int2 counts = *a.counts;
    if (index >= (uint32_t)counts.y) return;
    const SharedItem x = a.items[index];
    SegmentOf it;
    it.s = x.s, it.first = (uint32_t)x.first, it.n = (uint32_t)x.n, it.cached = (uint32_t)x.cached;
    it.tile = (uint32_t)x.tile, it.st0 = (uint32_t)x.st0, it.st1 = (uint32_t)x.st1, it.slot = x.slot;
    it.begin = (uint32_t)x.begin;
    TileArgs t = a.t;
    const bool is_prefix = index < (uint32_t)counts.x;
    t.tokens = is_prefix ? RP / t.group : RS / t.group;
    if (g == 0 && x.st0 == 0) {  // where the tile's tokens find their parts
        const int i0 = x.tile * (int)t.tokens, n = min((int)t.tokens, x.n - i0);
        if (x.slot0 == x.slot || x.slot < 0)
            for (int i = tid; i < n; i += kThreads) {
                int4* rec = a.records + 2 * (size_t)(x.first + i0 + i);
                rec[is_prefix] = make_int4(x.slot0, x.stride, x.slot < 0 ? 0 : x.parts, i * (int)t.group);
                if (!is_prefix && x.begin == 0) rec[1] = make_int4(0, 0, 0, 0);
            }
    }
    if (is_prefix) {
        attend_tile<HD, RP, kPrefix>(t, it, g, false, smem);
    } else {
        t.part = a.part_s, t.ml = a.ml_s;
        attend_tile<HD, RS, kOwnRows>(t, it, g, false, smem);
    }
}

struct SharedMergeArgs {
    const int4* records;
    const float *part_p, *part_s;
    const float2 *ml_p, *ml_s;
    float* att;
    int64_t total;  // units of four dims, of all tokens
    int nkv, group, rows_p, rows_s;
};

// att from each token's parts
template <int HD, int LANES>
__global__ __launch_bounds__(kJoinThreads) void shared_merge_kernel(SharedMergeArgs a) {
    constexpr int UNITS = kJoinThreads / LANES;
    const int64_t u = (int64_t)blockIdx.x * UNITS + threadIdx.x % UNITS;
    const int64_t head = min(u, a.total - 1) / (HD / 4);
    const int d = 4 * (int)(u % (HD / 4)), nh = a.nkv * a.group;
    const int64_t t = head / nh;
    const int hq = (int)(head - t * nh), g = hq / a.group, hg = hq - g * a.group;
    const int4 own = a.records[2 * t], pre = a.records[2 * t + 1];
    const bool any = u < a.total && own.z >= 0 && own.z + pre.z > 0;  // (else: no sequence's, or done)
    const auto where = [&](int z, float2& x, float4& v) __attribute__((always_inline)) {
        const bool p = z < pre.z;
        const int64_t slot = p ? pre.x + (int64_t)z * pre.y : own.x + (int64_t)(z - pre.z) * own.y;
        const int64_t at = (slot * a.nkv + g) * (p ? a.rows_p : a.rows_s) + (p ? pre.w : own.w) + hg;
        x = (p ? a.ml_p : a.ml_s)[at];
        v = *reinterpret_cast<const float4*>((p ? a.part_p : a.part_s) + at * HD + d);
    };
    join_parts<LANES>(own.z + pre.z, where, any ? a.att + head * HD + d : nullptr);
}

PagedSize shared_size(const PagedArgs& a, int nh) {
    return PagedSize{a.n_seq, a.n_tokens, (int64_t)a.table_ld << a.page_shift, a.nkv, nh / a.nkv, device_cus()};
}

template <int HD, int RP, int RS>
int launch(const SharedArgs& a, const SharedShape& sh, hipStream_t st) {
    constexpr int LDS = lds_bytes(HD, RP) > lds_bytes(HD, RS) ? lds_bytes(HD, RP) : lds_bytes(HD, RS);
    static bool attr_set = false;  // above 64 KiB of LDS needs the opt-in, once per kernel
    if (!attr_set && LDS > 65536) {
        if (hipFuncSetAttribute((const void*)attention_shared_kernel<HD, RP, RS>,
                                hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const unsigned items = (unsigned)(sh.items_p + sh.items_s), y = std::min(items, 32768u);
    hipLaunchKernelGGL((attention_shared_kernel<HD, RP, RS>),
                       dim3((unsigned)a.t.pg.nkv, y, (items + y - 1) / y), dim3(kThreads), LDS, st, a);
    return MXH_OK;
}

template <int HD>
int launch_hd(const SharedArgs& a, const SharedShape& sh, hipStream_t st) {
    const int rc = sh.rows_s == 64   ? launch<HD, 64, 64>(a, sh, st)
                   : sh.rows_p == 64 ? launch<HD, 64, 16>(a, sh, st)
                                     : launch<HD, 16, 16>(a, sh, st);
    if (rc) return rc;
    const int64_t total = (int64_t)a.t.pg.n_tokens * a.t.nh() * (HD / 4);
    const int lanes = join_lanes(total, device_cus());
    const dim3 grid((unsigned)((total + kJoinThreads / lanes - 1) / (kJoinThreads / lanes)));
    const SharedMergeArgs m{a.records, a.t.part, a.part_s, a.t.ml, a.ml_s, a.t.att, total, a.t.pg.nkv,
                            (int)a.t.group, sh.rows_p, sh.rows_s};
    if (lanes == 1) hipLaunchKernelGGL((shared_merge_kernel<HD, 1>), grid, dim3(kJoinThreads), 0, st, m);
    else hipLaunchKernelGGL((shared_merge_kernel<HD, 4>), grid, dim3(kJoinThreads), 0, st, m);
    return MXH_OK;
}

}  // namespace

size_t attention_shared_work_bytes(const PagedArgs& a, int n_groups, int nh, int hd) {
    const PagedSize size = shared_size(a, nh);
    if (!shared_pays(size, hd, n_groups)) return attention_paged_work_bytes(a, nh, hd);
    return shared_work(shared_shape(size, n_groups), a.n_tokens, a.nkv, hd).bytes;
}

size_t attention_shared_work_bound(const PagedArgs& a, int n_groups, int nh, int hd) {
    const PagedSize size = shared_size(a, nh);
    const size_t paged = attention_paged_work_bound(a, nh, hd);
    // (fewer tokens may pay where these do not; fewer sequences or groups do not)
    if (!shared_pays(PagedSize{size.n_seq, 1, size.table_rows, size.nkv, size.group, size.cus}, hd, n_groups)) return paged;
    return std::max(paged, shared_work(shared_bound(size, n_groups), shared_bound(size, a.n_seq), shared_tokens(size),
                                       a.nkv, hd).bytes);
}

int attention_shared_launch(const PagedArgs& a, int n_groups, const int* group_start, const int* group_shared,
                            const float* q, int nh, int hd, float* att, void* work, hipStream_t st) {
    if (!shared_pays(shared_size(a, nh), hd, n_groups)) return attention_paged_launch(a, q, nh, hd, att, work, st);
    const SharedShape sh = shared_shape(shared_size(a, nh), n_groups);
    const SharedWork w = shared_work(sh, a.n_tokens, a.nkv, hd);
    const uint32_t group = (uint32_t)(nh / a.nkv);
    uint8_t* at = static_cast<uint8_t*>(work);
    const SharedPlanArgs plan{a, group_start, group_shared, n_groups, sh, (uint32_t)sh.rows_p / group,
                              (uint32_t)sh.rows_s / group, reinterpret_cast<int2*>(at),
                              reinterpret_cast<SharedItem*>(at + w.items), reinterpret_cast<int4*>(at + w.records)};
    static bool attr_set = false;
    if (!attr_set) {
        if (hipFuncSetAttribute((const void*)shared_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)plan_lds(kPagedSeqMax, kPagedSeqMax)) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const unsigned threads = a.n_seq + n_groups > 512 ? 64 * kPlanWaves : 256;
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1 + ((unsigned)a.n_tokens + threads - 1) / threads), dim3(threads),
                       plan_lds(a.n_seq, n_groups), st, plan);
    const SharedArgs args{{a, q, att, reinterpret_cast<float*>(at + w.part_p), reinterpret_cast<float2*>(at + w.ml_p),
                           1.4426950408889634f / sqrtf((float)hd), group, 0, (65536 + group - 1) / group},
                          reinterpret_cast<float*>(at + w.part_s),
                          reinterpret_cast<float2*>(at + w.ml_s),
                          plan.counts,
                          plan.items,
                          plan.records};
    return hd == 32 ? launch_hd<32>(args, sh, st) : hd == 64 ? launch_hd<64>(args, sh, st) : launch_hd<128>(args, sh, st);
}

}  // namespace mxh
