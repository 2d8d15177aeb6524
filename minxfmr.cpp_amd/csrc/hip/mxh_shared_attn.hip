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

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* s) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) v += s[w];
    __syncthreads();
    return v;
}

// Workgroup 0 writes the items, the others the records of tokens that no sequence
// may have.  A group's rows in common are whole pages, no more than any of its
// sequences with tokens has cached (group_start that falls or leaves the batch:
// no rows in common).
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedPlanArgs a) {
    extern __shared__ int lds[];
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        const int t = (int)(blockIdx.x - 1) * kPlanThreads + tid;
        if (t < a.pg.n_tokens) a.records[2 * t] = make_int4(0, 0, -1, 0);
        return;
    }
    __shared__ uint64_t sums[kPlanThreads / 64];
    const int ng = a.n_groups, ns = a.pg.n_seq, runs = ng + ns;
    int *gstart = lds, *common = gstart + ng + 1, *lead = common + ng;  // lead: the group's first sequence with tokens
    uint32_t* base = (uint32_t*)(lead + ng);                            // items before the run's
    const int64_t table_rows = (int64_t)a.pg.table_ld << a.pg.page_shift;
    const int page = ~((1 << a.pg.page_shift) - 1);
    bool bad = false;
    for (int g = tid; g <= ng && ng > 0; g += kPlanThreads) {
        const int at = a.group_start[g];
        bad |= at < 0 || at > ns || (g < ng && a.group_start[g + 1] < at);
        gstart[g] = at;
        if (g < ng) common[g] = (int)min((int64_t)max(a.group_shared[g], 0), table_rows) & page, lead[g] = INT_MAX;
    }
    const bool grouped = ng > 0 && !__syncthreads_or(bad);
    const auto group_of = [&](int s) {  // -1: none
        if (!grouped || s < gstart[0] || s >= gstart[ng]) return -1;
        int lo = 0, hi = ng;  // gstart[lo] <= s < gstart[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (gstart[mid] <= s) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    PagedLine line(a.sh.rows_s, a.tokens_s, a.pg.parent != nullptr, 0);
    const auto seq = [&](int s) {
        return line.seq(a.pg.start[s], a.pg.start[s + 1], a.pg.cached[s], a.pg.n_tokens, (uint64_t)table_rows);
    };
    bool falls = false;
    for (int s = tid; s < ns; s += kPlanThreads) {
        const PagedSeq q = seq(s);
        falls |= a.pg.start[s + 1] < a.pg.start[s];
        const int g = group_of(s);
        if (q.n > 0 && g >= 0) {
            atomicMin(&common[g], (int)q.cached & page);
            atomicMin(&lead[g], s);
        }
    }
    if (__syncthreads_or(falls)) {
        if (tid == 0) *a.counts = make_int2(0, 0);
        return;
    }
    // (a group's tokens: those of all its sequences)
    const auto prefix = [&](int g, int& first, int& n) {
        first = max(a.pg.start[gstart[g]], 0);
        n = max(min(a.pg.start[gstart[g + 1]], a.pg.n_tokens) - first, 0);
    };
    const auto run = [&](int r) {
        if (r < ng) {
            int first, n;
            if (!grouped || lead[r] == INT_MAX || common[r] == 0) return SharedRun{0, 0};
            prefix(r, first, n);
            return shared_run((uint32_t)n, (uint32_t)common[r], a.sh.rows_p, a.tokens_p);
        }
        const PagedSeq q = seq(r - ng);
        const int g = group_of(r - ng);
        const uint32_t rows = (uint32_t)min((int64_t)q.cached + q.n, table_rows);
        return shared_run(q.n, rows - (uint32_t)(g >= 0 && q.n > 0 ? common[g] : 0), a.sh.rows_s, a.tokens_s);
    };
    uint64_t units = 0;
    for (int r = tid; r < runs; r += kPlanThreads) units += run(r).units();
    const uint32_t per = shared_per(block_sum(units, sums), a.sh.target);
    // items before each run's: a thread has the runs [tid part, (tid + 1) part)
    const int part = (runs + kPlanThreads - 1) / kPlanThreads, r0 = min(tid * part, runs), r1 = min(r0 + part, runs);
    uint32_t mine = 0;
    for (int r = r0; r < r1; ++r) {
        const SharedRun x = run(r);
        mine += x.tiles * x.parts(per);
    }
    uint32_t upto = mine;
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t v = (uint32_t)__shfl_up((int)upto, off);
        if ((tid & 63) >= off) upto += v;
    }
    if ((tid & 63) == 63) sums[tid >> 6] = upto;
    __syncthreads();
    uint32_t total = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < tid >> 6) upto += (uint32_t)sums[w];
        total += (uint32_t)sums[w];
    }
    uint32_t at = upto - mine;
    for (int r = r0; r < r1; ++r) {
        const SharedRun x = run(r);
        base[r] = at;
        at += x.tiles * x.parts(per);
    }
    if (tid == 0) base[runs] = total;
    __syncthreads();
    const uint32_t total_p = base[ng];
    if (tid == 0) *a.counts = make_int2((int)total_p, (int)total);
    for (uint32_t i = (uint32_t)tid; i < total; i += kPlanThreads) {
        int lo = 0, hi = runs;  // base[lo] <= i < base[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (base[mid] <= i) lo = mid;
            else hi = mid;
        }
        const SharedRun x = run(lo);
        const uint32_t local = i - base[lo], parts = x.parts(per);
        // (the tiles of a part next to one another: they read the same rows)
        const uint32_t z = local / x.tiles, tile = local - z * x.tiles;
        SharedItem it;
        it.tile = (int)tile, it.begin = 0;
        it.st0 = (int)((uint64_t)x.stages * z / parts), it.st1 = (int)((uint64_t)x.stages * (z + 1) / parts);
        it.parts = (int)parts, it.stride = (int)x.tiles;
        it.slot0 = (int)(base[lo] + tile), it.slot = (int)i;
        if (lo < ng) {
            it.s = lead[lo], it.cached = common[lo];
            prefix(lo, it.first, it.n);
        } else {
            const PagedSeq q = seq(lo - ng);
            const int g = group_of(lo - ng);
            it.s = lo - ng, it.first = (int)q.first, it.n = (int)q.n, it.cached = (int)q.cached;
            it.begin = g >= 0 ? common[g] : 0;
            it.slot0 -= (int)total_p, it.slot -= (int)total_p;
            if (it.begin == 0 && parts == 1) it.slot = -1;  // (nothing to join)
        }
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
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), tid = threadIdx.x;
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
        attend_tile<HD, RP, kPrefix>(t, it, g, tid, wave, false, smem);
    } else {
        t.part = a.part_s, t.ml = a.ml_s;
        attend_tile<HD, RS, kOwnRows>(t, it, g, tid, wave, false, smem);
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
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void shared_merge_kernel(SharedMergeArgs a) {
    const int64_t u = (int64_t)blockIdx.x * kJoinUnits + threadIdx.x % kJoinUnits;
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
    join_parts(own.z + pre.z, where, any ? a.att + head * HD + d : nullptr);
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
    const int64_t total = (int64_t)a.t.pg.n_tokens * a.t.nh * (HD / 4), units = kJoinUnits;
    const SharedMergeArgs m{a.records, a.t.part, a.part_s, a.t.ml, a.ml_s, a.t.att, total, a.t.pg.nkv,
                            (int)a.t.group, sh.rows_p, sh.rows_s};
    hipLaunchKernelGGL(shared_merge_kernel<HD>, dim3((unsigned)((total + units - 1) / units)), dim3(kJoinThreads), 0,
                       st, m);
    return MXH_OK;
}

}  // namespace

size_t attention_shared_work_bytes(const PagedArgs& a, int n_groups, int nh, int hd) {
    return shared_work(shared_shape(shared_size(a, nh), n_groups), a.n_tokens, a.nkv, hd).bytes;
}

size_t attention_shared_work_bound(const PagedArgs& a, int n_groups, int nh, int hd) {
    const PagedSize size = shared_size(a, nh);
    return shared_work(shared_bound(size, n_groups), shared_bound(size, a.n_seq), a.n_tokens, a.nkv, hd).bytes;
}

int attention_shared_launch(const PagedArgs& a, int n_groups, const int* group_start, const int* group_shared,
                            const float* q, int nh, int hd, float* att, void* work, hipStream_t st) {
    const SharedShape sh = shared_shape(shared_size(a, nh), n_groups);
    const SharedWork w = shared_work(sh, a.n_tokens, a.nkv, hd);
    const uint32_t group = (uint32_t)(nh / a.nkv);
    uint8_t* at = static_cast<uint8_t*>(work);
    const SharedPlanArgs plan{a, group_start, group_shared, n_groups, sh, (uint32_t)sh.rows_p / group,
                              (uint32_t)sh.rows_s / group, reinterpret_cast<int2*>(at),
                              reinterpret_cast<SharedItem*>(at + w.items), reinterpret_cast<int4*>(at + w.records)};
    const size_t lds = sizeof(int) * ((size_t)4 * n_groups + a.n_seq + 2);
    static bool attr_set = false;
    if (!attr_set) {
        if (hipFuncSetAttribute((const void*)shared_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(int) * (5 * kPagedSeqMax + 2)) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1 + (unsigned)((a.n_tokens + kPlanThreads - 1) / kPlanThreads)),
                       dim3(kPlanThreads), lds, st, plan);
    const SharedArgs args{{a, q, att, reinterpret_cast<float*>(at + w.part_p), reinterpret_cast<float2*>(at + w.ml_p),
                           nh, 1.4426950408889634f / sqrtf((float)hd), group, 0, (65536 + group - 1) / group},
                          reinterpret_cast<float*>(at + w.part_s),
                          reinterpret_cast<float2*>(at + w.ml_s),
                          plan.counts,
                          plan.items,
                          plan.records};
    return hd == 32 ? launch_hd<32>(args, sh, st) : hd == 64 ? launch_hd<64>(args, sh, st) : launch_hd<128>(args, sh, st);
}

}  // namespace mxh
