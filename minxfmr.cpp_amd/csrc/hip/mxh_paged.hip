// mxh_paged.hip — what fills and moves the rows of a paged K/V cache, and the
// C ABI of everything that works on one (include/minxfmr_hip.h).
//
// qk_rope_append: per token the reference layer's bias, (Qwen3) per-head
// rmsnorm and RoPE (transformer.cpp:189-214, rope.cpp:6-57), with the values
// of head_prep in mxh_layer.hip, then the cache append (kv_cache.cpp:50-75).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <new>
#include <vector>

#include "../host/mxh_pages.h"
#include "mxh_device.h"
#include "mxh_internal.h"
#include "mxh_paged.h"

namespace mxh {

namespace {

struct RopeArgs {
    PagedArgs pg;
    const float *qkv, *bias, *q_norm, *k_norm;
    const double* inv_freq;
    float* q;
    int64_t ld;
    float eps;
    int neox, nh;
};

// sum over aligned groups of LPH (4, 8 or 16) lanes, in every lane
template <int LPH>
__device__ __forceinline__ double head_sum(double v) {
    v += dpp_d<0xb1>(v);
    v += dpp_d<0x4e>(v);
    if constexpr (LPH >= 8) v += dpp_d<0x141>(v);
    if constexpr (LPH >= 16) v += dpp_d<0x140>(v);
    return v;
}

// One workgroup per token.  HD / 8 lanes hold a head, lane j its dims
// 4 j .. +4 and HD / 2 + 4 j .. +4: whole 16-byte pieces either way, and both
// halves of every pair in one lane for either pairing.  Wave 0 finds the
// token's place and turns the angles (one pair a lane) while the first heads'
// loads are in flight; from there on a lane works on one head with the next two
// on their way, in few registers, so that six workgroups fit a CU.  Bound by its
// bytes: 6,410 tokens of 32/8 heads of 128, both norms, 59 us = 4.9 TB/s read
// and written; four heads unrolled held 201 registers, so two workgroups a CU,
// and took 90.  One token takes 5 us, little over an empty launch.
constexpr int kRopeThreads = 256;

template <int HD>
__global__ __launch_bounds__(kRopeThreads, 6) void qk_rope_append_kernel(RopeArgs a) {
    constexpr int LPH = HD / 8, STEP = kRopeThreads / LPH;  // heads per pass over the workgroup
    __shared__ double2 cs[HD / 2];
    __shared__ int64_t place;  // the token's cache row, -1: none; -2: the token is no sequence's
    const int tid = threadIdx.x, j = tid % LPH;
    const int nkv = a.pg.nkv, heads = a.nh + 2 * nkv, t = blockIdx.x;
    const int d0 = 4 * j, d1 = HD / 2 + 4 * j;
    const float* row = a.qkv + (size_t)t * a.ld;
    struct Head {
        float4 lo, hi;
    };
    const auto load = [&](int h) __attribute__((always_inline)) {  // (past the last head: the last again, unused)
        const float* p = row + (size_t)min(h, heads - 1) * HD;
        return Head{*reinterpret_cast<const float4*>(p + d0), *reinterpret_cast<const float4*>(p + d1)};
    };
    Head cur = load(tid / LPH), next = load(tid / LPH + STEP);
    if (tid < 64) {
        const int s = paged_seq_of(a.pg, t);
        int64_t at = -2;
        int pos = 0;
        if (s >= 0) {
            const int first = a.pg.start[s], i = t - first;
            const int cached = min(max(a.pg.cached[s], 0), 1 << 30);
            pos = cached + i;
            bool mine = true;
            if (a.pg.parent) {
                const int n = min(max(min(a.pg.start[s + 1], a.pg.n_tokens), first) - first, kTreeMax);
                const uint64_t path = tree_path(tree_parent(a.pg, first, n));
                pos = cached + __shfl((int)__popcll(path), i & 63) - 1;
                mine = i < kTreeMax;
            }
            if (mine) at = paged_row(a.pg, s, cached + i);
        }
        if (tid < HD / 2) {
            double sn, c;
            sincospi((double)pos * a.inv_freq[tid] * 0.31830988618379067154, &sn, &c);
            cs[tid] = make_double2(c, sn);
        }
        if (tid == 0) place = at;
    }
    __syncthreads();
    const int64_t at = place;
    if (at == -2) return;
    // the lane's pairs: of elements e and e + 4 (neox), or (0, 1), (2, 3) of both pieces
    double2 turn[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) turn[e] = cs[a.neox ? 4 * j + e : (e < 2 ? 2 * j + e : HD / 4 + 2 * j + e - 2)];
#pragma unroll 1
    for (int h = tid / LPH; h < heads; h += STEP) {  // (whole heads: their lanes stay together)
        float x[8] = {cur.lo.x, cur.lo.y, cur.lo.z, cur.lo.w, cur.hi.x, cur.hi.y, cur.hi.z, cur.hi.w};
        cur = next;
        next = load(h + 2 * STEP);
        if (a.bias) {
            const float4 b0 = *reinterpret_cast<const float4*>(a.bias + h * HD + d0);
            const float4 b1 = *reinterpret_cast<const float4*>(a.bias + h * HD + d1);
            x[0] += b0.x, x[1] += b0.y, x[2] += b0.z, x[3] += b0.w;
            x[4] += b1.x, x[5] += b1.y, x[6] += b1.z, x[7] += b1.w;
        }
        if (h < a.nh + nkv) {
            const float* w = h < a.nh ? a.q_norm : a.k_norm;
            if (w) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += (double)x[e] * x[e];
                const double inv = 1.0 / sqrt(head_sum<LPH>(ss) / (double)HD + (double)a.eps);
                const float4 w0 = *reinterpret_cast<const float4*>(w + d0);
                const float4 w1 = *reinterpret_cast<const float4*>(w + d1);
                const float g[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)((double)x[e] * inv) * g[e];
            }
            const auto rotate = [&](float& p, float& q, const double2& c) {
                const double x0 = p, x1 = q;
                p = (float)(x0 * c.x - x1 * c.y);
                q = (float)(x0 * c.y + x1 * c.x);
            };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (a.neox) rotate(x[e], x[e + 4], turn[e]);
                else rotate(x[2 * e], x[2 * e + 1], turn[e]);
            }
        }
        if (h < a.nh) {
            float* out = a.q + ((size_t)t * a.nh + h) * HD;
            *reinterpret_cast<float4*>(out + d0) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(out + d1) = make_float4(x[4], x[5], x[6], x[7]);
        } else if (at >= 0) {
            const int g = h - a.nh;
            __half* out = (g < nkv ? a.pg.k + ((size_t)at * nkv + g) * HD : a.pg.v + ((size_t)at * nkv + g - nkv) * HD);
            union {
                __half2 h2[4];
                uint2 u2[2];
            } o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.h2[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
            *reinterpret_cast<uint2*>(out + d0) = o.u2[0];
            *reinterpret_cast<uint2*>(out + d1) = o.u2[1];
        }
    }
}

// ---- moving rows ----------------------------------------------------------

// Lists travel in the kernel's arguments (at most 4 KiB of them): no copy to
// the device before the launch, and a recorded call holds its own.
constexpr int kCopyPairs = 448;
constexpr int kCopyThreads = 256;

struct CopyArgs {
    uint4 *k, *v;
    int64_t layer16;         // 16-byte pieces from a layer to the next
    int page16, chunks;      // pieces of a page; workgroups per page
    int src[kCopyPairs], dst[kCopyPairs];
};

typedef uint32_t piece __attribute__((ext_vector_type(4)));  // 16 bytes

// Workgroup (chunk and K or V, pair, layer): 4 KB, a 16-byte piece a thread.  Bound
// by its bytes; one page in 28 layers 5 us, little over an empty launch.  Two, four
// and eight pieces a thread, all in flight before its first store, took 235, 237 and
// 314 us for 256 pages of 16 rows of 8 heads of 128 in 36 layers (one 230), for 16
// pages 23.5, 24.7 and 28.7 (13.6).
// ONCE: copies larger than the 256 MB of the last cache do not fill it: 256 pages 216
// us = 5.6 TB/s; 16 pages whose rows it may hold 16.0 (13.8).
template <bool ONCE>
__global__ __launch_bounds__(kCopyThreads) void kv_copy_pages_kernel(CopyArgs a) {
    const int chunk = blockIdx.x >> 1, i = chunk * kCopyThreads + threadIdx.x;
    if (i >= a.page16) return;
    uint4* base = (blockIdx.x & 1 ? a.v : a.k) + blockIdx.z * a.layer16 + i;
    const piece* from = reinterpret_cast<const piece*>(base + (int64_t)a.src[blockIdx.y] * a.page16);
    piece* to = reinterpret_cast<piece*>(base + (int64_t)a.dst[blockIdx.y] * a.page16);
    if (ONCE) __builtin_nontemporal_store(__builtin_nontemporal_load(from), to);
    else *to = *from;
}

// A move is 16 bits for the row it reads and 16 for the one it writes: 6 for
// one of its sequence's pages, 10 for the row of the page.
constexpr int kMoves = 480, kKeepPages = 300, kKeepGroups = 190, kKeepSlots = 64;
struct KeepArgs {
    uint4 *k, *v;
    int64_t layer16;
    int row16, page_rows, columns;  // 16-byte pieces of a row; columns: of all layers' K and V rows together
    uint32_t moves[kMoves];
    int pages[kKeepPages];
    uint32_t group[kKeepGroups + 1];  // first move (up to the next group's) | first page << 16
};
static_assert(sizeof(KeepArgs) <= 4096 && sizeof(CopyArgs) <= 4096, "");

// A thread moves one 16-byte column of one sequence's rows.  The moves go in
// ascending order with dst <= src, so a row is written only after it was read
// (dst of a move is below the src of every later one), however many loads of
// later moves come before a store.  Bound by its bytes: 337 moved rows of 64
// sequences, 2 KB of K and of V in 36 layers, 18 us = 5.5 TB/s (20.4 with stores that
// fill the caches, 23.5 with such loads as well); four rows of one sequence 5.5 us,
// little over an empty launch.  (As an array the eight pieces went to scratch memory:
// 38 us, twice the bytes written.)
__global__ __launch_bounds__(256) void kv_keep_rows_kernel(KeepArgs a) {
    const int g = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;  // (the sequences of a layer next to each other)
    if (c >= a.columns) return;
    const int per = 2 * a.row16, layer = c / per, in = c - layer * per;
    piece* base = reinterpret_cast<piece*>((in < a.row16 ? a.k + in : a.v + in - a.row16) + layer * a.layer16);
    const int first = (int)(a.group[g] & 0xffff), end = (int)(a.group[g + 1] & 0xffff);
    const int* pages = a.pages + (a.group[g] >> 16);
    const auto at = [&](uint32_t code) {
        return ((int64_t)pages[code >> 10] * a.page_rows + (code & 1023)) * a.row16;
    };
    for (int m = first; m < end; m += 8) {
        // (past the end the last again: all loads are in flight at once)
        const auto get = [&](int u) { return base[at(a.moves[min(m + u, end - 1)] & 0xffff)]; };
        const auto put = [&](int u, piece x) {
            if (m + u < end) __builtin_nontemporal_store(x, base + at(a.moves[m + u] >> 16));
        };
        const piece x0 = get(0), x1 = get(1), x2 = get(2), x3 = get(3);
        const piece x4 = get(4), x5 = get(5), x6 = get(6), x7 = get(7);
        put(0, x0), put(1, x1), put(2, x2), put(3, x3), put(4, x4), put(5, x5), put(6, x6), put(7, x7);
    }
}

// ---- checks -----------------------------------------------------------------

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

int64_t layer_elems(const mxh_kv_pool* p) {
    return p->layer_stride ? p->layer_stride : (int64_t)p->n_pages * p->page_rows * p->n_kv * p->head_dim;
}

int check_pool(const char* who, const mxh_kv_pool* p) {
    if (!p) return set_error(MXH_ERR_ARG, "%s: null pool", who);
    if (!p->k || !p->v || !al16(p->k) || !al16(p->v))
        return set_error(MXH_ERR_ARG, "%s: k and v must be non-null and 16-byte aligned", who);
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128)
        return set_error(MXH_ERR_ARG, "%s: head_dim %d is not 32, 64 or 128", who, p->head_dim);
    if (p->page_rows < 16 || p->page_rows > 1024 || (p->page_rows & (p->page_rows - 1)))
        return set_error(MXH_ERR_ARG, "%s: page_rows %d is not a power of two from 16 to 1024", who, p->page_rows);
    if (p->n_layer < 1 || p->n_layer > 65535 || p->n_pages < 1 || p->n_kv < 1 || p->n_kv > 1024 ||
        (int64_t)p->n_layer * p->n_kv * p->head_dim > 65535 * 1024 ||  // (kv_keep_rows' grid)
        (int64_t)p->n_pages * p->page_rows > INT_MAX)
        return set_error(MXH_ERR_ARG, "%s: unsupported pool of %d layers, %d pages of %d rows, %d kv heads", who,
                         p->n_layer, p->n_pages, p->page_rows, p->n_kv);
    if (p->layer_stride && (p->layer_stride % 8 ||
                            p->layer_stride < (int64_t)p->n_pages * p->page_rows * p->n_kv * p->head_dim))
        return set_error(MXH_ERR_ARG, "%s: layer_stride %lld is less than a layer or no multiple of 8", who,
                         (long long)p->layer_stride);
    return MXH_OK;
}

// pool, layer, batch and heads of a per-layer call
int check_step(const char* who, const mxh_kv_pool* p, int layer, const mxh_kv_batch* b, int nh) {
    if (int rc = check_pool(who, p)) return rc;
    if (layer < 0 || layer >= p->n_layer)
        return set_error(MXH_ERR_ARG, "%s: layer %d of %d", who, layer, p->n_layer);
    if (nh < 1 || !attention_supported(nh, p->n_kv, p->head_dim))
        return set_error(MXH_ERR_ARG, "%s: unsupported heads: nh %d, n_kv %d, head_dim %d", who, nh, p->n_kv,
                         p->head_dim);
    if (!b) return set_error(MXH_ERR_ARG, "%s: null batch", who);
    if (b->n_seq < 0 || b->n_seq > kPagedSeqMax || b->n_tokens < 0 || b->n_tokens > 1 << 20)
        return set_error(MXH_ERR_ARG, "%s: %d sequences (0..%d) of %d tokens (0..%d)", who, b->n_seq, kPagedSeqMax,
                         b->n_tokens, 1 << 20);
    if (b->n_seq == 0 || b->n_tokens == 0) return MXH_OK;
    if (!b->start || !b->cached || !b->table || b->table_ld < 1)
        return set_error(MXH_ERR_ARG, "%s: the batch lacks start, cached or table", who);
    return MXH_OK;
}

PagedArgs paged_args(const mxh_kv_pool* p, int layer, const mxh_kv_batch* b) {
    PagedArgs a{};
    a.k = static_cast<__half*>(p->k) + layer * layer_elems(p);
    a.v = static_cast<__half*>(p->v) + layer * layer_elems(p);
    a.start = b->start, a.cached = b->cached, a.table = b->table, a.parent = b->parent;
    a.n_seq = b->n_seq, a.n_tokens = b->n_tokens, a.table_ld = b->table_ld, a.n_pages = p->n_pages;
    a.page_shift = __builtin_ctz((unsigned)p->page_rows), a.nkv = p->n_kv;
    return a;
}

// marks ids (a bit a page); false where one is marked already
bool mark_pages(const int* ids, int n, std::vector<uint64_t>& seen) {
    for (int i = 0; i < n; ++i) {
        uint64_t& w = seen[(size_t)ids[i] >> 6];
        const uint64_t bit = 1ull << (ids[i] & 63);
        if (w & bit) return false;
        w |= bit;
    }
    return true;
}

// every fault of mxh_kv_keep_rows' lists; keep is read only where all of
// keep_start makes sense
int check_keep(const mxh_kv_pool* p, const int* table, int table_ld, const int* cached, const int* keep_start,
               const int* keep, int n_seq) {
    const char* who = "kv_keep_rows";
    const int pr = p->page_rows;
    if (keep_start[0] < 0) return set_error(MXH_ERR_ARG, "%s: keep_start begins at %d", who, keep_start[0]);
    for (int s = 0; s < n_seq; ++s)
        if (keep_start[s + 1] < keep_start[s])
            return set_error(MXH_ERR_ARG, "%s: keep_start decreases at sequence %d", who, s);
    if (!keep && keep_start[n_seq] > keep_start[0]) return set_error(MXH_ERR_ARG, "%s: null array", who);
    std::vector<int> pages;  // every page that holds a kept row, of all sequences
    for (int s = 0; s < n_seq; ++s) {
        const int n = keep_start[s + 1] - keep_start[s];
        if (n == 0) continue;
        const int* kept = keep + keep_start[s];
        if (kept[0] < 0) return set_error(MXH_ERR_ARG, "%s: sequence %d keeps token %d", who, s, kept[0]);
        for (int i = 1; i < n; ++i)
            if (kept[i] <= kept[i - 1])
                return set_error(MXH_ERR_ARG, "%s: the kept tokens of sequence %d do not ascend", who, s);
        if (cached[s] < 0 || (int64_t)cached[s] + kept[n - 1] >= std::min((int64_t)table_ld * pr, (int64_t)INT_MAX))
            return set_error(MXH_ERR_ARG, "%s: row %lld of sequence %d is past its table", who,
                             (long long)cached[s] + kept[n - 1], s);
        const int* ids = table + (size_t)s * table_ld;
        // the pages of the rows written, one after the other, then those of rows
        // that are only read
        int last = -1;
        for (int pass = 0; pass < 2; ++pass)
            for (int i = 0; i < n; ++i) {
                const int q = (cached[s] + (pass ? kept[i] : i)) / pr;
                if (q <= last) continue;
                last = q;
                if (ids[q] < 0 || ids[q] >= p->n_pages)
                    return set_error(MXH_ERR_ARG, "%s: page %d of sequence %d is %d, not in the pool", who, q, s,
                                     ids[q]);
                pages.push_back(ids[q]);
            }
    }
    std::sort(pages.begin(), pages.end());
    const auto twice = std::adjacent_find(pages.begin(), pages.end());
    if (twice != pages.end())
        return set_error(MXH_ERR_ARG, "%s: page %d holds kept rows of two places", who, *twice);
    return MXH_OK;
}

}  // namespace

}  // namespace mxh

using namespace mxh;

struct mxh_pages {
    PageBook book;
};

extern "C" {

int mxh_qk_rope_append(const mxh_kv_pool* pool, int layer, const mxh_kv_batch* batch, const float* qkv, int64_t ld,
                       const float* bias, const float* q_norm, const float* k_norm, float eps, const double* inv_freq,
                       int neox, int nh, float* q) {
    const char* who = "qk_rope_append";
    if (int rc = check_step(who, pool, layer, batch, nh)) return rc;
    if (batch->n_seq == 0 || batch->n_tokens == 0) return MXH_OK;
    const int64_t width = ((int64_t)nh + 2 * pool->n_kv) * pool->head_dim;
    if (!qkv || !q || !inv_freq || !al16(qkv) || !al16(q) || !al16(bias) || !al16(q_norm) || !al16(k_norm) ||
        ((uintptr_t)inv_freq & 7))
        return set_error(MXH_ERR_ARG, "%s: qkv, q and inv_freq must be non-null, every array aligned to 16 bytes", who);
    if (ld < width || ld % 4 || ld > INT_MAX)
        return set_error(MXH_ERR_ARG, "%s: ld %lld for rows of %lld floats", who, (long long)ld, (long long)width);
    if (!(eps >= 0.f)) return set_error(MXH_ERR_ARG, "%s: eps %g", who, (double)eps);
    if (overlap(qkv, sizeof(float) * (size_t)((batch->n_tokens - 1) * ld + width), q,
                sizeof(float) * (size_t)batch->n_tokens * nh * pool->head_dim))
        return set_error(MXH_ERR_ARG, "%s: q overlaps qkv", who);
    if (!mxh_is_available()) return MXH_ERR_NODEV;
    const RopeArgs a{paged_args(pool, layer, batch), qkv, bias, q_norm, k_norm, inv_freq, q, ld, eps, neox, nh};
    const dim3 grid((unsigned)batch->n_tokens), block(kRopeThreads);
    switch (pool->head_dim) {
    case 32: hipLaunchKernelGGL(qk_rope_append_kernel<32>, grid, block, 0, lib_stream(), a); break;
    case 64: hipLaunchKernelGGL(qk_rope_append_kernel<64>, grid, block, 0, lib_stream(), a); break;
    default: hipLaunchKernelGGL(qk_rope_append_kernel<128>, grid, block, 0, lib_stream(), a); break;
    }
    return check_hip(hipGetLastError(), "qk_rope_append launch");
}

int mxh_attention_paged_workspace(const mxh_kv_pool* pool, const mxh_kv_batch* batch, int nh, size_t* bytes) {
    if (!bytes) return set_error(MXH_ERR_ARG, "attention_paged_workspace: null output pointer");
    *bytes = 0;
    if (int rc = check_step("attention_paged_workspace", pool, 0, batch, nh)) return rc;
    if (batch->n_seq == 0 || batch->n_tokens == 0) return MXH_OK;
    if (!mxh_is_available()) return MXH_ERR_NODEV;
    *bytes = attention_paged_work_bound(paged_args(pool, 0, batch), nh, pool->head_dim);
    return MXH_OK;
}

int mxh_attention_paged(const mxh_kv_pool* pool, int layer, const mxh_kv_batch* batch, const float* q, int nh,
                        float* att, void* work, size_t work_bytes) {
    const char* who = "attention_paged";
    if (int rc = check_step(who, pool, layer, batch, nh)) return rc;
    if (batch->n_seq == 0 || batch->n_tokens == 0) return MXH_OK;
    if (!q || !att || !al16(q) || !al16(att) || !al16(work))
        return set_error(MXH_ERR_ARG, "%s: q and att must be non-null, every array aligned to 16 bytes", who);
    const size_t bytes = sizeof(float) * (size_t)batch->n_tokens * nh * pool->head_dim;
    if (overlap(q, bytes, att, bytes)) return set_error(MXH_ERR_ARG, "%s: att overlaps q", who);
    if (!mxh_is_available()) return MXH_ERR_NODEV;
    const PagedArgs a = paged_args(pool, layer, batch);
    const size_t need = attention_paged_work_bytes(a, nh, pool->head_dim);
    if (need && (!work || work_bytes < need))
        return set_error(MXH_ERR_ARG, "%s: %zu bytes of work, %zu needed", who, work ? work_bytes : 0, need);
    if (need && (overlap(work, need, q, bytes) || overlap(work, need, att, bytes)))
        return set_error(MXH_ERR_ARG, "%s: work overlaps q or att", who);
    if (int rc = attention_paged_launch(a, q, nh, pool->head_dim, att, work, lib_stream()))
        return set_error(rc, "%s: launch", who);
    return check_hip(hipGetLastError(), "attention_paged launch");
}

int mxh_kv_copy_pages(const mxh_kv_pool* pool, const int* src, const int* dst, int n) try {
    const char* who = "kv_copy_pages";
    if (int rc = check_pool(who, pool)) return rc;
    if (n < 0 || (n > 0 && (!src || !dst))) return set_error(MXH_ERR_ARG, "%s: bad list of %d pages", who, n);
    for (int i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= pool->n_pages || dst[i] < 0 || dst[i] >= pool->n_pages)
            return set_error(MXH_ERR_ARG, "%s: page %d to %d in a pool of %d", who, src[i], dst[i], pool->n_pages);
    std::vector<uint64_t> seen(((size_t)pool->n_pages + 63) / 64, 0);
    if (!mark_pages(dst, n, seen)) return set_error(MXH_ERR_ARG, "%s: a page is written twice", who);
    for (int i = 0; i < n; ++i)
        if (seen[(size_t)src[i] >> 6] >> (src[i] & 63) & 1)
            return set_error(MXH_ERR_ARG, "%s: page %d is read and written", who, src[i]);
    if (n == 0) return MXH_OK;
    if (!mxh_is_available()) return MXH_ERR_NODEV;
    CopyArgs a{};
    a.k = static_cast<uint4*>(pool->k), a.v = static_cast<uint4*>(pool->v);
    a.layer16 = layer_elems(pool) / 8;
    a.page16 = pool->page_rows * pool->n_kv * pool->head_dim / 8;
    a.chunks = (a.page16 + kCopyThreads - 1) / kCopyThreads;
    const bool once = 4.0 * 16 * a.page16 * n * pool->n_layer > 256e6;  // read and written, K and V
    for (int i = 0; i < n; i += kCopyPairs) {
        const int m = std::min(kCopyPairs, n - i);
        std::copy(src + i, src + i + m, a.src);
        std::copy(dst + i, dst + i + m, a.dst);
        const dim3 grid(2u * (unsigned)a.chunks, (unsigned)m, (unsigned)pool->n_layer);
        if (once) hipLaunchKernelGGL(kv_copy_pages_kernel<true>, grid, dim3(kCopyThreads), 0, lib_stream(), a);
        else hipLaunchKernelGGL(kv_copy_pages_kernel<false>, grid, dim3(kCopyThreads), 0, lib_stream(), a);
    }
    return check_hip(hipGetLastError(), "kv_copy_pages launch");
} catch (const std::bad_alloc&) {
    return set_error(MXH_ERR_OOM, "kv_copy_pages: out of host memory");
}

int mxh_kv_keep_rows(const mxh_kv_pool* pool, const int* table, int table_ld, const int* cached,
                     const int* keep_start, const int* keep, int n_seq) try {
    const char* who = "kv_keep_rows";
    if (int rc = check_pool(who, pool)) return rc;
    if (n_seq < 0 || n_seq > kPagedSeqMax) return set_error(MXH_ERR_ARG, "%s: %d sequences", who, n_seq);
    if (n_seq == 0) return MXH_OK;
    if (!table || table_ld < 1 || !cached || !keep_start)
        return set_error(MXH_ERR_ARG, "%s: null array", who);
    if (int rc = check_keep(pool, table, table_ld, cached, keep_start, keep, n_seq)) return rc;
    KeepArgs a{};
    a.k = static_cast<uint4*>(pool->k), a.v = static_cast<uint4*>(pool->v);
    a.layer16 = layer_elems(pool) / 8;
    a.row16 = pool->n_kv * pool->head_dim / 8, a.page_rows = pool->page_rows;
    a.columns = pool->n_layer * 2 * a.row16;
    int moves = 0, pages = 0, groups = 0;
    const auto flush = [&] {
        if (!groups) return;
        a.group[groups] = (uint32_t)moves;
        hipLaunchKernelGGL(kv_keep_rows_kernel, dim3((unsigned)groups, (unsigned)((a.columns + 255) / 256)), dim3(256),
                           0, lib_stream(), a);
        moves = pages = groups = 0;
    };
    bool ready = false;
    for (int s = 0; s < n_seq; ++s) {
        const int* ids = table + (size_t)s * table_ld;
        bool open = false;  // a group of this sequence, in the launch to come
        int page0 = 0, src_q = -1, dst_q = -1, src_slot = 0, dst_slot = 0;
        for (int i = 0; i < keep_start[s + 1] - keep_start[s]; ++i) {
            const int kept = keep[keep_start[s] + i];
            if (kept == i) continue;  // in place
            if (!ready && !mxh_is_available()) return MXH_ERR_NODEV;
            ready = true;
            // a sequence that does not fit goes on in another launch (in order, as
            // launches of a stream are), in a group of its own
            if (moves == kMoves || pages + 2 > kKeepPages ||
                (open ? pages - page0 + 2 > kKeepSlots : groups == kKeepGroups))
                flush(), open = false;
            if (!open) {
                open = true;
                a.group[groups] = (uint32_t)moves | (uint32_t)pages << 16;
                ++groups;
                page0 = pages, src_q = dst_q = -1;
            }
            const int from = cached[s] + kept, to = cached[s] + i, pr = pool->page_rows;
            if (to / pr != dst_q) dst_q = to / pr, dst_slot = pages - page0, a.pages[pages++] = ids[dst_q];
            if (from / pr == dst_q) src_q = dst_q, src_slot = dst_slot;
            if (from / pr != src_q) src_q = from / pr, src_slot = pages - page0, a.pages[pages++] = ids[src_q];
            a.moves[moves++] = (uint32_t)(src_slot << 10 | from % pr) | (uint32_t)(dst_slot << 10 | to % pr) << 16;
        }
    }
    if (!ready) return MXH_OK;
    flush();
    return check_hip(hipGetLastError(), "kv_keep_rows launch");
} catch (const std::bad_alloc&) {
    return set_error(MXH_ERR_OOM, "kv_keep_rows: out of host memory");
}

// ---- page bookkeeping ---------------------------------------------------------

int mxh_pages_create(int n_pages, int page_rows, int max_seqs, mxh_pages** out) try {
    if (!out) return set_error(MXH_ERR_ARG, "pages_create: null output pointer");
    *out = nullptr;
    if (n_pages < 1 || max_seqs < 1 || max_seqs > 1 << 20 || page_rows < 16 || page_rows > 1024 ||
        (page_rows & (page_rows - 1)) ||
        (int64_t)n_pages * page_rows > INT_MAX)
        return set_error(MXH_ERR_ARG, "pages_create: unsupported %d pages of %d rows for %d sequences", n_pages,
                         page_rows, max_seqs);
    *out = new mxh_pages{PageBook(n_pages, page_rows, max_seqs)};
    return MXH_OK;
} catch (const std::bad_alloc&) {
    return set_error(MXH_ERR_OOM, "pages_create: out of host memory");
}

void mxh_pages_destroy(mxh_pages* p) { delete p; }

static int check_seq(const char* who, const mxh_pages* p, int seq) {
    if (!p) return set_error(MXH_ERR_ARG, "%s: null pages", who);
    if (!p->book.valid(seq)) return set_error(MXH_ERR_ARG, "%s: no sequence %d", who, seq);
    return MXH_OK;
}

int mxh_pages_open(mxh_pages* p, int* seq) {
    if (!p || !seq) return set_error(MXH_ERR_ARG, "pages_open: null argument");
    *seq = p->book.open();
    return *seq >= 0 ? MXH_OK : set_error(MXH_ERR_OOM, "pages_open: every sequence id is in use");
}

int mxh_pages_fork(mxh_pages* p, int seq, int* child) try {
    if (!child) return set_error(MXH_ERR_ARG, "pages_fork: null output pointer");
    *child = -1;
    if (int rc = check_seq("pages_fork", p, seq)) return rc;
    *child = p->book.fork(seq);
    return *child >= 0 ? MXH_OK : set_error(MXH_ERR_OOM, "pages_fork: every sequence id is in use");
} catch (const std::bad_alloc&) {
    return set_error(MXH_ERR_OOM, "pages_fork: out of host memory");
}

int mxh_pages_close(mxh_pages* p, int seq) {
    if (int rc = check_seq("pages_close", p, seq)) return rc;
    p->book.close(seq);
    return MXH_OK;
}

int mxh_pages_extend(mxh_pages* p, int seq, int rows, int* src, int* dst, int* copies) try {
    if (!src || !dst || !copies) return set_error(MXH_ERR_ARG, "pages_extend: null output pointer");
    *copies = 0;
    if (int rc = check_seq("pages_extend", p, seq)) return rc;
    if (rows < 0 || rows > INT_MAX - p->book.length(seq))
        return set_error(MXH_ERR_ARG, "pages_extend: %d rows behind %d", rows, p->book.length(seq));
    if (!p->book.extend(seq, rows, src, dst))
        return set_error(MXH_ERR_OOM, "pages_extend: %d free pages do not hold %d more rows", p->book.free_pages(),
                         rows);
    *copies = *src >= 0;
    return MXH_OK;
} catch (const std::bad_alloc&) {
    return set_error(MXH_ERR_OOM, "pages_extend: out of host memory");
}

int mxh_pages_set_length(mxh_pages* p, int seq, int rows) {
    if (int rc = check_seq("pages_set_length", p, seq)) return rc;
    const int most = std::max(p->book.length(seq), p->book.reserved(seq));
    if (rows < 0 || rows > most) return set_error(MXH_ERR_ARG, "pages_set_length: %d rows of at most %d", rows, most);
    p->book.set_length(seq, rows);
    return MXH_OK;
}

int mxh_pages_length(const mxh_pages* p, int seq) {
    if (int rc = check_seq("pages_length", p, seq)) return rc;
    return p->book.length(seq);
}

int mxh_pages_free(const mxh_pages* p) {
    return p ? p->book.free_pages() : set_error(MXH_ERR_ARG, "pages_free: null pages");
}

int mxh_pages_table(const mxh_pages* p, const int* seqs, int n, int* table, int table_ld, int* cached) {
    if (!p || n < 0 || (n > 0 && (!seqs || !table)) || table_ld < 1)
        return set_error(MXH_ERR_ARG, "pages_table: bad arguments");
    for (int i = 0; i < n; ++i) {
        if (int rc = check_seq("pages_table", p, seqs[i])) return rc;
        if (p->book.pages(seqs[i]).size() > (size_t)table_ld)
            return set_error(MXH_ERR_ARG, "pages_table: sequence %d has %zu pages, rows of %d", seqs[i],
                             p->book.pages(seqs[i]).size(), table_ld);
    }
    for (int i = 0; i < n; ++i) {
        const std::vector<int>& ids = p->book.pages(seqs[i]);
        int* row = table + (size_t)i * table_ld;
        std::fill(std::copy(ids.begin(), ids.end(), row), row + table_ld, -1);
        if (cached) cached[i] = p->book.length(seqs[i]);
    }
    return MXH_OK;
}

}  // extern "C"
