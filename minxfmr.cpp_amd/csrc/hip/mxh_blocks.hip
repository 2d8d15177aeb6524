// mxh_blocks.hip — long contexts by blocks of rows (include/minxfmr_hip.h:
// mxh_kv_block_bounds, mxh_kv_select_blocks, mxh_attention_blocks): the least and
// the greatest key of each block, a value a dimension; the blocks whose bounds
// allow a query the largest scores; attention over the rows of those.
//
// With least <= k <= greatest in every dimension, q.k is at most
//     sum_d max(q_d, 0) greatest_d + min(q_d, 0) least_d,
// which is a product with the bounds as they lie in memory.  A block's score for a
// token and kv head is the largest of the kv head's q heads' bounds.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mxh_blocks.h"
#include "mxh_internal.h"
#include "mxh_paged.h"
#include "mxh_paged_tile.h"

namespace mxh {

namespace {

// Bounds of a block and kv head: [least | greatest], HD halves each, in the order
// of the pool's rows: [page][block of the page][kv head]
struct BlockArgs {
    PagedArgs pg;
    __half* bounds;  // the layer's first
    int block_shift, n_first, n_last, n_select;
    int n_blocks;  // of a row of the table
};

__device__ __forceinline__ int64_t block_place(const BlockArgs& a, int s, int b) {  // -1: absent
    if (b < 0 || b >= a.n_blocks) return -1;
    const int64_t row = paged_row(a.pg, s, b << a.block_shift);
    return row < 0 ? -1 : row >> a.block_shift;
}

// A token's sequence and its index there; s -1: none (past the 64th of a drafted
// tree too)
struct TokenAt {
    int s, i, cached, n;  // cached rows, tokens of the sequence
};
__device__ __forceinline__ TokenAt token_at(const PagedArgs& a, int t) {
    TokenAt x{paged_seq_of(a, t), 0, 0, 0};
    if (x.s < 0) return x;
    const int first = a.start[x.s];
    x.i = t - first;
    x.n = min(a.start[x.s + 1], a.n_tokens) - first;
    if (a.parent) x.n = min(x.n, kTreeMax);
    x.cached = min(max(a.cached[x.s], 0), 1 << 30);
    if (x.i >= x.n) x.s = -1;
    return x;
}

// ---- bounds ---------------------------------------------------------------

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// Workgroup (tokens [chunk x, + chunk), 64 pieces of 8 dims): the blocks that the
// tokens are the first new rows of, one after the other; all rows of a block by
// threads that each take every RG-th, joined through LDS.
constexpr int kBoundThreads = 256;
__global__ __launch_bounds__(kBoundThreads) void kv_block_bounds_kernel(BlockArgs a, int chunk, int pieces, int hd8) {
    __shared__ half8 least[kBoundThreads], greatest[kBoundThreads];
    const int tid = threadIdx.x;
    const int c = min(pieces - 64 * (int)blockIdx.y, 64), rg = kBoundThreads / c;
    const int mine = tid / c, col = 64 * (int)blockIdx.y + tid % c;
    const int rows = 1 << a.block_shift;
    int t = (int)blockIdx.x * chunk;
    const int end = min(t + chunk, a.pg.n_tokens);
    while (t < end) {
        const TokenAt x = token_at(a.pg, t);
        if (x.s < 0) {
            ++t;
            continue;
        }
        const int row = x.cached + x.i, b = row >> a.block_shift;
        const int next = t + rows - (row & (rows - 1));  // the first token of the block behind, if the sequence has it
        const bool here = x.i == 0 || (row & (rows - 1)) == 0;
        const int64_t place = here ? block_place(a, x.s, b) : -1;
        t = min(next, t - x.i + x.n);
        if (place < 0) continue;
        const int n = min(x.cached + x.n - (b << a.block_shift), rows);
        half8 lo, hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = (_Float16)INFINITY, hi[e] = -(_Float16)INFINITY;
        if (mine < rg) {
            const half8* p = reinterpret_cast<const half8*>(a.pg.k) + ((place << a.block_shift) + mine) * pieces + col;
#pragma unroll 8
            for (int r = mine; r < n; r += rg, p += (int64_t)rg * pieces) {
                const half8 v = *p;
                lo = __builtin_elementwise_min(lo, v);
                hi = __builtin_elementwise_max(hi, v);
            }
        }
        least[tid] = lo, greatest[tid] = hi;
        __syncthreads();
        if (tid < c) {
            for (int m = 1; m < rg; ++m) {
                lo = __builtin_elementwise_min(lo, least[tid + m * c]);
                hi = __builtin_elementwise_max(hi, greatest[tid + m * c]);
            }
            const int g = col / hd8, d = col - g * hd8;
            half8* out = reinterpret_cast<half8*>(a.bounds) + (place * a.pg.nkv + g) * 2 * hd8 + d;
            out[0] = lo, out[hd8] = hi;
        }
        __syncthreads();
    }
}

// ---- selection -------------------------------------------------------------

// Scores as 64-bit integers that order as the doubles do, NaN as +infinity
__device__ __forceinline__ uint64_t order_key(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x == x ? x + 0.0 : (double)INFINITY);
    return u ^ (u >> 63 ? ~0ull : 1ull << 63);
}

struct SelectArgs {
    BlockArgs b;
    const float* q;
    int nh, group, tokens;  // q heads of a kv head; tokens of a tile
    int t0, t1;             // tokens of this launch
    uint64_t* keys;         // [t1 - t0][nkv][n_blocks]
    int* chosen;            // [n_tokens][nkv][n_select]
};

// The blocks that compete for token x: [n_first, end), none where all of its
// blocks are taken; own: the last
struct Rivals {
    int own, end;
};
__device__ __forceinline__ Rivals rivals(const BlockArgs& a, const TokenAt& x) {
    Rivals r;
    r.own = min((x.cached + x.i) >> a.block_shift, a.n_blocks - 1);
    r.end = r.own + 1 > a.n_select ? r.own + 1 - a.n_last : 0;
    return r;
}

// Workgroup (64 `iters` blocks, kv head, tile of tokens): a wave takes 16 blocks
// and the tile's 16 rows of q at a time, v_mfma_f64_16x16x4_f64: in 64 bits the
// choice depends neither on how the work is split nor on the order of sums.
constexpr int kScoreThreads = 256;
typedef double f64x4 __attribute__((ext_vector_type(4)));
template <int HD>
__global__ __launch_bounds__(kScoreThreads) void block_score_kernel(SelectArgs a, int iters, int chunks) {
    constexpr int STEPS = HD / 2;  // products; a lane's halves of a block's bounds
    __shared__ double qs[STEPS * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, kk = lane >> 4;
    const int nkv = a.b.pg.nkv;
    const int chunk = (int)(blockIdx.x % chunks), g = (int)(blockIdx.x / chunks % nkv);
    const int first = a.t0 + (int)(blockIdx.x / chunks / nkv) * a.tokens, last = min(first + a.tokens, a.t1);
    const int lo = chunk * 64 * iters;
    bool staged = false;
    for (int t = first; t < last;) {
        const TokenAt x = token_at(a.b.pg, t);
        if (x.s < 0) {
            ++t;
            continue;
        }
        const int stop = min(t - x.i + x.n, last);  // the run of this sequence's tokens
        const int hi = rivals(a.b, TokenAt{x.s, x.i + stop - 1 - t, x.cached, x.n}).end;
        if (hi > lo) {
            if (!staged) {
                // column c of the tile: token c / group, q head c % group
                for (int i = tid; i < STEPS * 64; i += kScoreThreads) {
                    const int c = i & 15, e = (i >> 4 & 3) * STEPS + (i >> 6), tt = first + c / a.group;
                    float v = 0.f;
                    if (c < a.tokens * a.group && tt < last) {
                        v = a.q[((int64_t)tt * a.nh + g * a.group + c % a.group) * HD + e % HD];
                        v = e < HD ? (v >= 0.f ? 0.f : v) : (v <= 0.f ? 0.f : v);
                    }
                    qs[i] = v;
                }
                __syncthreads();
                staged = true;
            }
            for (int b0 = lo + 16 * wave; b0 < min(lo + 64 * iters, hi); b0 += 64) {
                const int64_t place = block_place(a.b, x.s, b0 + m);
                half8 v[STEPS / 8];
#pragma unroll
                for (int i = 0; i < STEPS / 8; ++i) {
                    const half8* p = reinterpret_cast<const half8*>(a.b.bounds + ((place < 0 ? 0 : place) * nkv + g) * 2 * HD +
                                                                    kk * STEPS);
                    v[i] = p[i];
                }
                f64x4 acc = {0., 0., 0., 0.};
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)v[i / 8][i % 8], qs[64 * i + lane], acc, 0,
                                                               0, 0);
                // lane: column m, blocks b0 + 4 r + kk
                const uint64_t gone = __ballot(place < 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    double best = acc[r];
                    for (int h = 1; h < a.group; ++h) {
                        const double o = __shfl(acc[r], min(lane + h, 63));
                        best = o > best || o != o ? o : best;
                    }
                    const int b = b0 + 4 * r + kk, tt = first + m / a.group;
                    if (gone >> (4 * r + kk) & 1) best = -INFINITY;
                    if (m % a.group == 0 && tt >= t && tt < stop && b < hi)
                        a.keys[((int64_t)(tt - a.t0) * nkv + g) * a.b.n_blocks + b] = order_key(best);
                }
            }
        }
        t = stop;
    }
}

// Workgroup (token, kv head): the n-th largest key, eight bits at a time, then the
// blocks from there on in their order.
constexpr int kPickThreads = 256;
__global__ __launch_bounds__(kPickThreads) void block_pick_kernel(SelectArgs a) {
    __shared__ uint32_t bins[256], wsum[kPickThreads / 64];
    __shared__ uint32_t found[2];  // the bin, keys wanted of it
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nkv = a.b.pg.nkv;
    const int t = a.t0 + (int)(blockIdx.x / nkv), g = (int)(blockIdx.x % nkv);
    const TokenAt x = token_at(a.b.pg, t);
    if (x.s < 0) return;
    const Rivals r = rivals(a.b, x);
    int* out = a.chosen + ((int64_t)t * nkv + g) * a.b.n_select;
    if (r.end == 0) {
        for (int i = tid; i < a.b.n_select; i += kPickThreads) out[i] = i <= r.own ? i : -1;
        return;
    }
    const int n0 = a.b.n_first, want = a.b.n_select - n0 - a.b.n_last;
    for (int i = tid; i < n0; i += kPickThreads) out[i] = i;
    for (int i = tid; i < a.b.n_last; i += kPickThreads) out[n0 + want + i] = r.end + i;
    if (want == 0) return;
    const uint64_t* keys = a.keys + ((int64_t)(t - a.t0) * nkv + g) * a.b.n_blocks;
    uint64_t prefix = 0;
    uint32_t need = (uint32_t)want;
    int shift = 64;
    const auto inclusive = [&](uint32_t v) {  // over the workgroup
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)v, off);
            if (lane >= off) v += o;
        }
        __syncthreads();
        if (lane == 63) wsum[wave] = v;
        __syncthreads();
        for (int w = 0; w < wave; ++w) v += wsum[w];
        return v;
    };
    for (;;) {
        shift -= 8;
        bins[tid] = 0;
        __syncthreads();
        for (int b = n0 + tid; b < r.end; b += kPickThreads) {
            const uint64_t k = keys[b];
            if (shift == 56 || k >> (shift + 8) == prefix) atomicAdd(&bins[k >> shift & 255], 1u);
        }
        __syncthreads();
        const uint32_t n = bins[255 - tid], upto = inclusive(n);
        if (upto >= need && upto - n < need) found[0] = 255 - tid, found[1] = need - (upto - n);
        __syncthreads();
        prefix = prefix << 8 | found[0], need = found[1];
        const bool all = bins[found[0]] == need;
        __syncthreads();
        if (all || shift == 0) break;
    }
    // those above the prefix, and the first `need` of those with it
    int done = n0;
    uint32_t ties = 0;
    for (int b0 = n0; b0 < r.end; b0 += kPickThreads) {
        const int b = b0 + tid;
        const uint64_t k = b < r.end ? keys[b] >> shift : 0;
        const bool above = b < r.end && k > prefix, same = b < r.end && k == prefix;
        const uint32_t before = inclusive(same) - same + ties;
        const bool take = above || (same && before < need);
        const uint32_t upto = inclusive(take);
        if (take) out[done + upto - 1] = b;
        __syncthreads();
        if (tid == kPickThreads - 1) found[0] = upto, found[1] = before + same;
        __syncthreads();
        done += found[0], ties = found[1];
        __syncthreads();
    }
}

// ---- attention -------------------------------------------------------------

struct BlockAttnArgs {
    TileArgs t;
    const int* chosen;  // [n_tokens][nkv][n_select]
    int n_select, block_shift, n_blocks, splits, words;
    int lists;  // LDS bytes before the lists
};

// Workgroup (kv head, tile and split): the blocks that any of a sequence's tokens
// in the tile has chosen, found as bits in LDS, then a share of their stages.
template <int HD>
__global__ __launch_bounds__(kThreads, 2) void attention_blocks_kernel(BlockAttnArgs a) {
    extern __shared__ __align__(256) uint8_t smem[];
    __shared__ uint32_t sums[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), tid = threadIdx.x, lane = tid & 63;
    const uint32_t g = blockIdx.x, nkv = (uint32_t)a.t.pg.nkv;
    const int64_t index = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
    const int T = (int)a.t.tokens, tile = (int)(index / a.splits), z = (int)(index - (int64_t)tile * a.splits);
    const int first = tile * T, last = min(first + T, a.t.pg.n_tokens);
    uint32_t* bits = reinterpret_cast<uint32_t*>(smem);  // [tokens][words]
    uint32_t* blocks = reinterpret_cast<uint32_t*>(smem + a.lists);
    uint16_t* who = reinterpret_cast<uint16_t*>(blocks + kListMax);
    for (int t = first; t < last;) {
        const TokenAt x = token_at(a.t.pg, t);
        if (x.s < 0) {  // (its rows of the part: to be left alone)
            if (a.splits > 1)
                for (int i = tid; i < (int)a.t.group; i += kThreads)
                    a.t.ml[(index * nkv + g) * 16 + (t - first) * (int)a.t.group + i] = make_float2(0.f, -1.f);
            ++t;
            continue;
        }
        const int n = min(t - x.i + x.n, last) - t;
        const int words = min((min((x.cached + x.i + n - 1) >> a.block_shift, a.n_blocks - 1) >> 5) + 1, a.words);
        for (int i = tid; i < n * words; i += kThreads) bits[i] = 0;
        __syncthreads();
        for (int i = tid; i < n * a.n_select; i += kThreads) {
            const int u = i / a.n_select;
            const int b = a.chosen[((int64_t)(t + u) * nkv + g) * a.n_select + (i - u * a.n_select)];
            const int own = min((x.cached + x.i + u) >> a.block_shift, a.n_blocks - 1);
            if (b >= 0 && b <= own) atomicOr(&bits[u * words + (b >> 5)], 1u << (b & 31));
        }
        __syncthreads();
        const int per = (words + kThreads - 1) / kThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
        const auto any = [&](int w) {
            uint32_t v = 0;
            for (int u = 0; u < n; ++u) v |= bits[u * words + w];
            return v;
        };
        uint32_t mine = 0;
        for (int w = w0; w < w1; ++w) mine += __popc(any(w));
        uint32_t upto = mine;
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)upto, off);
            if (lane >= off) upto += o;
        }
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        uint32_t total = 0;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) upto += sums[w];
            total += sums[w];
        }
        uint32_t at = upto - mine;
        for (int w = w0; w < w1; ++w)
            for (uint32_t v = any(w); v; v &= v - 1) {
                const int bit = __ffs((int)v) - 1;
                uint32_t m = 0;
                for (int u = 0; u < n; ++u) m |= (bits[u * words + w] >> bit & 1) << u;
                blocks[at] = (uint32_t)(32 * w + bit), who[at] = (uint16_t)m;
                ++at;
            }
        __syncthreads();
        SegmentOf it;
        it.s = x.s, it.first = (uint32_t)(t - x.i), it.n = (uint32_t)x.n, it.cached = (uint32_t)x.cached;
        it.tile = 0, it.begin = 0, it.i0 = (uint32_t)x.i, it.tokens = (uint32_t)n;
        it.blocks = blocks, it.who = who;
        it.n_blocks = (uint32_t)__builtin_amdgcn_readfirstlane((int)total), it.block_shift = (uint32_t)a.block_shift;
        const uint32_t stages = ((it.n_blocks << a.block_shift) + 127) >> 7;
        it.st0 = stages * (uint32_t)z / (uint32_t)a.splits, it.st1 = stages * (uint32_t)(z + 1) / (uint32_t)a.splits;
        it.slot = a.splits > 1 ? (int)index : -1;
        it.row0 = (uint32_t)(t - first) * a.t.group;
        attend_tile<HD, 16, kListed>(a.t, it, g, tid, wave, false, smem);
        t += n;
        if (t < last) __syncthreads();
    }
}

struct BlockMergeArgs {
    const float* part;
    const float2* ml;
    float* att;
    int64_t total;  // units of four dims, of all tokens
    int nkv, group, tokens, splits;
};

template <int HD>
__global__ __launch_bounds__(kJoinThreads) void blocks_merge_kernel(BlockMergeArgs a) {
    const int64_t u = (int64_t)blockIdx.x * kJoinUnits + threadIdx.x % kJoinUnits;
    const int64_t head = min(u, a.total - 1) / (HD / 4);
    const int d = 4 * (int)(u % (HD / 4)), nh = a.nkv * a.group;
    const int64_t t = head / nh, tile = t / a.tokens;
    const int hq = (int)(head - t * nh), g = hq / a.group;
    const int row = (int)(t - tile * a.tokens) * a.group + hq - g * a.group;
    const auto place = [&](int z) { return ((tile * a.splits + z) * a.nkv + g) * 16 + row; };
    const auto where = [&](int z, float2& x, float4& v) __attribute__((always_inline)) {
        const int64_t at = place(z);
        x = a.ml[at];
        v = *reinterpret_cast<const float4*>(a.part + at * HD + d);
    };
    const bool any = u < a.total && !(a.ml[place(0)].y < 0.f);  // (else no sequence's)
    join_parts(a.splits, where, any ? a.att + head * HD + d : nullptr);
}

BlockSize block_size(const BlockArgs& a, int nh) {
    return BlockSize{a.pg.n_seq, a.pg.n_tokens, a.n_blocks, a.pg.nkv, nh / a.pg.nkv, a.n_select, 1 << a.block_shift,
                     device_cus()};
}

BlockArgs block_args(const PagedArgs& pg, const BlocksOf& b) {
    return BlockArgs{pg, b.bounds, b.block_shift, b.n_first, b.n_last, b.n_select, (int)blocks_of_table(pg, b.block_shift)};
}

template <int HD>
int launch_attention(const BlockAttnArgs& a, int64_t tiles, hipStream_t st) {
    constexpr int RING = lds_bytes(HD, 16);
    BlockAttnArgs args = a;
    args.lists = std::max(RING, (int)((a.t.tokens * (size_t)a.words * 4 + 255) / 256 * 256));
    const size_t lds = (size_t)args.lists + kListMax * 6;
    static bool attr_set = false;
    if (!attr_set) {
        if (hipFuncSetAttribute((const void*)attention_blocks_kernel<HD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                std::max(RING, kBitBytes) + kListMax * 6) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const int64_t items = tiles * a.splits, y = std::min<int64_t>(items, 32768);
    hipLaunchKernelGGL(attention_blocks_kernel<HD>,
                       dim3((unsigned)a.t.pg.nkv, (unsigned)y, (unsigned)((items + y - 1) / y)), dim3(kThreads), lds, st,
                       args);
    if (a.splits > 1) {
        const int64_t total = (int64_t)a.t.pg.n_tokens * a.t.nh * (HD / 4);
        const BlockMergeArgs m{a.t.part, a.t.ml, a.t.att, total, a.t.pg.nkv, (int)a.t.group, (int)a.t.tokens, a.splits};
        hipLaunchKernelGGL(blocks_merge_kernel<HD>, dim3((unsigned)((total + kJoinUnits - 1) / kJoinUnits)),
                           dim3(kJoinThreads), 0, st, m);
    }
    return MXH_OK;
}

template <int HD>
void launch_scores(const SelectArgs& a, int64_t tiles, hipStream_t st) {
    // blocks of a workgroup: 64 where that leaves few workgroups
    const int64_t few = (a.b.n_blocks + 63) / 64;
    const int iters = few * tiles * a.b.pg.nkv > 4096 ? 4 : 1;
    const int chunks = (a.b.n_blocks + 64 * iters - 1) / (64 * iters);
    hipLaunchKernelGGL(block_score_kernel<HD>, dim3((unsigned)(chunks * tiles * a.b.pg.nkv)), dim3(kScoreThreads), 0, st,
                       a, iters, chunks);
}

}  // namespace

void block_bounds_launch(const PagedArgs& pg, const BlocksOf& b, int hd, hipStream_t st) {
    const BlockArgs a = block_args(pg, b);
    // tokens of a workgroup: a block's where sequences have as many
    const int chunk = std::max(1, std::min(1 << b.block_shift, pg.n_tokens / pg.n_seq));
    const int pieces = pg.nkv * hd / 8;
    hipLaunchKernelGGL(kv_block_bounds_kernel,
                       dim3((unsigned)((pg.n_tokens + chunk - 1) / chunk), (unsigned)((pieces + 63) / 64)),
                       dim3(kBoundThreads), 0, st, a, chunk, pieces, hd / 8);
}

size_t select_blocks_work_bytes(const PagedArgs& pg, const BlocksOf& b) {
    return select_work_bytes(pg.n_tokens, blocks_of_table(pg, b.block_shift), pg.nkv);
}

void select_blocks_launch(const PagedArgs& pg, const BlocksOf& b, const float* q, int nh, int hd, int* chosen,
                          void* work, hipStream_t st) {
    SelectArgs a{block_args(pg, b), q, nh, nh / pg.nkv, 0, 0, 0, static_cast<uint64_t*>(work), chosen};
    a.tokens = pg.n_tokens > 2 * (int64_t)pg.n_seq ? 16 / a.group : 1;
    const int64_t step = select_tokens(pg.n_tokens, a.b.n_blocks, pg.nkv);
    for (int64_t t = 0; t < pg.n_tokens; t += step) {
        a.t0 = (int)t, a.t1 = (int)std::min<int64_t>(t + step, pg.n_tokens);
        const int64_t n = a.t1 - a.t0, tiles = (n + a.tokens - 1) / a.tokens;
        if (a.b.n_blocks > b.n_select) {  // (else no token has more blocks than it takes)
            if (hd == 32) launch_scores<32>(a, tiles, st);
            else if (hd == 64) launch_scores<64>(a, tiles, st);
            else launch_scores<128>(a, tiles, st);
        }
        hipLaunchKernelGGL(block_pick_kernel, dim3((unsigned)(n * pg.nkv)), dim3(kPickThreads), 0, st, a);
    }
}

size_t attention_blocks_work_bytes(const PagedArgs& pg, const BlocksOf& b, int nh, int hd) {
    return block_work_bytes(block_size(block_args(pg, b), nh), hd);
}

size_t attention_blocks_work_bound(const PagedArgs& pg, const BlocksOf& b, int nh, int hd) {
    return block_work_bound(block_size(block_args(pg, b), nh), hd);
}

int attention_blocks_launch(const PagedArgs& pg, const BlocksOf& b, const int* chosen, const float* q, int nh, int hd,
                            float* att, void* work, hipStream_t st) {
    const BlockArgs ba = block_args(pg, b);
    const BlockSize size = block_size(ba, nh);
    const int splits = block_splits(size);
    const int64_t tiles = block_tiles(size);
    const uint32_t group = (uint32_t)size.group;
    float* part = static_cast<float*>(work);
    const BlockAttnArgs a{{pg, q, att, part, reinterpret_cast<float2*>(part + (size_t)tiles * splits * pg.nkv * 16 * hd),
                           nh, 1.4426950408889634f / sqrtf((float)hd), group, (uint32_t)block_tokens(size),
                           (65536 + group - 1) / group},
                          chosen, b.n_select, b.block_shift, ba.n_blocks, splits, (ba.n_blocks + 31) / 32, 0};
    return hd == 32   ? launch_attention<32>(a, tiles, st)
           : hd == 64 ? launch_attention<64>(a, tiles, st)
                      : launch_attention<128>(a, tiles, st);
}

}  // namespace mxh
