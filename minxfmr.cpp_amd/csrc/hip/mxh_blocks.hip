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
    // (as paged_seq_of, with what is read of the sequence in flight together)
    const int lane = threadIdx.x & 63, part = (a.n_seq + 63) / 64;
    int s = 0;
    if (part > 1) {
        const int e = (lane + 1) * part;
        s = part * (int)__popcll(__ballot(e <= a.n_seq && a.start[min(e, a.n_seq)] <= t));
    }
    const int e = s + lane + 1;
    s += (int)__popcll(__ballot(a.start[min(e, a.n_seq)] <= t && e <= a.n_seq));
    const int at = min(s, a.n_seq - 1), first = a.start[at], end = a.start[at + 1], cached = a.cached[at];
    TokenAt x{s, t - first, min(max(cached, 0), 1 << 30), min(end, a.n_tokens) - first};
    if (a.parent) x.n = min(x.n, kTreeMax);
    if (s >= a.n_seq || first < 0 || x.i < 0 || x.i >= x.n) x.s = -1;
    return x;
}

// ---- bounds ---------------------------------------------------------------

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// Workgroup (tokens [chunk x, + chunk), 64 pieces of 8 dims): the blocks that the
// tokens are the first new rows of, one after the other; all rows of a block by
// threads that each take every RG-th, joined through LDS.  Seven prompts of up to
// 6,000 tokens (35 MB of K with 8 heads of 128) 11 us, one token 4: a launch, and the
// loads of lengths, page and rows one after the other.  (8 / 16 / 32 / 128 pieces a
// workgroup 44 / 23 / 16 / 13 us, eight waves 13; sixteen rows at a time 12.7)
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
            const half8* p = reinterpret_cast<const half8*>(a.pg.k) + (place << a.block_shift) * pieces + col;
            for (int r = mine; r < n; r += 8 * rg) {  // (past the last row the last again)
                half8 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)min(r + i * rg, n - 1) * pieces];
#pragma unroll
                for (int i = 0; i < 8; ++i) lo = __builtin_elementwise_min(lo, v[i]), hi = __builtin_elementwise_max(hi, v[i]);
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

// Scores as 64-bit integers that order as the doubles do, NaN above all of them (0 is
// below all: absent blocks)
__device__ __forceinline__ uint64_t order_key(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return x != x ? ~0ull : u ^ (u >> 63 ? ~0ull : 1ull << 63);
}

// Of a row of scores (of a token and kv head) the workspace has ld floats, the blocks'
// scores in units of the row's own (of absent blocks -infinity), and from there one
// for every 16 blocks, how far their scores may be off.  Where that does not decide,
// 64-bit keys take their place.
struct SelectArgs {
    BlockArgs b;
    const float* q;
    int nh, group, tokens;  // q heads of a kv head; tokens of a tile
    int t0, t1;             // tokens of this launch
    int ld;                 // scores of a row, n_blocks and up to a multiple of 16
    float* scores;          // [t1 - t0][nkv][2 ld]
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

// max over the q heads of a kv head, in the lane of its first: lanes m .. m + group - 1
// of a row of 16.  (Two instructions a value for group 4, six as C++; a lane's value
// may be read by its neighbours two instructions after it was written.)
#define MXH_MAX4(PERM)                                                                                        \
    asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 " PERM " row_mask:0xf bank_mask:0xf"                             \
        "\n\tv_max_f32_dpp %1, %1, %1 " PERM " row_mask:0xf bank_mask:0xf"                                    \
        "\n\tv_max_f32_dpp %2, %2, %2 " PERM " row_mask:0xf bank_mask:0xf"                                    \
        "\n\tv_max_f32_dpp %3, %3, %3 " PERM " row_mask:0xf bank_mask:0xf"                                    \
        : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w))
__device__ __forceinline__ void heads_max(float4& v, int group) {
    if ((group & (group - 1)) == 0) {
        if (group >= 2) MXH_MAX4("quad_perm:[1,0,3,2]");  // the other of a pair
        if (group >= 4) MXH_MAX4("quad_perm:[2,3,0,1]");  // of a quad's pairs
        if (group >= 8) MXH_MAX4("row_half_mirror");      // of eight lanes' quads
        return;
    }
    const float4 o = v;
    for (int h = 1; h < group; ++h) {
        v.x = fmaxf(v.x, __shfl_down(o.x, (unsigned)h)), v.y = fmaxf(v.y, __shfl_down(o.y, (unsigned)h));
        v.z = fmaxf(v.z, __shfl_down(o.z, (unsigned)h)), v.w = fmaxf(v.w, __shfl_down(o.w, (unsigned)h));
    }
}
#undef MXH_MAX4

// Scores on the fp16 matrix cores, 16 blocks and the 16 rows of q of a tile of
// tokens at a time, v_mfma_f32_16x16x32_f16: least | greatest of a block as they lie
// there times min(q, 0) | max(q, 0), q in fp16 after the power of two that brings the
// largest |q| of the token's kv head to [2^13, 2^14).
//
// What the sums may be off by: q by 2^-11 of itself and 2^-25, and up to 256
// additions, each by 2^-23 of the sum of the magnitudes at most (were they cut
// off).  A second product sums magnitudes, with |q| raised to 2^-3 where it is less,
// so that 1.25 x 2^-11 of it is over all of that; block_pick_kernel decides what that
// leaves open in 64 bits, some five blocks of a thousand.  (All scores in 64 bits,
// v_mfma_f64_16x16x4_f64: 125 us for 512 tokens at 30,000 rows, 26 now, and 60 for 48
// single tokens at up to 16,000, 18 now.)
// magnitudes of halves (the sign bits of pairs at a time), and an eighth at least (as
// integers: a maximum of halves costs an instruction more for every operand)
__device__ __forceinline__ f16x8 magnitudes(f16x8 v) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(f16x8, __builtin_bit_cast(words, v) & 0x7fff7fffu);
}
__device__ __forceinline__ f16x8 at_least(f16x8 v, uint32_t eighth) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    const u16x8 y = (uint16_t)eighth;
    return __builtin_bit_cast(f16x8, __builtin_elementwise_max(__builtin_bit_cast(u16x8, magnitudes(v)), y));
}

// SIZES: whether the magnitudes of q stay in registers
template <int HD, bool SIZES>
struct ScoreTile {
    static constexpr int KS = HD / 16;  // products
    f16x8 q[KS], q_size[SIZES ? KS : 1];
    // the largest sum of magnitudes of a lane's column, as bits: those of infinity and
    // above where scores are no numbers; odd: whether those of any block are
    uint32_t size, odd;
    // column m of the tile: token first + m / group, q head m % group; lane: dims
    // 32 i + 8 kk + e
    __device__ __forceinline__ void stage(const SelectArgs& a, int first, int last, int g, int m, int kk) {
        const int u = m / a.group, tt = first + u;
        const bool there = u < a.tokens && tt < last;
        const float* row =
            a.q + ((int64_t)(there ? tt : min(first, a.t1 - 1)) * a.nh + g * a.group + (there ? m % a.group : 0)) * HD;
        const auto at = [&](int i, int e) { return *reinterpret_cast<const float4*>(row + 32 * i + 8 * kk + e); };
        uint32_t big = 0;  // the largest magnitude's bits; past those of infinity where there is a NaN
#pragma unroll
        for (int i = 0; i < KS / 2; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 y = at(i, e);
                big = max(max(big, max(__float_as_uint(y.x) << 1, __float_as_uint(y.y) << 1)),
                          max(__float_as_uint(y.z) << 1, __float_as_uint(y.w) << 1));
            }
        big = there ? big : 0;
        big = max(big, __float_as_uint(lane_xor<16>(__uint_as_float(big))));
        big = max(big, __float_as_uint(lane_xor<32>(__uint_as_float(big))));
        const int c0 = u * a.group;     // the kv head's columns of the token
        uint32_t most = 0;
        for (int h = 0; h < a.group; ++h) most = max(most, (uint32_t)__shfl((int)big, min(c0 + h, 15)));
        size = odd = most < 0xff000000u ? 0u : 0x7f800000u;
        const int f = min(14 - __builtin_amdgcn_frexp_expf(__uint_as_float(most >> 1)), 120);
        const float scale = there && odd == 0 ? __uint_as_float((uint32_t)(127 + f) << 23) : 0.f;
#pragma unroll
        for (int i = 0; i < KS / 2; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 y = at(i, e);
                const f16x2 z[2] = {__builtin_convertvector((f32x2{y.x * scale, y.y * scale}), f16x2),
                                    __builtin_convertvector((f32x2{y.z * scale, y.w * scale}), f16x2)};
#pragma unroll
                for (int c = 0; c < 2; ++c) {  // least with min(q, 0), greatest with max(q, 0)
                    const f16x2 none = {0, 0}, neg = __builtin_elementwise_min(z[c], none),
                                pos = __builtin_elementwise_max(z[c], none);
                    q[i][e + 2 * c] = neg[0], q[i][e + 2 * c + 1] = neg[1];
                    q[KS / 2 + i][e + 2 * c] = pos[0], q[KS / 2 + i][e + 2 * c + 1] = pos[1];
                }
            }
        if constexpr (SIZES)
#pragma unroll
            for (int i = 0; i < KS; ++i) q_size[i] = at_least(q[i], 0x3000);
    }
    // bounds(i): lane's 8 of block m of 16.  The scores of the tile's token u, the largest
    // of its q heads', go to to[u stride], 16
    template <class Bounds>
    __device__ __forceinline__ void score(const SelectArgs& a, const Bounds& bounds, int place, float* to, int stride,
                                          int m, int kk) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f}, sum = s;
        uint32_t eighth = 0x3000;
        if constexpr (!SIZES) asm volatile("" : "+v"(eighth));  // (else the magnitudes of q stay in registers)
        constexpr int BATCH = KS < 4 ? KS : 4;
        f16x8 v[BATCH];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (i % BATCH == 0)
#pragma unroll
                for (int k = 0; k < BATCH; ++k) v[k] = bounds(i + k);
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i % BATCH], q[i], s, 0, 0, 0);
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                magnitudes(v[i % BATCH]), SIZES ? q_size[SIZES ? i : 0] : at_least(q[i], eighth), sum, 0, 0, 0);
        }
        // lane: column m, blocks 4 kk + r.  (Absent ones' bounds are zeros, their sums too)
        const uint32_t gone = (uint32_t)__ballot(place < 0) >> (4 * kk);
        float4 x;
        x.x = gone & 1 ? -INFINITY : s[0], x.y = gone & 2 ? -INFINITY : s[1];
        x.z = gone & 4 ? -INFINITY : s[2], x.w = gone & 8 ? -INFINITY : s[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) size = max(size, __float_as_uint(sum[r]));
        heads_max(x, a.group);
        if (m % a.group == 0 && m / a.group < a.tokens) *reinterpret_cast<float4*>(to + m / a.group * stride + 4 * kk) = x;
    }
    // The scores of tokens [t, stop) of the tile, `steps` of 16 blocks b0 + apart j, out
    // of LDS (`kept`, as score left them), with what they are off by
    __device__ __forceinline__ void flush(const SelectArgs& a, const float* kept, int stride, int steps, int b0, int apart,
                                          int first, int t, int stop, int g, int lane) {
        float off = size < 0x7f800000u ? __uint_as_float(size) * (1.25f / 2048.f) : INFINITY;
        off = fmaxf(off, lane_xor<16>(off));
        off = fmaxf(off, lane_xor<32>(off));
        size = odd;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        for (int tt = t; tt < stop; ++tt) {
            const int u = tt - first;
            float far = 0.f;
            for (int h = 0; h < a.group; ++h) far = fmaxf(far, __shfl(off, u * a.group + h));
            float* row = a.scores + ((int64_t)(tt - a.t0) * a.b.pg.nkv + g) * 2 * a.ld;
            for (int i = lane; i < 16 * steps; i += 64) row[b0 + apart * (i >> 4) + (i & 15)] = kept[u * stride + i];
            for (int i = lane; i < steps; i += 64) row[a.ld + ((b0 + apart * i) >> 4)] = far;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
};

// the lane's pieces of a block's bounds, of head g: every fourth 16 bytes from there
__device__ uint4 no_bounds[2 * 128 / 8];  // (of absent blocks: zeros)
template <int HD>
__device__ __forceinline__ const half8* bounds_at(const SelectArgs& a, int place, int g, int kk) {
    const half8* p = reinterpret_cast<const half8*>(a.b.bounds) + ((int64_t)place * a.b.pg.nkv + g) * (HD / 4);
    return (place < 0 ? reinterpret_cast<const half8*>(no_bounds) : p) + kk;
}

// Places of `steps` times 16 blocks, b0 + apart j, of a wave's, into LDS before the
// loop that reads them: a table load in there would have every step wait for it.
// Blocks below n_first and from `end` on compete for no token of the run: -1, as what
// lies in their bounds (nothing yet, behind the sequence) is not to count in `size`
__device__ __forceinline__ void find_places(const SelectArgs& a, int s, int b0, int apart, int steps, int end, int* places,
                                            int lane) {
    for (int i = lane; i < 16 * steps; i += 64) {
        const int b = b0 + apart * (i >> 4) + (i & 15);
        places[i] = b >= a.b.n_first && b < end ? (int)block_place(a.b, s, b) : -1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

// Few tokens: a workgroup takes a tile, its waves different blocks (16 `iters` each).
// 48 single tokens at up to 16,000 rows, blocks of 32: 18 us for 39 MB of bounds, of
// which waves wait 56%; one at 60,000, blocks of 64, 6 us.
constexpr int kScoreThreads = 256, kScoreWaves = 4;
template <int HD>
__global__ __launch_bounds__(kScoreThreads, 3) void block_score_kernel(SelectArgs a, int iters, int chunks) {
    extern __shared__ __align__(16) float kept_lds[];  // [waves][tokens][16 iters], places [waves][16 iters]
    constexpr int KS = ScoreTile<HD, false>::KS, STEP = 16 * kScoreWaves;
    const int lane = threadIdx.x & 63, m = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), nkv = a.b.pg.nkv;
    const int chunk = (int)(blockIdx.x % chunks), rest = (int)(blockIdx.x / chunks), g = rest % nkv, tile = rest / nkv;
    const int first = a.t0 + tile * a.tokens, last = min(first + a.tokens, a.t1);
    const int lo = max(chunk * iters * STEP, a.b.n_first & ~15) + 16 * wave, top = (chunk + 1) * iters * STEP;
    float* kept = kept_lds + wave * a.tokens * 16 * iters;
    int* places = reinterpret_cast<int*>(kept_lds + kScoreWaves * a.tokens * 16 * iters) + wave * 16 * iters;
    ScoreTile<HD, false> st;
    bool staged = false;
    for (int t = first; t < last;) {
        const TokenAt x = token_at(a.b.pg, t);
        if (x.s < 0) {
            ++t;
            continue;
        }
        const int stop = min(t - x.i + x.n, last);  // the run of this sequence's tokens
        const int hi = min(rivals(a.b, TokenAt{x.s, x.i + stop - 1 - t, x.cached, x.n}).end, top);
        if (hi > lo) {
            const int steps = (hi - lo + STEP - 1) / STEP;
            find_places(a, x.s, lo, STEP, steps, hi, places, lane);
            int place = places[m];
            half8 v[KS];
#pragma unroll
            for (int i = 0; i < KS; ++i) v[i] = bounds_at<HD>(a, place, g, kk)[4 * i];
            if (!staged) st.stage(a, first, last, g, m, kk), staged = true;
            for (int j = 0; j < steps; ++j) {
                const int place_next = places[16 * min(j + 1, steps - 1) + m];
                const half8* p = bounds_at<HD>(a, place_next, g, kk);
                const auto bounds = [&](int i) __attribute__((always_inline)) {
                    const f16x8 y = v[i];
                    v[i] = p[4 * i];  // the next step's
                    return y;
                };
                st.score(a, bounds, place, kept + 16 * j, 16 * iters, m, kk);
                place = place_next;
            }
            st.flush(a, kept, 16 * iters, steps, lo, STEP, first, t, stop, g, lane);
        }
        t = stop;
    }
}

// Many tokens: a workgroup takes four tiles, a wave each, and 16 `iters` blocks, whose
// bounds the waves bring into LDS together, two steps ahead in registers.  512 tokens,
// 469 blocks: 26 us, of which waves wait half; bounds straight into every wave's
// registers, as above, take 8 KB of loads a step from the L2s for each of them.
template <int HD>
__global__ __launch_bounds__(kScoreThreads, 2) void block_score_rows_kernel(SelectArgs a, int iters, int chunks) {
    extern __shared__ __align__(16) float kept_lds[];  // [waves][tokens][16 iters], places [waves][16 iters]
    constexpr int KS = ScoreTile<HD, true>::KS, OWN = KS < kScoreWaves ? 1 : KS / kScoreWaves;  // pieces a wave brings
    __shared__ half8 ring[2][KS][64];
    const int lane = threadIdx.x & 63, m = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), nkv = a.b.pg.nkv;
    const int chunk = (int)(blockIdx.x % chunks), rest = (int)(blockIdx.x / chunks), g = rest % nkv, tile = rest / nkv;
    const int first = a.t0 + kScoreWaves * tile * a.tokens, last = min(first + kScoreWaves * a.tokens, a.t1);
    const int mine = first + wave * a.tokens;  // the wave's first token
    const int lo = max(chunk * iters * 16, a.b.n_first & ~15), top = (chunk + 1) * iters * 16;
    const int piece0 = min(wave * OWN, KS - OWN);  // (HD = 32: waves that bring a piece again)
    float* kept = kept_lds + wave * a.tokens * 16 * iters;
    int* places = reinterpret_cast<int*>(kept_lds + kScoreWaves * a.tokens * 16 * iters) + wave * 16 * iters;
    ScoreTile<HD, true> st;
    bool staged = false;
    for (int t = first; t < last;) {  // (all waves together)
        const TokenAt x = token_at(a.b.pg, t);
        if (x.s < 0) {
            ++t;
            continue;
        }
        const int stop = min(t - x.i + x.n, last);
        const int hi = min(rivals(a.b, TokenAt{x.s, x.i + stop - 1 - t, x.cached, x.n}).end, top);
        if (hi > lo) {
            const int steps = (hi - lo + 15) >> 4;
            find_places(a, x.s, lo, 16, steps, hi, places, lane);
            // step `at`'s place and pieces, steps in their order (past the last the last's again)
            int at = 0;
            const auto fetch = [&](half8 (&v)[OWN]) __attribute__((always_inline)) {
                const int place = places[16 * min(at++, steps - 1) + m];
                const half8* p = bounds_at<HD>(a, place, g, kk);
#pragma unroll
                for (int i = 0; i < OWN; ++i) v[i] = p[4 * (piece0 + i)];
                return place;
            };
            const auto keep = [&](const half8 (&v)[OWN], int slot) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < OWN; ++i) ring[slot][piece0 + i][lane] = v[i];
            };
            half8 v0[OWN], v1[OWN], v2[OWN];
            int place = fetch(v0), place1 = fetch(v1), place2 = fetch(v2);
            if (!staged) st.stage(a, mine, min(mine + a.tokens, a.t1), g, m, kk), staged = true;
            keep(v0, 0);
            __syncthreads();
            int j = 0;
            // Three steps by name: registers that loads are on their way to cannot be moved.
            // (And all three each time, past the last one too, unused: with ways out in
            // between every round began by waiting for all loads.)
            const auto step = [&](half8 (&into)[OWN], const half8 (&next)[OWN]) __attribute__((always_inline)) {
                const int place3 = fetch(into);
                const auto bounds = [&](int i) __attribute__((always_inline)) { return ring[j & 1][i][lane]; };
                st.score(a, bounds, place, kept + 16 * j, 16 * iters, m, kk);
                ++j;
                keep(next, j & 1);
                place = place1, place1 = place2, place2 = place3;
                __syncthreads();
            };
            while (j < steps) step(v0, v1), step(v1, v2), step(v2, v0);
            st.flush(a, kept, 16 * iters, steps, lo, 16, mine, max(t, mine), min(stop, min(mine + a.tokens, a.t1)), g, lane);
        }
        t = stop;
    }
}

// A block's score in 64 bits as order_key has it, by 16 lanes (in all of them); q: the
// kv head's q heads
template <int HD>
__device__ __forceinline__ uint64_t exact_key(const BlockArgs& a, int s, int b, int g, const float4* q, int group) {
    constexpr int PER = HD / 16;
    typedef _Float16 piece __attribute__((ext_vector_type(PER)));
    typedef float qpiece __attribute__((ext_vector_type(PER)));
    const int d = (threadIdx.x & 15) * PER;
    const int64_t place = block_place(a, s, b);
    const __half* p = a.bounds + (max(place, (int64_t)0) * a.pg.nkv + g) * 2 * HD + d;
    const piece least = *reinterpret_cast<const piece*>(p), greatest = *reinterpret_cast<const piece*>(p + HD);
    double best = -INFINITY;
    for (int h = 0; h < group; ++h) {
        const qpiece y = *reinterpret_cast<const qpiece*>(reinterpret_cast<const float*>(q) + h * HD + d);
        double sum = 0.;
#pragma unroll
        for (int e = 0; e < PER; ++e)
            sum += (double)(y[e] <= 0.f ? 0.f : y[e]) * (double)greatest[e] +
                   (double)(y[e] >= 0.f ? 0.f : y[e]) * (double)least[e];
        sum += dpp_d<0xb1>(sum);  // over the row of 16 lanes
        sum += dpp_d<0x4e>(sum);
        sum += dpp_d<0x141>(sum);
        sum += dpp_d<0x140>(sum);
        best = best != best ? best : sum > best || sum != sum ? sum : best;
    }
    return place < 0 ? 0 : order_key(best);
}

// Workgroup (token, kv head).  The scores' range in equal bins; the bin that the
// n-th largest falls into; what lies above it by more than scores are off is taken,
// what lies below by as much is not, and the few in between are ordered by their
// scores in 64 bits.  Where they are not few, or scores are not finite, all of them
// are, a few bits of the n-th largest at a time.
// One token's 8 rows of 938 blocks 10 us, one after the other: its lengths 0.7, scores
// 2, bins 1, those that are open 0.8, their 64 bits 2.6, the list 1.4.  512 tokens' 4,096
// rows of 469 blocks 22: some 1,000 vector instructions a wave.
constexpr int kPickKeys = 4096, kOpenMax = 128;
template <int HD, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void block_pick_kernel(SelectArgs a) {
    constexpr int WAVES = THREADS / 64, BINS = 2 * THREADS, DIGIT = THREADS < 256 ? 4 : 8, DIGITS = 1 << DIGIT;
    __shared__ uint32_t bins[BINS], wsum[WAVES];
    __shared__ float red[WAVES][3];
    extern __shared__ float keys_lds[];  // [kPickKeys], of n_blocks at most
    __shared__ uint32_t found[2], n_open, n_above;  // a bin, keys wanted of it; blocks that are open, taken
    __shared__ int open[kOpenMax];
    __shared__ uint64_t open_key[kOpenMax];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nkv = a.b.pg.nkv;
    const int t = a.t0 + (int)(blockIdx.x / nkv), g = (int)(blockIdx.x % nkv);
    const TokenAt x = token_at(a.b.pg, t);
    if (x.s < 0) return;
    const Rivals r = rivals(a.b, x);
    int* out = a.chosen + ((int64_t)t * nkv + g) * a.b.n_select;
    if (r.end == 0) {
        for (int i = tid; i < a.b.n_select; i += THREADS) out[i] = i <= r.own ? i : -1;
        return;
    }
    const int n0 = a.b.n_first, n = r.end - n0, want = a.b.n_select - n0 - a.b.n_last;
    for (int i = tid; i < n0; i += THREADS) out[i] = i;
    for (int i = tid; i < a.b.n_last; i += THREADS) out[n0 + want + i] = r.end + i;
    if (want == 0) return;
    float* row = a.scores + ((int64_t)(t - a.t0) * nkv + g) * 2 * a.ld;
    float* scores = row + n0;
    // (q comes while the scores do)
    constexpr int PIECES = 2 * HD > THREADS ? 2 * HD / THREADS : 1;
    __shared__ float4 q[2 * HD];  // [group][HD]
    const int q_pieces = a.group * (HD / 4);
    float4 q_mine[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
        q_mine[i] = reinterpret_cast<const float4*>(a.q + ((int64_t)t * a.nh + g * a.group) * HD)
            [min(tid + i * THREADS, q_pieces - 1)];
    const auto inclusive = [&](uint32_t v) {  // over the workgroup
        v = wave_scan(v);
        __syncthreads();
        if (lane == 63) wsum[wave] = v;
        __syncthreads();
        for (int w = 0; w < wave; ++w) v += wsum[w];
        return v;
    };

    // the range of the scores, the most one is off
    const bool held = n <= kPickKeys;
    float least = INFINITY, most = -INFINITY, off = 0.f;
    for (int i = tid; i < BINS; i += THREADS) bins[i] = 0;
    if (tid == 0) n_open = n_above = 0;
    for (int i = tid; i < n; i += THREADS) {
        const float s = scores[i];
        if (held) keys_lds[i] = s;
        if (s > -INFINITY) least = fminf(least, s);
        most = fmaxf(most, s);
        if (s != s) off = INFINITY;
    }
    for (int i = (n0 >> 4) + tid; i <= (r.end - 1) >> 4; i += THREADS) off = fmaxf(off, row[a.ld + i]);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) q[min(tid + i * THREADS, q_pieces - 1)] = q_mine[i];
    least = -wave_max_all(-least), most = wave_max_all(most), off = wave_max_all(off);
    if (lane == 0) red[wave][0] = least, red[wave][1] = most, red[wave][2] = off;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) least = fminf(least, red[w][0]), most = fmaxf(most, red[w][1]), off = fmaxf(off, red[w][2]);
    const auto key = [&](int i) { return held ? keys_lds[i] : scores[i]; };
    bool exact = !(off < INFINITY) || !(fabsf(least) < INFINITY) || !(fabsf(most) < INFINITY);
    float above = 0.f, below = 0.f;
    int taken_above = 0;
    if (!exact) {
        const float range = most - least, scale = range > 0.f ? (float)(BINS - 1) / range : 0.f;
        const auto bin = [&](float s) { return min((int)((s - least) * scale), BINS - 1); };
        exact = !(scale < INFINITY) || !(range < INFINITY);
        for (int i = tid; i < n && !exact; i += THREADS) {
            const float s = key(i);
            if (s > -INFINITY) atomicAdd(&bins[bin(s)], 1u);
        }
        __syncthreads();
        // bins from the top, two a thread
        const uint32_t c0 = bins[BINS - 1 - 2 * tid], c1 = bins[BINS - 2 - 2 * tid];
        const uint32_t upto = inclusive(c0 + c1), before = upto - c0 - c1, w = (uint32_t)want;
        if (tid == 0) found[0] = 0xffffffffu;
        __syncthreads();
        if (before < w && before + c0 >= w) found[0] = (uint32_t)(BINS - 1 - 2 * tid);
        else if (before + c0 < w && upto >= w) found[0] = (uint32_t)(BINS - 2 - 2 * tid);
        __syncthreads();
        if (found[0] == 0xffffffffu) exact = true;  // (fewer blocks are there than wanted)
        else {
            // the bin's edges, with what the sums above round
            const float width = range / (float)(BINS - 1), at = least + (float)found[0] * width;
            const float slack = 2.f * off + range * 0x1p-18f + fmaxf(fabsf(least), fabsf(most)) * 0x1p-20f;
            above = at + width + slack, below = at - slack;
            uint32_t mine = 0;  // (the wave's)
            for (int i = tid; i < n; i += THREADS) {
                const float s = key(i);
                mine += (uint32_t)__popcll(__ballot(s > above));
                if (s >= below && s <= above) {
                    const uint32_t e = atomicAdd(&n_open, 1u);
                    if (e < (uint32_t)kOpenMax) open[e] = i;
                }
            }
            mine = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine);  // (its first lane took part to the end)
            if (lane == 0) atomicAdd(&n_above, mine);
            __syncthreads();
            taken_above = (int)n_above;
            exact = n_open > (uint32_t)kOpenMax;
        }
    }
    if (!exact) {
        const int ours = (int)n_open, need = want - taken_above;
        if (ours != need) {
            for (int j = tid / 16; j < ours; j += THREADS / 16) {
                const uint64_t k = exact_key<HD>(a.b, x.s, n0 + open[j], g, q, a.group);
                if ((tid & 15) == 0) open_key[j] = k;
            }
            __syncthreads();
            for (int i = tid; i < ours; i += THREADS) {
                int rank = 0;
                for (int j = 0; j < ours; ++j)
                    rank += open_key[j] > open_key[i] || (open_key[j] == open_key[i] && open[j] < open[i]);
                const float s = rank < need ? INFINITY : -INFINITY;
                if (held) keys_lds[open[i]] = s;
                else scores[open[i]] = s;
            }
            __syncthreads();
        }
        const bool edge = ours == need;  // (all that are open are taken)
        // each wave a stretch of the blocks: how many it takes, then which
        const auto take = [&](int i) {
            if (i >= n) return false;
            const float s = key(i);
            return edge ? s >= below : s > above;
        };
        const int stretch = (n + 64 * WAVES - 1) / (64 * WAVES) * 64, i0 = wave * stretch, i1 = min(i0 + stretch, n);
        uint32_t count = 0;
        for (int i = i0; i < i1; i += 64) count += (uint32_t)__popcll(__ballot(i + lane < i1 && take(i + lane)));
        if (lane == 0) wsum[wave] = count;
        __syncthreads();
        int at = n0;
        for (int w = 0; w < wave; ++w) at += (int)wsum[w];
        for (int i = i0; i < i1; i += 64) {
            const bool on = i + lane < i1 && take(i + lane);
            const uint64_t all = __ballot(on);
            if (on) out[at + (int)__popcll(all & ((1ull << lane) - 1))] = n0 + i + lane;
            at += (int)__popcll(all);
        }
        return;
    }

    // all scores in 64 bits, where the others were
    uint64_t* keys = reinterpret_cast<uint64_t*>(row);
    for (int i = tid / 16; i < n; i += THREADS / 16) {
        const uint64_t k = exact_key<HD>(a.b, x.s, n0 + i, g, q, a.group);
        if ((tid & 15) == 0) keys[i] = k;
    }
    __syncthreads();
    uint64_t prefix = 0;
    uint32_t need = (uint32_t)want;
    int shift = 64;
    for (;;) {
        shift -= DIGIT;
        if (tid < DIGITS) bins[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t k = keys[i];
            if (shift + DIGIT == 64 || k >> (shift + DIGIT) == prefix) atomicAdd(&bins[k >> shift & (DIGITS - 1)], 1u);
        }
        __syncthreads();
        const uint32_t c = tid < DIGITS ? bins[DIGITS - 1 - tid] : 0, upto = inclusive(c);
        if (upto >= need && upto - c < need) found[0] = DIGITS - 1 - tid, found[1] = need - (upto - c);
        __syncthreads();
        prefix = prefix << DIGIT | found[0], need = found[1];
        const bool all = bins[found[0]] == need;
        __syncthreads();
        if (all || shift == 0) break;
    }
    // those above the prefix, and the first `need` of those with it
    int done = n0;
    uint32_t ties = 0;
    for (int i0 = 0; i0 < n; i0 += THREADS) {
        const int i = i0 + tid;
        const uint64_t k = i < n ? keys[i] >> shift : 0;
        const bool larger = i < n && k > prefix, same = i < n && k == prefix;
        const uint32_t before = inclusive(same) - same + ties;
        const bool take = larger || (same && before < need);
        const uint32_t upto = inclusive(take);
        if (take) out[done + upto - 1] = n0 + i;
        __syncthreads();
        if (tid == THREADS - 1) found[0] = upto, found[1] = before + same;
        __syncthreads();
        done += found[0], ties = found[1];
        __syncthreads();
    }
}

// ---- attention -------------------------------------------------------------

struct BlockAttnArgs {
    TileArgs t;
    const int* chosen;  // [n_tokens][nkv][n_select]
    int n_select, block_shift, n_blocks, splits, words, once;  // once: rows that a call reads do not stay for the next
    int lists;  // LDS bytes before the lists
};

// Workgroup (kv head, tile and split): the blocks that any of a sequence's tokens
// in the tile has chosen, found as bits in LDS, then a share of their stages.
template <int HD, int R>
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
                    a.t.ml[(index * nkv + g) * R + (t - first) * (int)a.t.group + i] = make_float2(0.f, -1.f);
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
        attend_tile<HD, R, kListed>(a.t, it, g, a.once, smem);
        t += n;
        if (t < last) __syncthreads();
    }
}

// (splits make few tiles into some two workgroups a CU, so units are few)
constexpr int kMergeLanes = 4, kMergeUnits = kJoinThreads / kMergeLanes;
struct BlockMergeArgs {
    const float* part;
    const float2* ml;
    float* att;
    int64_t total;  // units of four dims, of all tokens
    int nkv, group, tokens, splits, rows;
};

template <int HD>
__global__ __launch_bounds__(kJoinThreads) void blocks_merge_kernel(BlockMergeArgs a) {
    const int64_t u = (int64_t)blockIdx.x * kMergeUnits + threadIdx.x % kMergeUnits;
    const int64_t head = min(u, a.total - 1) / (HD / 4);
    const int d = 4 * (int)(u % (HD / 4)), nh = a.nkv * a.group;
    const int64_t t = head / nh, tile = t / a.tokens;
    const int hq = (int)(head - t * nh), g = hq / a.group;
    const int row = (int)(t - tile * a.tokens) * a.group + hq - g * a.group;
    const auto place = [&](int z) { return ((tile * a.splits + z) * a.nkv + g) * a.rows + row; };
    const auto where = [&](int z, float2& x, float4& v) __attribute__((always_inline)) {
        const int64_t at = place(z);
        x = a.ml[at];
        v = *reinterpret_cast<const float4*>(a.part + at * HD + d);
    };
    const bool any = u < a.total && !(a.ml[place(0)].y < 0.f);  // (else no sequence's)
    join_parts<kMergeLanes>(a.splits, where, any ? a.att + head * HD + d : nullptr);
}

BlockSize block_size(const BlockArgs& a, int nh) {
    return BlockSize{a.pg.n_seq, a.pg.n_tokens, a.n_blocks, a.pg.nkv, nh / a.pg.nkv, a.n_select, 1 << a.block_shift,
                     device_cus()};
}

BlockArgs block_args(const PagedArgs& pg, const BlocksOf& b) {
    return BlockArgs{pg, b.bounds, b.block_shift, b.n_first, b.n_last, b.n_select, (int)blocks_of_table(pg, b.block_shift)};
}

template <int HD, int R>
int launch_rows(const BlockAttnArgs& a, int64_t tiles, hipStream_t st) {
    constexpr int RING = lds_bytes(HD, R);
    BlockAttnArgs args = a;
    args.lists = std::max(RING, (int)((a.t.tokens * (size_t)a.words * 4 + 255) / 256 * 256));
    const size_t lds = (size_t)args.lists + kListMax * 6;
    static bool attr_set = false;
    if (!attr_set) {
        if (hipFuncSetAttribute((const void*)attention_blocks_kernel<HD, R>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                std::max(RING, kBitBytes) + kListMax * 6) != hipSuccess)
            return MXH_ERR_HIP;
        attr_set = true;
    }
    const int64_t items = tiles * a.splits, y = std::min<int64_t>(items, 32768);
    hipLaunchKernelGGL((attention_blocks_kernel<HD, R>),
                       dim3((unsigned)a.t.pg.nkv, (unsigned)y, (unsigned)((items + y - 1) / y)), dim3(kThreads), lds, st,
                       args);
    if (a.splits > 1) {
        const int64_t total = (int64_t)a.t.pg.n_tokens * a.t.nh() * (HD / 4);
        const BlockMergeArgs m{a.t.part, a.t.ml, a.t.att, total, a.t.pg.nkv, (int)a.t.group, (int)a.t.tokens, a.splits, R};
        hipLaunchKernelGGL(blocks_merge_kernel<HD>, dim3((unsigned)((total + kMergeUnits - 1) / kMergeUnits)),
                           dim3(kJoinThreads), 0, st, m);
    }
    return MXH_OK;
}

template <int HD>
int launch_attention(const BlockAttnArgs& a, int rows, int64_t tiles, hipStream_t st) {
    return rows == 32 ? launch_rows<HD, 32>(a, tiles, st) : launch_rows<HD, 16>(a, tiles, st);
}

template <int HD>
void launch_select(const SelectArgs& a, hipStream_t st) {
    const int64_t n = a.t1 - a.t0, tiles = (n + a.tokens - 1) / a.tokens, nkv = a.b.pg.nkv;
    if (a.b.n_blocks > a.b.n_select) {  // (else no token has more blocks than it takes)
        // steps of a workgroup: so many that there are some four workgroups a CU
        const bool many = tiles >= kScoreWaves && a.tokens > 1;
        const int64_t rows = many ? (tiles + kScoreWaves - 1) / kScoreWaves : tiles, step = many ? 16 : 16 * kScoreWaves;
        const int64_t one = (a.b.n_blocks + step - 1) / step;
        int64_t iters = one * rows * nkv / (many ? 512 : 1024);
        iters = std::max<int64_t>(1, std::min<int64_t>({one, iters, 64 / a.tokens, 15}));  // (at most 26 KB of LDS)
        if (many) iters = (iters + 2) / 3 * 3;  // (as its steps are taken)
        const int64_t chunks = (one + iters - 1) / iters;
        const size_t lds = sizeof(float) * kScoreWaves * (a.tokens + 1) * 16 * (size_t)iters;
        const dim3 grid((unsigned)(chunks * rows * nkv));
        if (many)
            hipLaunchKernelGGL(block_score_rows_kernel<HD>, grid, dim3(kScoreThreads), lds, st, a, (int)iters, (int)chunks);
        else hipLaunchKernelGGL(block_score_kernel<HD>, grid, dim3(kScoreThreads), lds, st, a, (int)iters, (int)chunks);
    }
    const dim3 rows((unsigned)(n * nkv));
    const size_t lds = sizeof(float) * std::min(a.b.n_blocks, kPickKeys);
    // four waves a row as long as all rows are taken at once, else two: 4,096 rows of 469
    // blocks 26.4 and 22.2 us, 384 of up to 500 9.4 and 12.2
    if (n * nkv > 8 * (int64_t)device_cus())
        hipLaunchKernelGGL((block_pick_kernel<HD, 128>), rows, dim3(128), lds, st, a);
    else hipLaunchKernelGGL((block_pick_kernel<HD, 256>), rows, dim3(256), lds, st, a);
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

size_t select_blocks_work_bound(const PagedArgs& pg, const BlocksOf& b) {
    return select_work_bound(pg.n_tokens, blocks_of_table(pg, b.block_shift), pg.nkv);
}

void select_blocks_launch(const PagedArgs& pg, const BlocksOf& b, const float* q, int nh, int hd, int* chosen,
                          void* work, hipStream_t st) {
    const BlockArgs ba = block_args(pg, b);
    SelectArgs a{ba, q, nh, nh / pg.nkv, 0, 0, 0, (int)select_row(ba.n_blocks), static_cast<float*>(work), chosen};
    // tokens by themselves also where that makes little work (64 blocks of a token and kv
    // head, 1.5 a CU), as those of a tile wait for one another's sequences.  Up to 8
    // tokens of 6 sequences of 16 blocks 5.0 us, in tiles 16.9, up to 15 of 4 of 28 5.3 and
    // 12.4; 8 of one of 469 (2) 9.4 and 8.4, 15 (4) 15.0 and 9.5, up to 30 of 4 of 156 (7)
    // 15.5 and 12.9
    const bool alone = pg.n_tokens <= 2 * (int64_t)pg.n_seq ||
                       2 * (int64_t)pg.n_tokens * pg.nkv * ((ba.n_blocks + 63) / 64) <= 3 * (int64_t)device_cus();
    a.tokens = alone ? 1 : 16 / a.group;
    const int64_t step = select_tokens(pg.n_tokens, ba.n_blocks, pg.nkv);
    for (int64_t t = 0; t < pg.n_tokens; t += step) {
        a.t0 = (int)t, a.t1 = (int)std::min<int64_t>(t + step, pg.n_tokens);
        if (hd == 32) launch_select<32>(a, st);
        else if (hd == 64) launch_select<64>(a, st);
        else launch_select<128>(a, st);
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
    // single tokens whose rows are more than half of the last cache's 256 MB: 48 of them
    // with 1,280 rows for each of 8 kv heads of 128 53 us, 47 so
    const bool once = pg.n_tokens <= 2 * (int64_t)pg.n_seq && (double)pg.n_tokens * pg.nkv * b.n_select * size.block_rows * hd * 4 > 128e6;
    const BlockAttnArgs a{{pg, q, att, part, reinterpret_cast<float2*>(part + (size_t)tiles * splits * pg.nkv * block_rows_of_tile(size) * hd),
                           1.4426950408889634f / sqrtf((float)hd), group, (uint32_t)block_tokens(size),
                           (65536 + group - 1) / group},
                          chosen, b.n_select, b.block_shift, ba.n_blocks, splits, (ba.n_blocks + 31) / 32, once, 0};
    const int rows = block_rows_of_tile(size);
    return hd == 32   ? launch_attention<32>(a, rows, tiles, st)
           : hd == 64 ? launch_attention<64>(a, rows, tiles, st)
                      : launch_attention<128>(a, rows, tiles, st);
}

}  // namespace mxh
