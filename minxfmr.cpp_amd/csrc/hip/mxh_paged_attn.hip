// mxh_paged_attn.hip — attention of packed tokens over a paged K/V cache
// (include/minxfmr_hip.h: mxh_attention_paged).
//
// Reference op: the attention of transformer.cpp:529-629 per token (scores
// q.k / sqrt(hd), softmax softmax.cpp:4-18, weighted sum of V rows), here over
// the rows of a sequence's pages, for drafted trees only along a token's path.
//
// One wave per token and head: 64 keys at a time, a key a lane for the scores,
// then the lanes turn to the dims for the sum of V rows.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "mxh_internal.h"
#include "mxh_paged.h"

namespace mxh {

namespace {

template <int HD>
__global__ __launch_bounds__(64) void attention_paged_simple_kernel(PagedArgs a, const float* __restrict__ q, int nh,
                                                                    float scale2, float* __restrict__ att) {
    __shared__ float qs[HD], ps[64];
    __shared__ int64_t at[64];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int s = paged_seq_of(a, t);
    if (s < 0) return;
    const int first = a.start[s], i = t - first, cached = min(max(a.cached[s], 0), 1 << 30);
    uint64_t path = ~0ull;
    if (a.parent) {
        const uint64_t mine = tree_path(a, first, min(min(a.start[s + 1], a.n_tokens) - first, kTreeMax));
        if (i >= kTreeMax) return;
        path = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(mine >> 32), i) << 32) | (uint32_t)__shfl((int)(uint32_t)mine, i);
    }
    const size_t at0 = ((size_t)t * nh + h) * HD;
    for (int d = lane; d < HD; d += 64) qs[d] = q[at0 + d] * scale2;
    __syncthreads();
    const int g = h / (nh / a.nkv);
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (int k0 = 0; k0 < cached + i + 1; k0 += 64) {
        const int key = k0 + lane;
        bool on = key <= cached + i && (key < cached || !a.parent || (path >> (key - cached) & 1));
        const int64_t row = on ? paged_row(a, s, key) : -1;
        on = row >= 0;
        float sc = -INFINITY;
        if (on) {
            const __half* kp = a.k + (row * a.nkv + g) * HD;
            sc = 0.f;
            for (int d = 0; d < HD; ++d) sc += qs[d] * __half2float(kp[d]);
        }
        const float mx = fmaxf(m, wave_max(sc));
        const float alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
        const float p = on ? exp2f(sc - mx) : 0.f;
        m = mx;
        l = l * alpha + wave_sum(p);
        ps[lane] = p;
        at[lane] = row;
        __syncthreads();
        o[0] *= alpha, o[1] *= alpha;
        for (int j = 0; j < 64; ++j) {
            if (at[j] < 0) continue;
            const __half* vp = a.v + (at[j] * a.nkv + g) * HD;
            for (int u = 0; u < 2; ++u)
                if (lane + 64 * u < HD) o[u] += ps[j] * __half2float(vp[lane + 64 * u]);
        }
        __syncthreads();
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < HD) att[at0 + lane + 64 * u] = o[u] * inv;
}

}  // namespace

size_t attention_paged_work_bytes(const PagedArgs&, int, int) { return 0; }

int attention_paged_launch(const PagedArgs& a, const float* q, int nh, int hd, float* att, void*, hipStream_t st) {
    const dim3 grid((unsigned)a.n_tokens, (unsigned)nh);
    const float scale2 = 1.4426950408889634f / sqrtf((float)hd);
    switch (hd) {
    case 32: hipLaunchKernelGGL(attention_paged_simple_kernel<32>, grid, dim3(64), 0, st, a, q, nh, scale2, att); break;
    case 64: hipLaunchKernelGGL(attention_paged_simple_kernel<64>, grid, dim3(64), 0, st, a, q, nh, scale2, att); break;
    default: hipLaunchKernelGGL(attention_paged_simple_kernel<128>, grid, dim3(64), 0, st, a, q, nh, scale2, att); break;
    }
    return MXH_OK;
}

}  // namespace mxh
