// mxh_paged.h — a batch of packed tokens over a paged K/V cache, as the
// kernels see it (host + device).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxh_device.h"
#include "mxh_paged_plan.h"

namespace mxh {

// One layer of the pool and the batch; device pointers.  Nothing that the
// arrays hold is trusted: ids, lengths and parents are bounded where they are read.
struct PagedArgs {
    __half *k, *v;  // the layer's first page
    const int *start, *cached, *table, *parent;
    int n_seq, n_tokens, table_ld, n_pages;
    int page_shift, nkv;  // page_rows = 1 << page_shift
};

// Row `row` of sequence s as a row of the pool, -1 where it does not exist.
__device__ __forceinline__ int64_t paged_row(const PagedArgs& a, int s, int row) {
    const int p = row >> a.page_shift;
    if (row < 0 || p >= a.table_ld) return -1;
    const int id = a.table[(size_t)s * a.table_ld + p];
    if ((unsigned)id >= (unsigned)a.n_pages) return -1;
    return ((int64_t)id << a.page_shift) + (row & ((1 << a.page_shift) - 1));
}

// The sequence that token row t (uniform, below n_tokens) belongs to, -1 for
// none: the number of sequences that end at or before t, counted by the wave:
// the bounds of up to 64 equal parts of the list first, then those in a part.
__device__ __forceinline__ int paged_seq_of(const PagedArgs& a, int t) {
    const int lane = threadIdx.x & 63, part = (a.n_seq + 63) / 64;
    int s = 0;
    if (part > 1) {
        const int e = (lane + 1) * part;
        s = part * (int)__popcll(__ballot(e <= a.n_seq && a.start[min(e, a.n_seq)] <= t));
    }
    const int e = s + lane + 1;  // (bounds past the part's are above t)
    s += (int)__popcll(__ballot(e <= a.n_seq && a.start[min(e, a.n_seq)] <= t));
    return s < a.n_seq && a.start[s] >= 0 && a.start[s] <= t ? s : -1;
}

// The parent of token `lane` of a drafted tree (`first`: the sequence's first
// token row, n of them, at most 64), -1 for a root and past the tree.
__device__ __forceinline__ int tree_parent(const PagedArgs& a, int first, int n) {
    const int lane = threadIdx.x & 63, p = lane < n ? a.parent[first + lane] : -1;
    return p < -1 || p >= lane ? -1 : p;
}

// Lane i of the wave gets the bits of token i and its ancestors, from the
// lanes' parents.  Every round a lane joins the mask of the token it points to
// and then points to what that one points to: 2^r ancestors after r rounds.
__device__ __forceinline__ uint64_t tree_path(int p) {
    const int lane = threadIdx.x & 63;
    uint64_t mask = 1ull << lane;
#pragma unroll
    for (int r = 0; r < 6; ++r) {
        const int from = p < 0 ? lane : p;
        const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)mask, from);
        const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)(mask >> 32), from);
        const int next = __shfl(p, from);
        mask |= ((uint64_t)hi << 32) | lo;
        p = p < 0 ? -1 : next;
    }
    return mask;
}

// lane i's bits, in every lane (i below 64, any lane's own)
__device__ __forceinline__ uint64_t path_of(uint64_t paths, int i) {
    const uint64_t hi = (uint32_t)__shfl((int)(uint32_t)(paths >> 32), i);
    return hi << 32 | (uint32_t)__shfl((int)(uint32_t)paths, i);
}

// attention over the paged cache (mxh_paged_attn.hip)
size_t attention_paged_work_bytes(const PagedArgs& a, int nh, int hd);  // of this batch
size_t attention_paged_work_bound(const PagedArgs& a, int nh, int hd);  // of any up to its n_seq, n_tokens, table_ld
int attention_paged_launch(const PagedArgs& a, const float* q, int nh, int hd, float* att, void* work, hipStream_t st);

}  // namespace mxh
