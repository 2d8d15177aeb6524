// mxh_attn.h — device helpers that the flash-form attention kernels share.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

namespace mxh {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kPaScale = 64.f, kPaSlack = 8.f;  // P at most scale 2^slack

// row m of a 32-key block -> key (bits 2 and 3 swapped)
__device__ __forceinline__ int pa_pi(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

template <int HD>
__device__ __forceinline__ int pa_swz(int key) {
    constexpr int NCH = HD / 8, RS = HD == 128 ? 0 : HD == 64 ? 1 : 2;  // rows per 256 bytes = 1 << RS
    return (key >> RS) & (NCH - 1);
}

// the larger / the sum of a value in lanes l and l ^ 32, in both
__device__ __forceinline__ float pa_pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// p - h[HALF] in one instruction (written as C++ it is a conversion and a
// subtraction; exact)
template <int HALF>
__device__ __forceinline__ float pa_rest(float p, f16x2 h) {
    float d;
    if constexpr (HALF)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(p));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(p));
    return d;
}

// a and b as fp16 hi + lo, both rounded to nearest (one instruction for a
// pair): cut off, a probability's halves left the V sums 7e-8 to 9e-8 low
// against lrun.  hi is made opaque: where a is a product the compiler would
// round it to fp16 in one step for lo and in two for hi, and where the two
// differ (one in some thousand q values) lo repairs an error that hi does not
// have (rms error of 200 queries at 0, 32/8 heads of 128: 4.1e-6).
__device__ __forceinline__ void pa_split(float a, float b, f16x2& hi, f16x2& lo) {
    hi = __builtin_convertvector((f32x2{a, b}), f16x2);
    asm("" : "+v"(hi));
    lo = __builtin_convertvector((f32x2{pa_rest<0>(a, hi), pa_rest<1>(b, hi)}), f16x2);
}

}  // namespace mxh
