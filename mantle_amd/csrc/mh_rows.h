// mh_rows.h -- pieces that the language-model losses share: exponentials that reach 0, and reductions over a
// workgroup in a fixed order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mh {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLog2eLo = 1.925963033500e-8f;  // log2(e) - kLog2e

// e^x to about an ulp for x <= 0: the rounding of x log2(e) is carried into the result. mexp stops at
// e^-88.4, as the reference does; here what a mask leaves is 0.
__device__ __forceinline__ float exp_neg(float x) {
    x = x < -1.0e4f ? -1.0e4f : x;  // keeps NaN, and infinity out of the fma
    const float t = x * kLog2e;
    const float r = __builtin_fmaf(x, kLog2eLo, __builtin_fmaf(x, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, r * 0.693147180559945f, e);
}

// e^x in 64 bits to about an ulp, for x of less than 700 (from -1000 down it is 0; a NaN stays one): 2^n e^r with n the whole
// number next to x log2(e), r = x - n ln 2 from ln 2 in two parts, and e^r by its series to r^13.
__device__ __forceinline__ double exp64(double x) {
    x = x < -1000.0 ? -1000.0 : x;
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(n, -0.69314718055994530942, x);
    r = __builtin_fma(n, -2.3190468138462996e-17, r);  // the rest of ln 2
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// Sums and maxima over a workgroup of W wavefronts; every thread gets the result. `red` holds W values and may
// be used again right after.
template <int W, typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (W == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) s += red[i];
    return s;
}
template <int W>
__device__ __forceinline__ float block_max(float v, float* red) {  // of numbers: a NaN is passed over
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o));
    if (W == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) s = __builtin_fmaxf(s, red[i]);
    return s;
}

}  // namespace mh
