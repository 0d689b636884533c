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
