// mh_lanes.h -- pieces that the routers share: rows held by groups of neighbouring lanes, their reductions, and the 8
// largest of a row by sorted lists.
#pragma once

#include <hip/hip_runtime.h>

#include "mh_internal.h"

namespace mh {

constexpr int kMaxExperts = 1024;
constexpr int kMaxChosen = 64;

// Reductions over groups of L neighbouring lanes, the result in every lane.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
template <int L, typename Op>
__device__ __forceinline__ int group_red(int v, Op op) {
    if (L >= 2) v = op(v, dpp<0xB1>(v));    // lanes 1 0 3 2
    if (L >= 4) v = op(v, dpp<0x4E>(v));    // lanes 2 3 0 1
    if (L >= 8) v = op(v, dpp<0x141>(v));   // 8 lanes mirrored: the other quad's
    if (L >= 16) v = op(v, dpp<0x140>(v));  // 16 lanes mirrored
    if (L >= 32) v = op(v, __shfl_xor(v, 16));
    if (L >= 64) v = op(v, __shfl_xor(v, 32));
    return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
    return __int_as_float(group_red<L>(__float_as_int(v), [](int a, int b) {
        return __float_as_int(__builtin_fmaxf(__int_as_float(a), __int_as_float(b)));
    }));
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    return __int_as_float(group_red<L>(__float_as_int(v), [](int a, int b) {
        return __float_as_int(__int_as_float(a) + __int_as_float(b));
    }));
}

// A float as an integer of the same order; NaN below every number, -0 as +0. Below them what is taken or past
// the experts.
constexpr int kTaken = INT32_MIN;
__device__ __forceinline__ int sort_key(float v) {
    const int b = __float_as_int(v + 0.0f);
    return v != v ? kTaken + 1 : (b < 0 ? b ^ 0x7fffffff : b);
}
__device__ __forceinline__ float key_value(int k) {
    return k == kTaken + 1 ? __builtin_nanf("") : __int_as_float(k < 0 ? k ^ 0x7fffffff : k);
}

// Loads lane l's elements of a row; past the experts minus infinity.
template <int L, int V>
__device__ __forceinline__ void load_row(const float* row, int E, int l, float* v) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        const int c = 4 * (i * L + l);
        if (c + 3 < E) {
            const vf4 q = *reinterpret_cast<const vf4u*>(row + c);
            v[4 * i] = q.x;
            v[4 * i + 1] = q.y;
            v[4 * i + 2] = q.z;
            v[4 * i + 3] = q.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = c + j < E ? row[c + j] : -__builtin_inff();
        }
    }
}

// A wavefront's LDS accesses so far come before those that follow.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// Lane l's elements to and from a row in LDS.
template <int L, int V>
__device__ __forceinline__ void put_row(float* row, int l, const float* v) {
    wave_sync();
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
        *reinterpret_cast<vf4*>(row + 4 * (i * L + l)) = vf4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    wave_sync();
}
template <int L, int V>
__device__ __forceinline__ void get_row(const float* row, int l, float* v) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        const vf4 q = *reinterpret_cast<const vf4*>(row + 4 * (i * L + l));
        v[4 * i] = q.x;
        v[4 * i + 1] = q.y;
        v[4 * i + 2] = q.z;
        v[4 * i + 3] = q.w;
    }
}

// Up to 8 choices: sorted lists. A logit's order and its index become the mantissa of a double in [1, 2), which
// the maximum and minimum of doubles sort, one instruction each and at full rate; a larger index is smaller.
// Each lane sorts its elements and keeps 8; neighbours' lists merge, and in the end each lane has the row's 8.
// [131072, 256], 8 of them: 84 us by rounds of a maximum, 60 by lists, which the sorting bounds (the read alone
// takes 24; loading a round ahead changed nothing).
constexpr int kList = 8;
__device__ __forceinline__ double list_key(int key, int index) {
    const uint32_t u = (uint32_t)key ^ 0x80000000u;
    return __hiloint2double((int)(0x3ff00000u | (u >> 22)), (int)(u << 10 | (uint32_t)(kMaxExperts - 1 - index)));
}
__device__ __forceinline__ int list_index(double d) { return kMaxExperts - 1 - (__double2loint(d) & (kMaxExperts - 1)); }
__device__ __forceinline__ int list_value(double d) {
    return (int)((((uint32_t)__double2hiint(d) << 22) | ((uint32_t)__double2loint(d) >> 10)) ^ 0x80000000u);
}
__device__ __forceinline__ double max_d(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double min_d(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ void order(double& a, double& b) {
    const double hi = max_d(a, b), lo = min_d(a, b);
    a = hi;
    b = lo;
}
__device__ __forceinline__ void sort4(double* d) {
    order(d[0], d[1]);
    order(d[2], d[3]);
    order(d[0], d[2]);
    order(d[1], d[3]);
    order(d[1], d[2]);
}
__device__ __forceinline__ void merge8(double* d) {  // 8 that rise and fall
#pragma unroll
    for (int s = 4; s > 0; s >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & s)) order(d[i], d[i + s]);
}
__device__ __forceinline__ void sort8(double* d) {
    sort4(d);
    sort4(d + 4);
    double t = d[4];
    d[4] = d[7];
    d[7] = t;
    t = d[5];
    d[5] = d[6];
    d[6] = t;
    merge8(d);
}
__device__ __forceinline__ void join8(double* d, const double* o) {  // the 8 largest of two sorted lists
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = max_d(d[i], o[7 - i]);
    merge8(d);
}
template <int STEP>
__device__ __forceinline__ int other_lane(int v) {
    return STEP == 1 ? dpp<0xB1>(v) : STEP == 2 ? dpp<0x4E>(v) : STEP == 4 ? dpp<0x141>(v) : STEP == 8 ? dpp<0x140>(v)
                                                                                                  : __shfl_xor(v, STEP);
}
template <int STEP, int L>
__device__ __forceinline__ void join_lanes(double* d) {
    if constexpr (STEP < L) {
        double o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = __hiloint2double(other_lane<STEP>(__double2hiint(d[i])), other_lane<STEP>(__double2loint(d[i])));
        join8(d, o);
        join_lanes<2 * STEP, L>(d);
    }
}
// From a lane's V keys in d to the row's 8 largest, in every lane.
template <int L, int V>
__device__ __forceinline__ void list_rows(double* d) {
    if constexpr (V == 4) {
        sort4(d);
    } else {
        sort8(d);
        if constexpr (V == 16) {
            sort8(d + 8);
            join8(d, d + 8);
        }
    }
    join_lanes<1, L>(d);
}
template <int L, int V>
__device__ __forceinline__ void row_list(const float* v, int E, int l, double* list) {
    double d[V < 8 ? 8 : V];
#pragma unroll
    for (int i = 0; i < (V < 8 ? 8 : V); ++i) {
        const int e = 4 * ((i / 4) * L + l) + (i & 3);
        d[i] = i < V && e < E ? list_key(sort_key(v[i < V ? i : 0]), e) : 1.0;
    }
    list_rows<L, V>(d);
#pragma unroll
    for (int i = 0; i < 8; ++i) list[i] = d[i];
}

}  // namespace mh
