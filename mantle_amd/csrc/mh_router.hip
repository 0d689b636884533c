// mh_router.hip -- a mixture-of-experts router: softmax over experts, the k largest logits of each row, their
// weights, how often each expert was chosen, the balance loss, and the gradient of the logits.
//
//   p = softmax(x); chosen = the k largest logits, ties to the lowest index; weights = p_chosen, normalised
//   over the chosen or not; f_e = counts_e / (n k); P_e = mean of p_e over the n kept rows; loss = E sum f_e P_e
//   with s = ug E / n and g the weights' gradient (0 where not chosen):
//     grad_j = p_j (A_j - sum_e A_e p_e),  A = g + s f                             (not normalised)
//     grad_j = w_j (g_j - sum_i g_i w_i) + p_j (s f_j - sum_e s f_e p_e)           (normalised)
//
// Bound by the logits' read and the gradient's write over long batches, by launches over short ones. L lanes
// hold a row in registers, V elements a lane in quads (element 4 (i L + lane) + c), so that the columns of a lane
// are the same for all its rows: the sums P_e and the loss's f_e stay in registers over the rows of a workgroup.
// Up to 8 choices come from sorted lists, more from rounds of a maximum over the lane's elements, then the row's
// lanes.
// Sums over rows are fp32 per workgroup and in a fixed order; counts are whole numbers.
#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxChosen = 64;
constexpr int kRThreads = 256;
constexpr int kRBlocks = 1024;  // workgroups of a forward at most: rows of its partials

struct RouterArg {
    const float* x;
    const int32_t* keep;  // or null: every row
    int64_t rows;
    int32_t experts, k;
    int32_t normalise, accumulate;
    // forward
    float* weights;
    int32_t* chosen;
    int32_t* counts;
    float* loss;
    float* part_p;     // [blocks][experts]
    int32_t* part_c;   // [blocks][experts]
    int32_t* part_n;   // [blocks] kept rows
    int32_t blocks;
    // backward
    float* grad;
    const float* gw;   // or null
    const float* ug;   // or null
    const int32_t* sel;
    const int32_t* cnt;
};

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

// v to e^(v - max); returns their sum and the maximum. Past the experts 0.
__device__ __forceinline__ float exp_diff(float v, float m) { return __builtin_amdgcn_exp2f((v - m) * kLog2e); }
template <int L, int V>
__device__ __forceinline__ float row_exp(float* v, float* top) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = __builtin_fmaxf(m, v[i]);
    m = group_max<L>(m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] = exp_diff(v[i], m);
        s += v[i];
    }
    *top = m;
    return group_sum<L>(s);
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
template <int L, int V>
__device__ __forceinline__ void row_list(const float* v, int E, int l, double* list) {
    double d[V < 8 ? 8 : V];
#pragma unroll
    for (int i = 0; i < (V < 8 ? 8 : V); ++i) {
        const int e = 4 * ((i / 4) * L + l) + (i & 3);
        d[i] = i < V && e < E ? list_key(sort_key(v[i < V ? i : 0]), e) : 1.0;
    }
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
#pragma unroll
    for (int i = 0; i < 8; ++i) list[i] = d[i];
}

// The counts and the loss from the workgroups' partials, by one workgroup of N threads: threads of 64 columns or
// as many as there are experts, the others along the partials. `red` and `buf` are LDS of N each.
template <int N>
__device__ void router_total(const RouterArg& a, float* red, float* buf) {
    int32_t n = 0;
    for (int b = threadIdx.x; b < a.blocks; b += N) n += a.part_n[b];
    n = block_sum<N / 64>(n, reinterpret_cast<int32_t*>(red));
    int32_t* buf_c = reinterpret_cast<int32_t*>(buf + N);
    int cols = 8;
    while (cols < 64 && cols < a.experts) cols *= 2;
    const int col = threadIdx.x % cols, part = threadIdx.x / cols, parts = N / cols;
    float s = 0.0f;
    for (int e0 = 0; e0 < a.experts; e0 += cols) {
        const int e = e0 + col;
        float p = 0.0f;
        int32_t c = 0;
        if (e < a.experts)
#pragma unroll 4
            for (int b = part; b < a.blocks; b += parts) {
                p += a.part_p[(int64_t)b * a.experts + e];
                c += a.part_c[(int64_t)b * a.experts + e];
            }
        __syncthreads();
        buf[threadIdx.x] = p;
        buf_c[threadIdx.x] = c;
        __syncthreads();
        if (part == 0 && e < a.experts) {
            for (int i = 1; i < parts; ++i) {
                p += buf[i * cols + col];
                c += buf_c[i * cols + col];
            }
            a.counts[e] = c;
            s += (float)c * p;
        }
    }
    s = block_sum<N / 64>(s, red);
    const float nk = n > 0 ? (float)n : 1.0f;
    if (threadIdx.x == 0) a.loss[0] = (float)a.experts * (s / nk / nk / (float)a.k);
}
__global__ __launch_bounds__(1024) void k_router_total(RouterArg a) {
    __shared__ float red[16], buf[2 * 1024];
    router_total<1024>(a, red, buf);
}

template <int L, int V, bool LIST>
__global__ __launch_bounds__(kRThreads) void k_router_fwd(RouterArg a) {
    constexpr int G = kRThreads / L;  // rows in flight in a workgroup
    constexpr int K = LIST ? kList : L * V < kMaxChosen ? L * V : kMaxChosen;
    __shared__ float red[kRThreads / 64];
    __shared__ int32_t cnt[L * V];
    __shared__ float pick[G][K];
    __shared__ int32_t pick_id[G][K];
    constexpr int kSums = (G > 1 ? G : 2) / 2 * L * V;
    __shared__ float sum_p[kSums > 2 * kRThreads ? kSums : 2 * kRThreads];  // for router_total at the end too
    const int tid = threadIdx.x, l = tid % L, g = tid / L;
    for (int e = tid; e < L * V; e += kRThreads) cnt[e] = 0;
    __syncthreads();
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    int32_t kept = 0;
    const int64_t stride = (int64_t)gridDim.x * G;
    // every wavefront walks whole rounds, so that its lanes reduce together
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const int64_t r = r0 + g;
        const bool in = r < a.rows;
        const bool keep = in && (!a.keep || a.keep[r] != 0);
        float v[V], m;
        load_row<L, V>(a.x + (in ? r : r0) * a.experts, a.experts, l, v);
        if constexpr (LIST) {
            double list[kList];
            row_list<L, V>(v, a.experts, l, list);
            wave_sync();
            if (l == 0) {
#pragma unroll
                for (int t = 0; t < kList; ++t) {
                    pick[g][t] = key_value(list_value(list[t]));
                    pick_id[g][t] = list_index(list[t]);
                }
            }
        } else {
            int key[V];
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = 4 * ((i / 4) * L + l) + (i & 3) < a.experts ? sort_key(v[i]) : kTaken;
            wave_sync();
            for (int t = 0; t < a.k; ++t) {
                int best = key[0];
#pragma unroll
                for (int i = 1; i < V; ++i) best = best > key[i] ? best : key[i];
                best = group_red<L>(best, [](int p, int q) { return p > q ? p : q; });
                int at = 0x7fffffff;  // the lowest index that holds it
#pragma unroll
                for (int i = V - 1; i >= 0; --i) at = key[i] == best ? 4 * (i / 4) * L + (i & 3) : at;
                at = at == 0x7fffffff ? at : at + 4 * l;
                at = group_red<L>(at, [](int p, int q) { return p < q ? p : q; });
                const int mine = at - 4 * l;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (mine == 4 * (i / 4) * L + (i & 3)) key[i] = kTaken;
                if (l == 0) {
                    pick[g][t] = key_value(best);
                    pick_id[g][t] = at;
                }
            }
        }
        const float inv = 1.0f / row_exp<L, V>(v, &m);
        if (keep) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += v[i] * inv;
            kept += l == 0;
        }
        wave_sync();
        float scale = inv;
        if (a.normalise) {
            float all = 0.0f;  // of the chosen's exponentials
            for (int t = l; t < a.k; t += L) all += exp_diff(pick[g][t], m);
            scale = 1.0f / group_sum<L>(all);
        }
        if (in)
            for (int t = l; t < a.k; t += L) {
                const int32_t id = pick_id[g][t];
                a.chosen[r * a.k + t] = keep ? id : -1;
                a.weights[r * a.k + t] = keep ? exp_diff(pick[g][t], m) * scale : 0.0f;
                if (keep) atomicAdd(&cnt[id], 1);
            }
    }
    // the workgroup's sums over its rows: halves of the groups added in turn
    kept = block_sum<kRThreads / 64>(kept, reinterpret_cast<int32_t*>(red));
#pragma unroll
    for (int half = G / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (g >= half && g < 2 * half) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum_p[((g - half) * V + i) * L + l] = acc[i];
        }
        __syncthreads();
        if (g < half) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += sum_p[(g * V + i) * L + l];
        }
    }
    __syncthreads();
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = 4 * ((i / 4) * L + l) + (i & 3);
            if (e < a.experts) {
                a.part_p[(int64_t)blockIdx.x * a.experts + e] = acc[i];
                a.part_c[(int64_t)blockIdx.x * a.experts + e] = cnt[e];
            }
        }
    }
    if (tid == 0) a.part_n[blockIdx.x] = kept;
    if (a.blocks == 1) {  // a short batch ends here
        __threadfence_block();
        __syncthreads();
        router_total<kRThreads>(a, red, sum_p);
    }
}

// An expert's partials, a workgroup each; the rows' count by the first.
__global__ __launch_bounds__(kRThreads) void k_router_join(RouterArg a) {
    __shared__ float red[kRThreads / 64];
    const int e = blockIdx.x;
    float p = 0.0f;
    int32_t c = 0, n = 0;
    for (int b = threadIdx.x; b < a.blocks; b += kRThreads) {
        p += a.part_p[(int64_t)b * a.experts + e];
        c += a.part_c[(int64_t)b * a.experts + e];
        n += a.part_n[b];
    }
    p = block_sum<kRThreads / 64>(p, red);
    c = block_sum<kRThreads / 64>(c, reinterpret_cast<int32_t*>(red));
    n = block_sum<kRThreads / 64>(n, reinterpret_cast<int32_t*>(red));
    if (threadIdx.x == 0) {
        a.counts[e] = c;
        const float nk = n > 0 ? (float)n : 1.0f;
        // the expert's term of the loss takes the place of nothing else: after the partials
        a.part_p[(int64_t)a.blocks * a.experts + e] = (float)c * p / nk / nk;
    }
}
__global__ __launch_bounds__(kRThreads) void k_router_loss(RouterArg a) {
    __shared__ float red[kRThreads / 64];
    float s = 0.0f;
    for (int e = threadIdx.x; e < a.experts; e += kRThreads) s += a.part_p[(int64_t)a.blocks * a.experts + e];
    s = block_sum<kRThreads / 64>(s, red);
    if (threadIdx.x == 0) a.loss[0] = (float)a.experts * (s / (float)a.k);
}

template <int L, int V>
__global__ __launch_bounds__(kRThreads) void k_router_bwd(RouterArg a) {
    constexpr int G = kRThreads / L;
    __shared__ __attribute__((aligned(16))) float buf[G][L * V], mark[G][L * V];
    __shared__ int32_t red[kRThreads / 64];
    const int tid = threadIdx.x, l = tid % L, g = tid / L;
    // kept rows: the counts add up to k of each
    float sf[V];
    {
        int32_t total = 0;
        if (a.ug)
            for (int e = tid; e < a.experts; e += kRThreads) total += a.cnt[e];
        total = block_sum<kRThreads / 64>(total, red);
        const float n = total > 0 ? (float)(total / a.k) : 1.0f;
        const float s = a.ug ? a.ug[0] * (float)a.experts / n : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = 4 * ((i / 4) * L + l) + (i & 3);
            sf[i] = a.ug && e < a.experts ? s * ((float)a.cnt[e] / (n * (float)a.k)) : 0.0f;
        }
    }
    const int64_t stride = (int64_t)gridDim.x * G;
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const int64_t r = r0 + g;
        const bool in = r < a.rows;
        const bool keep = in && (!a.keep || a.keep[r] != 0);
        const int64_t row = (in ? r : r0) * a.experts;
        float v[V], t[V];
        load_row<L, V>(a.x + row, a.experts, l, v);
        float top;
        const float inv = 1.0f / row_exp<L, V>(v, &top);
        // normalised weights w = e / sum of the chosen's e: their softmax's gradient first, from the row's
        // exponentials in LDS
        float w = 0.0f, mean = 0.0f;
        if (a.normalise && a.gw) {
            put_row<L, V>(buf[g], l, v);
            float all = 0.0f, own = 0.0f;
            if (keep)
                for (int c = l; c < a.k; c += L) {
                    const int32_t id = a.sel[r * a.k + c];
                    const float e = id >= 0 && id < a.experts ? buf[g][id] : 0.0f;
                    all += e;
                    own += e * a.gw[r * a.k + c];
                }
            w = 1.0f / group_sum<L>(all);
            mean = group_sum<L>(own) * w;
        }
        // what the chosen get: g, or w (g - mean) where that is the gradient already
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = 0.0f;
        if (a.gw) {
            put_row<L, V>(mark[g], l, t);
            if (keep)
                for (int c = l; c < a.k; c += L) {
                    const int32_t id = a.sel[r * a.k + c];
                    if (id < 0 || id >= a.experts) continue;
                    const float gr = a.gw[r * a.k + c];
                    mark[g][id] = a.normalise ? buf[g][id] * w * (gr - mean) : gr;
                }
            wave_sync();
            get_row<L, V>(mark[g], l, t);
            wave_sync();
        }
        float inner = 0.0f;
        if (a.normalise) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] *= inv;
                inner += v[i] * sf[i];
            }
            inner = group_sum<L>(inner);
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] += v[i] * (sf[i] - inner);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] *= inv;
                t[i] += sf[i];
                inner += v[i] * t[i];
            }
            inner = group_sum<L>(inner);
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = v[i] * (t[i] - inner);
        }
        if (!in || (!keep && a.accumulate)) continue;  // a padding row: as it was, or zero
        float* o = a.grad + row;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const int c = 4 * (i * L + l);
#pragma unroll
            for (int j = 0; j < 4; ++j) t[4 * i + j] = keep ? t[4 * i + j] : 0.0f;
            if (c + 3 < a.experts) {
                vf4 q = {t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]};
                if (a.accumulate) {
                    const vf4 old = ld_ntu(o + c);
                    q = {old.x + q.x, old.y + q.y, old.z + q.z, old.w + q.w};
                }
                st_ntu(o + c, q);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < a.experts) o[c + j] = a.accumulate ? o[c + j] + t[4 * i + j] : t[4 * i + j];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
// Lanes and elements of a lane by the experts, 16 elements a lane at most: 32 would make the lanes' part of the
// selection shorter, but take 152 and 174 registers a thread (over [131072, 256] 65 and 78 us forward and
// backward, against 60 and 56 with 16).
#define MH_ROUTER(CALL)                      \
    do {                                     \
        if (a.experts <= 8) CALL(2, 4);      \
        else if (a.experts <= 16) CALL(4, 4);   \
        else if (a.experts <= 32) CALL(4, 8);   \
        else if (a.experts <= 64) CALL(8, 8);   \
        else if (a.experts <= 128) CALL(8, 16); \
        else if (a.experts <= 256) CALL(16, 16); \
        else if (a.experts <= 512) CALL(32, 16); \
        else CALL(64, 16);                   \
    } while (0)

int router_lanes(int experts) {
    return experts <= 8 ? 2 : experts <= 32 ? 4 : experts <= 128 ? 8 : experts <= 256 ? 16 : experts <= 512 ? 32 : 64;
}

int router_check(const char* what, int64_t rows, int64_t experts, int64_t k) {
    if (rows < 0 || experts < 1 || experts > kMaxExperts || k < 1 || k > kMaxChosen || k > experts)
        return fail(MH_ERR_INVALID, "%s: needs rows >= 0, 1 <= experts <= %d, 1 <= k <= min(%d, experts) (%lld, %lld, %lld)",
                    what, kMaxExperts, kMaxChosen, (long long)rows, (long long)experts, (long long)k);
    if (rows > 0x7fffffff / k) return fail(MH_ERR_OVERFLOW, "%s: more than 2^31 - 1 choices", what);
    return MH_OK;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_router_fwd(float* weights, int32_t* chosen, int32_t* counts, float* loss, const float* x, const int32_t* keep,
                  int64_t rows, int64_t experts, int64_t k, int normalise) {
    MH_TRACE("mh_router_fwd");
    MH_TRY(router_check("mh_router_fwd", rows, experts, k));
    if (!counts || !loss || (rows > 0 && (!weights || !chosen || !x))) return fail(MH_ERR_NULL, "mh_router_fwd: null tensor");
    MH_TRY(require_init());
    if (rows == 0) {  // zero bits are the whole number 0 too
        MH_TRY(mh_zero(reinterpret_cast<float*>(counts), experts));
        return mh_fill(loss, 0.0f, 1);
    }
    RouterArg a = {};
    a.x = x;
    a.keep = keep;
    a.rows = rows;
    a.experts = (int32_t)experts;
    a.k = (int32_t)k;
    a.normalise = normalise != 0;
    a.weights = weights;
    a.chosen = chosen;
    a.counts = counts;
    a.loss = loss;
    const int64_t group = kRThreads / router_lanes(a.experts);
    int64_t blocks = (rows + group - 1) / group;
    if (blocks > kRBlocks) blocks = kRBlocks;
    if (blocks <= 2) blocks = 1;  // one launch rather than three
    a.blocks = (int32_t)blocks;
    const size_t n = (size_t)(blocks + 1) * experts;
    float* base = nullptr;
    MH_TRY(scratch((2 * n + blocks) * 4, reinterpret_cast<void**>(&base)));
    a.part_p = base;
    a.part_c = reinterpret_cast<int32_t*>(base + n);
    a.part_n = reinterpret_cast<int32_t*>(base + 2 * n);
    hipStream_t st = ctx().stream;
#define MH_CALL(L, V)                                                                                               \
    do {                                                                                                           \
        if (a.k <= kList) hipLaunchKernelGGL((k_router_fwd<L, V, true>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a); \
        else hipLaunchKernelGGL((k_router_fwd<L, V, false>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a);   \
    } while (0)
    MH_ROUTER(MH_CALL);
#undef MH_CALL
    // few partials: one workgroup adds them up in the time of a launch; else a workgroup an expert, and the loss
    if (blocks > 1 && blocks * experts <= 16384) {
        hipLaunchKernelGGL(k_router_total, dim3(1), dim3(1024), 0, st, a);
    } else if (blocks > 1) {
        hipLaunchKernelGGL(k_router_join, dim3((unsigned)experts), dim3(kRThreads), 0, st, a);
        hipLaunchKernelGGL(k_router_loss, dim3(1), dim3(kRThreads), 0, st, a);
    }
    return finish("mh_router_fwd");
}

int mh_router_bwd(float* grad_x, const float* x, const int32_t* keep, const int32_t* chosen, const int32_t* counts,
                  const float* grad_weights, const float* ug, int64_t rows, int64_t experts, int64_t k, int normalise,
                  int accumulate) {
    MH_TRACE("mh_router_bwd");
    MH_TRY(router_check("mh_router_bwd", rows, experts, k));
    if (rows == 0) return MH_OK;
    if (!grad_x || !x || !counts || (grad_weights && !chosen)) return fail(MH_ERR_NULL, "mh_router_bwd: null tensor");
    MH_TRY(require_init());
    RouterArg a = {};
    a.x = x;
    a.keep = keep;
    a.rows = rows;
    a.experts = (int32_t)experts;
    a.k = (int32_t)k;
    a.normalise = normalise != 0;
    a.accumulate = accumulate != 0;
    a.grad = grad_x;
    a.gw = grad_weights;
    a.ug = ug;
    a.sel = chosen;
    a.cnt = counts;
    const int64_t group = kRThreads / router_lanes(a.experts);
    int64_t blocks = (rows + group - 1) / group;
    if (blocks > 2048) blocks = 2048;
    hipStream_t st = ctx().stream;
#define MH_CALL(L, V) hipLaunchKernelGGL((k_router_bwd<L, V>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a)
    MH_ROUTER(MH_CALL);
#undef MH_CALL
    return finish("mh_router_bwd");
}

}  // extern "C"
