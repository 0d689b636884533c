// mh_optim.hip -- Adam.step (mantle/nn/optim.mojo:94-140) on device-resident parameters.
//
// Per element, in the reference's expression order (v_step, optim.mojo:101-132; built with
// -ffp-contract=off, so every product and sum rounds on its own):
//   m = beta1 * m + (1 - beta1) * g;           store m;   mh = m / (1 - beta1 ** iter)
//   v = beta2 * v + ((1 - beta2) * g) * g;     store v;   vh = v / (1 - beta2 ** iter)
//   p = p - lr * (mh / (sqrt(vh) + eps))
// The scalars 1 - beta and 1 - beta ** iter are Scalar[f32] arithmetic, beta ** iter being
// Mojo's SIMD ** Int (square-and-multiply); they are computed once on the host in f32.
// 28 bytes per element: p, g, m, v read; p, m, v written.
//
// mh_adam_step updates one tensor; mh_adam_step_multi updates every parameter of a model
// with one launch per 80 tensors (the reference parallelises over parameters,
// optim.mojo:140): threads walk the concatenated element quads of the launch's tensors and
// find their tensor by a wave-uniform binary search in a table passed by value, so a model of
// many small tensors costs a launch per 80 tensors, not one per tensor.
//
// mh_grad_norm, mh_clip_grad_norm, mh_adam_clip_step_multi: the norm of all gradients together,
// N = sqrt(sum g^2), and c = min(1, max_norm / N) times them, in place or on their way into Adam
// (which saves the 8 bytes an element of writing them and reading them again). Bound by memory: 4
// bytes an element for the norm, 8 more to scale them, 28 for Adam. The squares are added in 64
// bits, which any fp32 gradient's fit: per thread, per workgroup, and over the workgroups by one
// workgroup, always in the same order.
#include <algorithm>
#include <cmath>
#include <new>

#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {

constexpr int kOThreads = 64;  // one-wavefront workgroups stream fastest on gfx950

struct AdamScal {
    float lr, b1, b2, eps, c1, c2, bc1, bc2;
};

// f32 x ** n by square-and-multiply (Mojo's SIMD ** Int), n >= 0.
static float host_powi(float x, int64_t n) {
    float a = x, res = 1.0f;
    for (uint64_t b = (uint64_t)n; b > 0; b >>= 1) {
        if (b & 1u) res = res * a;
        a = a * a;
    }
    return res;
}

static AdamScal adam_scalars(float lr, float b1, float b2, float eps, int64_t iter) {
    AdamScal s;
    s.lr = lr;
    s.b1 = b1;
    s.b2 = b2;
    s.eps = eps;
    s.c1 = 1.0f - b1;
    s.c2 = 1.0f - b2;
    s.bc1 = 1.0f - host_powi(b1, iter);
    s.bc2 = 1.0f - host_powi(b2, iter);
    return s;
}

__device__ __forceinline__ void adam1(float& p, float g, float& m, float& v, const AdamScal& s) {
    float mj = s.b1 * m + s.c1 * g;
    m = mj;
    mj = mj / s.bc1;
    float vj = s.b2 * v + s.c2 * g * g;
    v = vj;
    vj = vj / s.bc2;
    p = p - s.lr * (mj / (__builtin_sqrtf(vj) + s.eps));
}

// Elements [e0, e0 + cnt) of one tensor, cnt <= 4; a full quad at a 16-byte aligned address
// moves as float4. CLIP: the gradients count c times.
template <bool CLIP>
__device__ __forceinline__ void adam_unit(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                          float* __restrict__ v, int64_t e0, int cnt, bool vec, const AdamScal& s, float c) {
    if (cnt == 4 && vec) {
        float4 pp = ld_nt4(p + e0, 0);
        float4 gg = ld_nt4(g + e0, 0);
        if (CLIP) gg = make_float4(gg.x * c, gg.y * c, gg.z * c, gg.w * c);
        float4 mm = ld_nt4(m + e0, 0);
        float4 vv = ld_nt4(v + e0, 0);
        adam1(pp.x, gg.x, mm.x, vv.x, s);
        adam1(pp.y, gg.y, mm.y, vv.y, s);
        adam1(pp.z, gg.z, mm.z, vv.z, s);
        adam1(pp.w, gg.w, mm.w, vv.w, s);
        st_nt4(p + e0, 0, pp);
        st_nt4(m + e0, 0, mm);
        st_nt4(v + e0, 0, vv);
    } else {
        for (int j = 0; j < cnt; ++j) {
            float pp = p[e0 + j], mm = m[e0 + j], vv = v[e0 + j];
            adam1(pp, CLIP ? g[e0 + j] * c : g[e0 + j], mm, vv, s);
            p[e0 + j] = pp;
            m[e0 + j] = mm;
            v[e0 + j] = vv;
        }
    }
}

// Units of a tensor. When the four pointers share one misalignment (the same offset into four
// aligned buffers, as a sliced arena gives), unit 0 takes the `head` = 0..3 elements before the
// first 16-byte boundary and every later unit is an aligned quad: unit k covers elements
// [max(0, 4k - sh), min(n, 4k + 4 - sh)), sh = (4 - head) & 3. Otherwise sh = 0 and units
// are scalar.
struct UnitMap {
    int sh;      // 0..3
    int vec;     // quads after the head are 16-byte aligned in all four tensors
};

__host__ __device__ __forceinline__ int64_t adam_units(int64_t n, int sh) { return (n + sh + 3) >> 2; }

template <bool CLIP>
__device__ __forceinline__ void adam_unit_k(float* __restrict__ p, const float* __restrict__ g,
                                            float* __restrict__ m, float* __restrict__ v, int64_t n, int64_t k,
                                            UnitMap um, const AdamScal& s, float c) {
    const int64_t lo = 4 * k - um.sh;
    const int64_t e0 = lo < 0 ? 0 : lo;
    const int64_t e1 = (lo + 4) < n ? (lo + 4) : n;
    adam_unit<CLIP>(p, g, m, v, e0, (int)(e1 - e0), um.vec != 0, s, c);
}

static inline UnitMap unit_map(const void* p, const void* g, const void* m, const void* v) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p) & 15;
    UnitMap um{0, 0};
    if ((a & 3) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == a && (reinterpret_cast<uintptr_t>(m) & 15) == a &&
        (reinterpret_cast<uintptr_t>(v) & 15) == a) {
        um.vec = 1;
        um.sh = (int)(a >> 2);  // head = (4 - a/4) & 3 elements, so sh = a/4
    }
    return um;
}

__global__ void __launch_bounds__(kOThreads)
    k_adam(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m, float* __restrict__ v,
           int64_t n, UnitMap um, AdamScal s) {
    const int64_t units = adam_units(n, um.sh);
    const int64_t stride = (int64_t)gridDim.x * kOThreads;
    for (int64_t u = (int64_t)blockIdx.x * kOThreads + threadIdx.x; u < units; u += stride)
        adam_unit_k<false>(p, g, m, v, n, u, um, s, 1.0f);
}

// The common case of k_adam (all four tensors 16-byte aligned, sh == 0): thread q takes quad q,
// with no unit arithmetic; the last n % 4 elements go to the thread after the last quad.
template <bool CLIP>
__global__ void __launch_bounds__(kOThreads)
    k_adam_al(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m, float* __restrict__ v,
              int64_t n, AdamScal s, const float* __restrict__ coef) {
    const float c = CLIP ? coef[0] : 1.0f;
    const int64_t q = (int64_t)blockIdx.x * kOThreads + threadIdx.x;
    const int64_t nq = n >> 2;
    if (q < nq) {
        adam_unit<CLIP>(p, g, m, v, 4 * q, 4, true, s, c);
    } else if (q == nq && (n & 3) != 0) {
        adam_unit<CLIP>(p, g, m, v, 4 * q, (int)(n & 3), false, s, c);
    }
}

// 48 bytes: the first unit of the tensor in the launch's concatenated unit space is a multiple
// of 64 (each tensor starts on a wave), so its low six bits carry the unit map: bits 0-1 sh,
// bit 2 vec.
struct AdamTensor {
    float* p;
    const float* g;
    float* m;
    float* v;
    int64_t n;
    int64_t u0m;
    __host__ __device__ int64_t unit0() const { return u0m & ~int64_t(63); }
    __host__ __device__ UnitMap um() const { return UnitMap{(int)(u0m & 3), (int)((u0m >> 2) & 1)}; }
};
static_assert(sizeof(AdamTensor) == 48, "table entry size");

// Up to kAdamPerLaunch tensors travel by value in the kernel arguments (3.8 KB of the 4 KB
// they may take), so a launch needs no device-side table. (With 56-byte entries and 64 per
// launch, 400 tensors of 1..2^18 elements took seven launches instead of five.)
constexpr int kAdamPerLaunch = 80;
struct AdamTable {
    AdamTensor t[kAdamPerLaunch];
    int32_t nt;
};

// Each tensor starts on a wave boundary of the concatenated quad space (unit0 a multiple of
// 64), so a wave belongs to one tensor: the search runs once per wave on wave-uniform values
// (scalar loads from the kernel arguments), and lanes past the tensor's end idle.
template <bool CLIP>
__global__ void __launch_bounds__(kOThreads) k_adam_multi(AdamTable tab, int64_t units, AdamScal s, const float* coef) {
    const float c = CLIP ? coef[0] : 1.0f;
    const int64_t stride = (int64_t)gridDim.x * kOThreads;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = (int)(threadIdx.x & 63);
    for (int64_t uw = (int64_t)blockIdx.x * kOThreads + wid * 64; uw < units; uw += stride) {
        int lo = 0, hi = tab.nt - 1;  // the last tensor whose unit0 <= uw
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (tab.t[mid].unit0() <= uw) lo = mid;
            else hi = mid - 1;
        }
        const AdamTensor& t = tab.t[lo];
        const UnitMap um = t.um();
        const int64_t k = uw - t.unit0() + lane;
        if (k < adam_units(t.n, um.sh)) adam_unit_k<CLIP>(t.p, t.g, t.m, t.v, t.n, k, um, s, c);
    }
}

static inline unsigned grid_units(int64_t units) { return (unsigned)grid_blocks(units, kOThreads); }

// k_adam_al gives every quad, and the tail after the last one, a thread of its own with no
// loop, so it takes the aligned tensors whose quads fit one dispatch; every other tensor goes
// through k_adam, which loops over its grid.
static LaunchShape adam_shape(int64_t n, UnitMap um) {
    const int64_t al_items = (n >> 2) + 1;
    if (um.vec && um.sh == 0 && al_items <= max_grid_blocks(kOThreads) * kOThreads)
        return LaunchShape{0, kOThreads, grid_blocks(al_items, kOThreads), 1};
    return LaunchShape{1, kOThreads, grid_blocks(adam_units(n, um.sh), kOThreads), 1};
}

LaunchShape adam_launch(int64_t n, bool aligned) { return adam_shape(n, UnitMap{0, aligned ? 1 : 0}); }

static int check_hyper(const char* what, float lr, float b1, float b2, float eps, int64_t iter) {
    if (iter < 1) return fail(MH_ERR_INVALID, "%s: iter %lld (Adam.step counts from 1)", what, (long long)iter);
    if (!std::isfinite(lr) || !std::isfinite(b1) || !std::isfinite(b2) || !std::isfinite(eps))
        return fail(MH_ERR_INVALID, "%s: non-finite hyper-parameter", what);
    return MH_OK;
}

static int check_adam(const char* what, int64_t ntensors, float* const* params, const float* const* grads, float* const* m,
                      float* const* v, const int64_t* sizes) {
    if (ntensors < 0) return fail(MH_ERR_INVALID, "%s: negative tensor count", what);
    if (ntensors > 0 && (!params || !grads || !m || !v || !sizes)) return fail(MH_ERR_NULL, "%s: null table", what);
    for (int64_t i = 0; i < ntensors; ++i) {  // validate everything before any launch
        if (sizes[i] < 0) return fail(MH_ERR_INVALID, "%s: negative size of tensor %lld", what, (long long)i);
        if (sizes[i] > 0 && (!params[i] || !grads[i] || !m[i] || !v[i]))
            return fail(MH_ERR_NULL, "%s: null pointer in tensor %lld", what, (long long)i);
    }
    return MH_OK;
}

template <bool CLIP>
static void adam_multi(int64_t ntensors, float* const* params, const float* const* grads, float* const* m, float* const* v,
                       const int64_t* sizes, const AdamScal& s, const float* coef) {
    AdamTable tab;
    int64_t i = 0;
    while (i < ntensors) {
        tab.nt = 0;
        int64_t units = 0;
        for (; i < ntensors && tab.nt < kAdamPerLaunch; ++i) {
            if (sizes[i] == 0) continue;
            AdamTensor& t = tab.t[tab.nt++];
            t.p = params[i];
            t.g = grads[i];
            t.m = m[i];
            t.v = v[i];
            t.n = sizes[i];
            const UnitMap um = unit_map(t.p, t.g, t.m, t.v);
            t.u0m = units | um.sh | (um.vec << 2);  // units: a multiple of 64
            units += (adam_units(t.n, um.sh) + 63) & ~int64_t(63);  // next tensor starts on a wave
        }
        if (tab.nt > 0)
            hipLaunchKernelGGL(k_adam_multi<CLIP>, dim3(grid_units(units)), dim3(kOThreads), 0, ctx().stream, tab, units, s,
                               coef);
    }
}

// ---------------------------------------------------------------------------------------
// the norm of many gradients
// ---------------------------------------------------------------------------------------
constexpr int kGradThreads = 256;
constexpr int kGradQuads = 4;                                          // quads a thread and chunk
constexpr int64_t kGradChunk = (int64_t)kGradThreads * kGradQuads;     // quads of a chunk
constexpr int64_t kGradBlocks = 2048;                                  // workgroups of a launch at most
// Workgroups whose last to arrive adds up: a tensor of 262144 5.9 us instead of 8.6 with a launch for it, 1048576 7.4; 512 of them
// wait for one counter, 10.3.
constexpr int64_t kGradOne = 256;
constexpr int kGradPerLaunch = 160;                                    // 3.8 KB of the 4 KB that arguments may take

// A tensor and the first chunk of it in the launch's chunks. Quad k of a tensor whose address is sh floats past a
// 16-byte boundary holds the elements [4k - sh, 4k - sh + 4) that it has, so whole quads are aligned.
struct GradTensor {
    float* g;
    int64_t n, chunk0;
};
struct GradTable {
    GradTensor t[kGradPerLaunch];
    int32_t nt;
};

__host__ __device__ __forceinline__ int grad_shift(const float* g) { return (int)((reinterpret_cast<uintptr_t>(g) >> 2) & 3); }

// The workgroups of a launch over chunks that each takes as many of, the last fewer.
static int64_t grad_blocks(int64_t chunks) {
    const int64_t each = (chunks + kGradBlocks - 1) / kGradBlocks;
    return chunks ? (chunks + each - 1) / each : 0;
}

// The tensors from *i on that a launch takes, and its chunks.
static int64_t grad_table(int64_t ntensors, const float* const* grads, const int64_t* sizes, int64_t* i, GradTable* tab) {
    int64_t chunks = 0;
    for (tab->nt = 0; *i < ntensors && tab->nt < kGradPerLaunch; ++*i) {
        if (sizes[*i] == 0) continue;
        GradTensor& t = tab->t[tab->nt++];
        t.g = const_cast<float*>(grads[*i]);
        t.n = sizes[*i];
        t.chunk0 = chunks;
        chunks += ((t.n + grad_shift(t.g) + 3) / 4 + kGradChunk - 1) / kGradChunk;
    }
    return chunks;
}

// The last tensor whose chunk0 <= chunk: each lane looks at three. (A binary search's eight reads wait for each other.)
__device__ __forceinline__ int grad_find(const GradTable& tab, int64_t chunk) {
    const int lane = threadIdx.x & 63;
    int at = -1;
#pragma unroll
    for (int i = 0; i < kGradPerLaunch; i += 64) {
        const bool is = i + lane < tab.nt && tab.t[i + lane < kGradPerLaunch ? i + lane : 0].chunk0 <= chunk;
        at += __builtin_popcountll(__ballot(is));
    }
    return __builtin_amdgcn_readfirstlane(at);
}

__device__ __forceinline__ double square_add(double s, float v) { return __builtin_fma((double)v, (double)v, s); }

// The squares of the chunks from c on, `step` apart and below `end`, by 256 threads; s gets each thread's.
__device__ __forceinline__ void chunk_squares(const GradTable& tab, int64_t c, int64_t end, int64_t step, int tid, double* s) {
    const float* g = nullptr;
    int64_t n = 0, chunk0 = 0, next = -1;  // of the tensor at hand, and the first chunk past it
    int sh = 0;
    for (; c < end; c += step) {
        if (c >= next) {
            const int at = grad_find(tab, c);
            const GradTensor& t = tab.t[at];
            g = t.g;
            n = t.n;
            chunk0 = t.chunk0;
            sh = grad_shift(g);
            next = at + 1 < tab.nt ? tab.t[at + 1].chunk0 : end;
        }
        const int64_t k0 = (c - chunk0) * kGradChunk;
        if (4 * k0 >= sh && 4 * (k0 + kGradChunk) - sh <= n) {  // whole quads
            vf4 v[kGradQuads];
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) v[i] = *reinterpret_cast<const vf4*>(g + 4 * (k0 + i * kGradThreads + tid) - sh);
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) {
                s[0] = square_add(s[0], v[i].x);
                s[1] = square_add(s[1], v[i].y);
                s[2] = square_add(s[2], v[i].z);
                s[3] = square_add(s[3], v[i].w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) {
                const int64_t e = 4 * (k0 + i * kGradThreads + tid) - sh;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e + j >= 0 && e + j < n) s[j] = square_add(s[j], g[e + j]);
            }
        }
    }
}

__device__ __forceinline__ void put_norm(double squares, float max_norm, float* norm, float* coef) {
    const double n = __builtin_sqrt(squares);
    if (norm) norm[0] = (float)n;
    // an infinity or a NaN among the gradients scales nothing
    coef[0] = n > (double)max_norm && n <= 1.7976931348623157e308 ? (float)((double)max_norm / n) : 1.0f;
}

// A workgroup takes neighbouring chunks, nearly always of one tensor. ONE: the last of them to arrive adds up, in their order.
template <bool ONE>
__global__ __launch_bounds__(kGradThreads) void k_grad_norm(GradTable tab, int64_t chunks, int64_t each, double* part, uint32_t* arrived,
                                                            float max_norm, float* norm, float* coef) {
    __shared__ double red[kGradThreads / 64];
    __shared__ int last;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    const int64_t c = blockIdx.x * each;
    chunk_squares(tab, c, c + each < chunks ? c + each : chunks, 1, threadIdx.x, s);
    const double sum = block_sum<kGradThreads / 64>((s[0] + s[1]) + (s[2] + s[3]), red);
    if constexpr (ONE) {
        if (threadIdx.x == 0) {  // the store is waited for, rather than the L2 written back
            __hip_atomic_store(&part[blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_s_waitcnt(0);
            last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        double all = 0.0;
        for (unsigned i = threadIdx.x; i < gridDim.x; i += kGradThreads)
            all += __hip_atomic_load(&part[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        all = block_sum<kGradThreads / 64>(all, red);
        if (threadIdx.x == 0) {
            put_norm(all, max_norm, norm, coef);
            __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    } else {
        if (threadIdx.x == 0) part[blockIdx.x] = sum;
    }
}

// The norm from the workgroups' sums, and what the gradients are scaled by.
__global__ __launch_bounds__(1024) void k_grad_total(const double* part, int64_t parts, float max_norm, float* norm, float* coef) {
    __shared__ double red[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += 1024) s += part[i];
    s = block_sum<16>(s, red);
    if (threadIdx.x == 0) put_norm(s, max_norm, norm, coef);
}

__global__ __launch_bounds__(kGradThreads) void k_clip_scale(GradTable tab, int64_t chunks, const float* coef) {
    const float m = coef[0];
    if (m == 1.0f) return;
    for (int64_t c = chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {  // from the end, which the caches hold
        const GradTensor& t = tab.t[grad_find(tab, c)];
        const int sh = grad_shift(t.g);
        const int64_t k0 = (c - t.chunk0) * kGradChunk;
        if (4 * k0 >= sh && 4 * (k0 + kGradChunk) - sh <= t.n) {
            vf4 v[kGradQuads];
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) v[i] = ld_ntv(t.g + 4 * (k0 + i * kGradThreads + threadIdx.x) - sh, 0);
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) st_ntv(t.g + 4 * (k0 + i * kGradThreads + threadIdx.x) - sh, 0, v[i] * m);
        } else {
#pragma unroll
            for (int i = 0; i < kGradQuads; ++i) {
                const int64_t e = 4 * (k0 + i * kGradThreads + threadIdx.x) - sh;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e + j >= 0 && e + j < t.n) t.g[e + j] *= m;
            }
        }
    }
}

static int check_grads(const char* what, int64_t ntensors, const float* const* grads, const int64_t* sizes, float max_norm) {
    if (ntensors < 0) return fail(MH_ERR_INVALID, "%s: negative tensor count", what);
    if (!(max_norm >= 0.0f)) return fail(MH_ERR_INVALID, "%s: a largest norm of %g", what, (double)max_norm);
    if (ntensors > 0 && (!grads || !sizes)) return fail(MH_ERR_NULL, "%s: null table", what);
    int64_t n = 0;
    for (int64_t i = 0; i < ntensors; ++i) {
        if (sizes[i] < 0) return fail(MH_ERR_INVALID, "%s: negative size of tensor %lld", what, (long long)i);
        if (sizes[i] > 0 && !grads[i]) return fail(MH_ERR_NULL, "%s: null pointer in tensor %lld", what, (long long)i);
        if (sizes[i] > 0 && (reinterpret_cast<uintptr_t>(grads[i]) & 3))
            return fail(MH_ERR_INVALID, "%s: tensor %lld is not aligned to 4 bytes", what, (long long)i);
        if (sizes[i] > ((int64_t)1 << 46) - n) return fail(MH_ERR_OVERFLOW, "%s: more than 2^46 elements", what);
        n += sizes[i];
    }
    return MH_OK;
}

// Refuses tensors that share elements, which would be scaled twice. Tensors in the order of their addresses, as an
// arena has them, take one look each.
static int check_apart(const char* what, int64_t ntensors, const float* const* grads, const int64_t* sizes) {
    const float* end = nullptr;
    bool rising = true;
    for (int64_t i = 0; i < ntensors && rising; ++i) {
        if (sizes[i] == 0) continue;
        rising = grads[i] >= end;
        end = grads[i] + sizes[i];
    }
    if (rising) return MH_OK;
    int64_t* order = new (std::nothrow) int64_t[ntensors];
    if (!order) return fail(MH_ERR_INVALID, "%s: no host memory for %lld tensors", what, (long long)ntensors);
    int64_t n = 0;
    for (int64_t i = 0; i < ntensors; ++i)
        if (sizes[i] > 0) order[n++] = i;
    std::sort(order, order + n, [&](int64_t p, int64_t q) { return grads[p] < grads[q]; });
    int64_t twice = -1;
    for (int64_t i = 1; i < n && twice < 0; ++i)
        if (grads[order[i - 1]] + sizes[order[i - 1]] > grads[order[i]]) twice = order[i];
    delete[] order;
    return twice < 0 ? MH_OK : fail(MH_ERR_INVALID, "%s: tensor %lld shares elements with another", what, (long long)twice);
}

// Queues the norm of all gradients; *coef is where what they are scaled by will lie.
static int norm_of(int64_t ntensors, const float* const* grads, const int64_t* sizes, float max_norm, float* norm, float** coef) {
    GradTable tab;
    int64_t parts = 0, first = 0, first_chunks = 0;
    for (int64_t i = 0; i < ntensors;) {
        const int64_t chunks = grad_table(ntensors, grads, sizes, &i, &tab);
        if (first == 0) first = i == ntensors ? grad_blocks(chunks) : kGradOne + 1;  // all of them, if one launch takes them
        first_chunks = first_chunks ? first_chunks : chunks;
        parts += grad_blocks(chunks);
    }
    double* part = nullptr;
    MH_TRY(scratch(8 * (size_t)(parts + 1), reinterpret_cast<void**>(&part)));
    *coef = reinterpret_cast<float*>(part + parts);
    if (first > 0 && first <= kGradOne) {
        uint32_t* arrived = nullptr;
        MH_TRY(tickets(1, &arrived));
        hipLaunchKernelGGL(k_grad_norm<true>, dim3((unsigned)first), dim3(kGradThreads), 0, ctx().stream, tab, first_chunks,
                           (first_chunks + kGradBlocks - 1) / kGradBlocks, part, arrived, max_norm, norm, *coef);
        return MH_OK;
    }
    double* at = part;
    for (int64_t i = 0; i < ntensors;) {
        const int64_t chunks = grad_table(ntensors, grads, sizes, &i, &tab);
        if (chunks == 0) continue;
        const int64_t blocks = grad_blocks(chunks);
        hipLaunchKernelGGL(k_grad_norm<false>, dim3((unsigned)blocks), dim3(kGradThreads), 0, ctx().stream, tab, chunks,
                           (chunks + kGradBlocks - 1) / kGradBlocks, at, nullptr, 0.0f, nullptr, nullptr);
        at += blocks;
    }
    hipLaunchKernelGGL(k_grad_total, dim3(1), dim3(1024), 0, ctx().stream, part, parts, max_norm, norm, *coef);
    return MH_OK;
}

}  // namespace mh

using namespace mh;

extern "C" {

int mh_adam_step(float* param, const float* grad, float* m, float* v, int64_t n, float lr, float beta1,
                 float beta2, float eps, int64_t iter) {
    MH_TRACE("mh_adam_step");
    MH_TRY(check_hyper("mh_adam_step", lr, beta1, beta2, eps, iter));
    if (n < 0) return fail(MH_ERR_INVALID, "mh_adam_step: negative count");
    if (n == 0) return MH_OK;
    if (!param || !grad || !m || !v) return fail(MH_ERR_NULL, "mh_adam_step: null tensor");
    MH_TRY(require_init());
    const AdamScal s = adam_scalars(lr, beta1, beta2, eps, iter);
    const UnitMap um = unit_map(param, grad, m, v);
    const LaunchShape ls = adam_shape(n, um);
    if (ls.kernel == 0)
        hipLaunchKernelGGL(k_adam_al<false>, dim3((unsigned)ls.blocks), dim3(ls.threads), 0, ctx().stream, param, grad, m,
                           v, n, s, (const float*)nullptr);
    else
        hipLaunchKernelGGL(k_adam, dim3((unsigned)ls.blocks), dim3(ls.threads), 0, ctx().stream, param, grad, m, v, n,
                           um, s);
    return finish("mh_adam_step");
}

int mh_adam_step_multi(int64_t ntensors, float* const* params, const float* const* grads, float* const* m,
                       float* const* v, const int64_t* sizes, float lr, float beta1, float beta2, float eps,
                       int64_t iter) {
    MH_TRACE("mh_adam_step_multi");
    MH_TRY(check_hyper("mh_adam_step_multi", lr, beta1, beta2, eps, iter));
    MH_TRY(check_adam("mh_adam_step_multi", ntensors, params, grads, m, v, sizes));
    if (ntensors == 0) return MH_OK;
    MH_TRY(require_init());
    adam_multi<false>(ntensors, params, grads, m, v, sizes, adam_scalars(lr, beta1, beta2, eps, iter), nullptr);
    return finish("mh_adam_step_multi");
}

int mh_grad_norm(int64_t ntensors, const float* const* grads, const int64_t* sizes, float* norm) {
    MH_TRACE("mh_grad_norm");
    MH_TRY(check_grads("mh_grad_norm", ntensors, grads, sizes, 0.0f));
    if (!norm) return fail(MH_ERR_NULL, "mh_grad_norm: null norm");
    MH_TRY(require_init());
    float* coef = nullptr;
    MH_TRY(norm_of(ntensors, grads, sizes, 0.0f, norm, &coef));
    return finish("mh_grad_norm");
}

int mh_clip_grad_norm(int64_t ntensors, float* const* grads, const int64_t* sizes, float max_norm, float* norm) {
    MH_TRACE("mh_clip_grad_norm");
    MH_TRY(check_grads("mh_clip_grad_norm", ntensors, grads, sizes, max_norm));
    MH_TRY(check_apart("mh_clip_grad_norm", ntensors, grads, sizes));
    MH_TRY(require_init());
    float* coef = nullptr;
    MH_TRY(norm_of(ntensors, grads, sizes, max_norm, norm, &coef));
    GradTable tab;
    for (int64_t i = 0; i < ntensors;) {
        const int64_t chunks = grad_table(ntensors, grads, sizes, &i, &tab);
        if (chunks > 0)
            hipLaunchKernelGGL(k_clip_scale, dim3((unsigned)(chunks < kGradBlocks ? chunks : kGradBlocks)), dim3(kGradThreads), 0,
                               ctx().stream, tab, chunks, coef);
    }
    return finish("mh_clip_grad_norm");
}

int mh_adam_clip_step_multi(int64_t ntensors, float* const* params, const float* const* grads, float* const* m,
                            float* const* v, const int64_t* sizes, float lr, float beta1, float beta2, float eps,
                            int64_t iter, float max_norm, float* norm) {
    MH_TRACE("mh_adam_clip_step_multi");
    MH_TRY(check_hyper("mh_adam_clip_step_multi", lr, beta1, beta2, eps, iter));
    MH_TRY(check_adam("mh_adam_clip_step_multi", ntensors, params, grads, m, v, sizes));
    MH_TRY(check_grads("mh_adam_clip_step_multi", ntensors, grads, sizes, max_norm));
    MH_TRY(require_init());
    const AdamScal s = adam_scalars(lr, beta1, beta2, eps, iter);
    float* coef = nullptr;
    MH_TRY(norm_of(ntensors, grads, sizes, max_norm, norm, &coef));
    if (ntensors == 1 && sizes[0] > 0) {
        const UnitMap um = unit_map(params[0], grads[0], m[0], v[0]);
        const LaunchShape ls = adam_shape(sizes[0], um);
        if (ls.kernel == 0) {
            hipLaunchKernelGGL(k_adam_al<true>, dim3((unsigned)ls.blocks), dim3(ls.threads), 0, ctx().stream, params[0], grads[0],
                               m[0], v[0], sizes[0], s, (const float*)coef);
            return finish("mh_adam_clip_step_multi");
        }
    }
    adam_multi<true>(ntensors, params, grads, m, v, sizes, s, coef);
    return finish("mh_adam_clip_step_multi");
}

}  // extern "C"
