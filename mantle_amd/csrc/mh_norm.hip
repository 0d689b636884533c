// mh_norm.hip -- root-mean-square norm over rows, with the residual's addition, forward and backward.
//
//   h = x + residual;  s = 1 / sqrt(mean h^2 + eps);  u = h s;  out = u w
//   grad_x = grad_sum + s (w g - u mean(w g u)),  g the gradient of out;  grad_w = sum over rows of g u
//
// Bound by memory: 16 bytes an element each way with the residual (x, residual in, h, out out; g, grad_sum, h in,
// grad_x out); over [16384, 4096] the forward takes 174 us, 6.2 TB/s, and the backward 183 and 5 for the sum of grad_w's
// partials, 5.7 TB/s. A row stays in registers between its sums and its results, L lanes of a wavefront a row or a whole
// workgroup, Q quads a lane, so each tensor moves once; rows of more than 16384 elements are read twice. The backward
// takes s again from h, which it reads anyway, rather than keep a tensor of it.
// The sums over a row are in 64 bits: their squares neither overflow nor vanish for any fp32 element, and the
// vector units have the time beside the stream. grad_w's sums over rows are fp32 per workgroup, then over workgroups, in
// a fixed order.
#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int64_t kMaxNormDim = (int64_t)1 << 30;

struct NormArg {
    const float* x;         // forward: x; backward: h
    const float* residual;  // or null
    const float* w;
    float* out;
    float* sum;  // or null
    // backward
    const float* g;
    const float* gsum;  // or null
    float* gx;          // or null
    float* part;        // [blocks][dim], or null without grad_w
    int64_t rows;
    int32_t dim;
    int32_t accumulate;
    double eps;
};

// The sums of two doubles over L neighbouring lanes, or a workgroup for L of more than a wavefront; every lane gets
// them. `red` holds two a wavefront.
template <int L>
__device__ __forceinline__ void row_sums(double& a, double& b, double* red) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    if constexpr (L > 64) {
        constexpr int W = L / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            red[threadIdx.x >> 6] = a;
            red[W + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();
        a = red[0];
        b = red[W];
#pragma unroll
        for (int i = 1; i < W; ++i) {
            a += red[i];
            b += red[W + i];
        }
    }
}

// Quad c of a row of `dim` elements; past its end zeros.
__device__ __forceinline__ vf4 load_quad(const float* row, int c, int dim) {
    if (c + 3 < dim) return *reinterpret_cast<const vf4u*>(row + c);
    vf4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < dim) v.x = row[c];
    if (c + 1 < dim) v.y = row[c + 1];
    if (c + 2 < dim) v.z = row[c + 2];
    return v;
}
__device__ __forceinline__ vf4 load_quad_nt(const float* row, int c, int dim) {
    if (c + 3 < dim) return ld_ntu(row + c);
    return load_quad(row, c, dim);
}
__device__ __forceinline__ void store_quad(float* row, int c, int dim, vf4 v) {
    if (c + 3 < dim) {
        st_ntu(row + c, v);
        return;
    }
    if (c < dim) row[c] = v.x;
    if (c + 1 < dim) row[c + 1] = v.y;
    if (c + 2 < dim) row[c + 2] = v.z;
}
__device__ __forceinline__ double dot4(vf4 a, vf4 b, double s) {
    s = __builtin_fma((double)a.x, (double)b.x, s);
    s = __builtin_fma((double)a.y, (double)b.y, s);
    s = __builtin_fma((double)a.z, (double)b.z, s);
    return __builtin_fma((double)a.w, (double)b.w, s);
}

// s = q 2^e, for s itself may be past fp32's range either way: x s is x 2^e, exact, times q.
struct Scale {
    float q;
    int32_t e;
    __device__ __forceinline__ explicit Scale(double s) : q((float)__builtin_amdgcn_frexp_mant(s)), e(__builtin_amdgcn_frexp_exp(s)) {}
    __device__ __forceinline__ Scale(float mant, int32_t exp) : q(mant), e(exp) {}
    __device__ __forceinline__ vf4 up(vf4 v) const {
        return vf4{__builtin_ldexpf(v.x, e), __builtin_ldexpf(v.y, e), __builtin_ldexpf(v.z, e), __builtin_ldexpf(v.w, e)};
    }
    __device__ __forceinline__ vf4 of(vf4 h) const { return up(h) * q; }
};

template <int L, int Q, int T>
__global__ __launch_bounds__(T) void k_norm_fwd(NormArg a) {
    constexpr int G = T / L;  // rows in flight in a workgroup
    __shared__ double red[2 * (T / 64)];
    const int l = threadIdx.x % L, g = threadIdx.x / L;
    vf4 w[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) w[i] = load_quad(a.w, 4 * (i * L + l), a.dim);
    const int64_t stride = (int64_t)gridDim.x * G;
    // every wavefront walks whole rounds, so that its lanes reduce together
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const bool in = r0 + g < a.rows;
        const int64_t at = (in ? r0 + g : r0) * a.dim;
        vf4 h[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) h[i] = load_quad_nt(a.x + at, 4 * (i * L + l), a.dim);
        if (a.residual) {
            vf4 r[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) r[i] = load_quad_nt(a.residual + at, 4 * (i * L + l), a.dim);
#pragma unroll
            for (int i = 0; i < Q; ++i) h[i] = h[i] + r[i];
        }
        double s = 0.0, none = 0.0;
#pragma unroll
        for (int i = 0; i < Q; ++i) s = dot4(h[i], h[i], s);
        row_sums<L>(s, none, red);
        const Scale scale(1.0 / __builtin_sqrt(s / (double)a.dim + a.eps));
        if (!in) continue;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int c = 4 * (i * L + l);
            if (a.sum) store_quad(a.sum + at, c, a.dim, h[i]);
            store_quad(a.out + at, c, a.dim, scale.of(h[i]) * w[i]);
        }
    }
}

// Rows that no workgroup holds: two reads.
__global__ __launch_bounds__(1024) void k_norm_fwd_long(NormArg a) {
    __shared__ double red[32];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t at = r * a.dim;
        double s = 0.0, none = 0.0;
        for (int c = 4 * threadIdx.x; c < a.dim; c += 4096) {
            vf4 h = load_quad(a.x + at, c, a.dim);
            if (a.residual) h = h + load_quad(a.residual + at, c, a.dim);
            s = dot4(h, h, s);
        }
        row_sums<1024>(s, none, red);
        const Scale scale(1.0 / __builtin_sqrt(s / (double)a.dim + a.eps));
        for (int c = 4 * threadIdx.x; c < a.dim; c += 4096) {
            vf4 h = load_quad(a.x + at, c, a.dim);
            if (a.residual) h = h + load_quad(a.residual + at, c, a.dim);
            if (a.sum) store_quad(a.sum + at, c, a.dim, h);
            store_quad(a.out + at, c, a.dim, scale.of(h) * load_quad(a.w, c, a.dim));
        }
    }
}

// s and mean(w g u) of a row from its sums of h^2 and w g h.
__device__ __forceinline__ Scale row_scales(double hh, double wgh, int dim, double eps, float& mean) {
    const double s = 1.0 / __builtin_sqrt(hh / (double)dim + eps);
    mean = (float)(wgh * s / (double)dim);
    return Scale(s);
}
__device__ __forceinline__ vf4 row_grad(vf4 wg, vf4 u, Scale scale, float mean) { return scale.up((wg - u * mean) * scale.q); }

template <int L, int Q, int T>
__global__ __launch_bounds__(T) void k_norm_bwd(NormArg a) {
    constexpr int G = T / L;
    constexpr bool kLate = T == 1024;  // 128 registers a thread: grad_sum is read behind the sums
    __shared__ double red[2 * (T / 64)];
    const int l = threadIdx.x % L, g = threadIdx.x / L;
    vf4 w[Q], acc[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        w[i] = load_quad(a.w, 4 * (i * L + l), a.dim);
        acc[i] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int64_t stride = (int64_t)gridDim.x * G;
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const bool in = r0 + g < a.rows;
        const int64_t at = (in ? r0 + g : r0) * a.dim;
        vf4 h[Q], d[Q], k[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) h[i] = load_quad_nt(a.x + at, 4 * (i * L + l), a.dim);
#pragma unroll
        for (int i = 0; i < Q; ++i) d[i] = load_quad_nt(a.g + at, 4 * (i * L + l), a.dim);
#pragma unroll
        for (int i = 0; i < Q; ++i)
            k[i] = !kLate && a.gsum ? load_quad_nt(a.gsum + at, 4 * (i * L + l), a.dim) : vf4{0.0f, 0.0f, 0.0f, 0.0f};
        double hh = 0.0, wgh = 0.0;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            hh = dot4(h[i], h[i], hh);
            wgh = dot4(d[i] * w[i], h[i], wgh);
        }
        row_sums<L>(hh, wgh, red);
        float mean;
        const Scale scale = row_scales(hh, wgh, a.dim, a.eps, mean);
        if (!in) continue;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int c = 4 * (i * L + l);
            const vf4 u = scale.of(h[i]);
            acc[i] += d[i] * u;
            if (a.gx) {
                vf4 o = row_grad(d[i] * w[i], u, scale, mean);
                if (a.gsum) o = o + (kLate ? load_quad_nt(a.gsum + at, c, a.dim) : k[i]);
                if (a.accumulate) o = o + load_quad_nt(a.gx + at, c, a.dim);
                store_quad(a.gx + at, c, a.dim, o);
            }
        }
    }
    if (!a.part) return;
    // the workgroup's rows together: halves of the groups in turn
    if constexpr (G > 1) {
        __shared__ vf4 buf[G / 2 * L * Q];
#pragma unroll
        for (int half = G / 2; half > 0; half >>= 1) {
            __syncthreads();
            if (g >= half && g < 2 * half) {
#pragma unroll
                for (int i = 0; i < Q; ++i) buf[((g - half) * Q + i) * L + l] = acc[i];
            }
            __syncthreads();
            if (g < half) {
#pragma unroll
                for (int i = 0; i < Q; ++i) acc[i] += buf[(g * Q + i) * L + l];
            }
        }
    }
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int c = 4 * (i * L + l);
            float* o = a.part + (int64_t)blockIdx.x * a.dim;
            if (c + 3 < a.dim) {
                *reinterpret_cast<vf4u*>(o + c) = acc[i];
            } else {
                if (c < a.dim) o[c] = acc[i].x;
                if (c + 1 < a.dim) o[c + 1] = acc[i].y;
                if (c + 2 < a.dim) o[c + 2] = acc[i].z;
            }
        }
    }
}

struct RowScale {
    float q;
    int32_t e;
    float mean;
};
// Long rows: their scales first, then workgroups of 4096 columns over a share of the rows.
__global__ __launch_bounds__(1024) void k_norm_scales_long(NormArg a, RowScale* scales) {
    __shared__ double red[32];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t at = r * a.dim;
        double hh = 0.0, wgh = 0.0;
        for (int c = 4 * threadIdx.x; c < a.dim; c += 4096) {
            const vf4 h = load_quad(a.x + at, c, a.dim);
            hh = dot4(h, h, hh);
            wgh = dot4(load_quad(a.g + at, c, a.dim) * load_quad(a.w, c, a.dim), h, wgh);
        }
        row_sums<1024>(hh, wgh, red);
        float mean;
        const Scale scale = row_scales(hh, wgh, a.dim, a.eps, mean);
        if (threadIdx.x == 0) scales[r] = RowScale{scale.q, scale.e, mean};
    }
}
__global__ __launch_bounds__(256) void k_norm_bwd_long(NormArg a, const RowScale* scales) {
    vf4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    const int c0 = 4096 * blockIdx.x + 4 * threadIdx.x;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const int64_t at = r * a.dim;
        const float mean = scales[r].mean;
        const Scale scale(scales[r].q, scales[r].e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 1024 * i;
            if (c >= a.dim) continue;
            const vf4 d = load_quad(a.g + at, c, a.dim), u = scale.of(load_quad(a.x + at, c, a.dim));
            acc[i] += d * u;
            if (a.gx) {
                vf4 o = row_grad(d * load_quad(a.w, c, a.dim), u, scale, mean);
                if (a.gsum) o = o + load_quad(a.gsum + at, c, a.dim);
                if (a.accumulate) o = o + load_quad(a.gx + at, c, a.dim);
                store_quad(a.gx + at, c, a.dim, o);
            }
        }
    }
    if (!a.part) return;
    float* o = a.part + (int64_t)blockIdx.y * a.dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = c0 + 1024 * i;
        if (c < a.dim) o[c] = acc[i].x;
        if (c + 1 < a.dim) o[c + 1] = acc[i].y;
        if (c + 2 < a.dim) o[c + 2] = acc[i].z;
        if (c + 3 < a.dim) o[c + 3] = acc[i].w;
    }
}

// grad_w from the workgroups' partials: 32 columns and 8 shares of the partials a workgroup.
__global__ __launch_bounds__(256) void k_norm_grad_w(const float* part, int32_t blocks, int32_t dim, float* grad_w,
                                                     int accumulate) {
    __shared__ float buf[256];
    const int col = threadIdx.x & 31, share = threadIdx.x >> 5;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < dim; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + col;
        float s = 0.0f;
        if (c < dim) {
#pragma unroll 8
            for (int b = share; b < blocks; b += 8) s += part[(int64_t)b * dim + c];
        }
        __syncthreads();
        buf[threadIdx.x] = s;
        __syncthreads();
        if (share != 0 || c >= dim) continue;
#pragma unroll
        for (int i = 1; i < 8; ++i) s += buf[32 * i + col];
        grad_w[c] = accumulate ? grad_w[c] + s : s;
    }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
// Lanes a row, quads a lane and threads a workgroup by the row's length.
#define MH_NORM(CALL)                            \
    do {                                         \
        if (a.dim <= 16) CALL(4, 1, 256);        \
        else if (a.dim <= 32) CALL(8, 1, 256);   \
        else if (a.dim <= 64) CALL(8, 2, 256);   \
        else if (a.dim <= 128) CALL(16, 2, 256); \
        else if (a.dim <= 256) CALL(32, 2, 256); \
        else if (a.dim <= 512) CALL(64, 2, 256); \
        else if (a.dim <= 768) CALL(64, 3, 256); \
        else if (a.dim <= 1024) CALL(64, 4, 256); \
        else if (a.dim <= 2048) CALL(256, 2, 256); \
        else if (a.dim <= 4096) CALL(256, 4, 256); \
        else if (a.dim <= 8192) CALL(512, 4, 512); \
        else CALL(1024, 4, 1024);                \
    } while (0)
constexpr int kNormRow = 16384;  // the longest row that a workgroup holds

// Rows in flight in a workgroup of MH_NORM's.
int norm_group(int dim) {
    return dim <= 16 ? 64 : dim <= 64 ? 32 : dim <= 128 ? 16 : dim <= 256 ? 8 : dim <= 1024 ? 4 : 1;
}

int norm_check(const char* what, int64_t rows, int64_t dim, float eps) {
    if (rows < 0 || dim < 1) return fail(MH_ERR_INVALID, "%s: needs rows >= 0 and dim >= 1 (%lld, %lld)", what, (long long)rows, (long long)dim);
    if (!(eps >= 0.0f) || eps > 3.4028234663852886e38f) return fail(MH_ERR_INVALID, "%s: eps %g is negative or no number", what, (double)eps);
    if (dim > kMaxNormDim || rows > ((int64_t)1 << 46) / dim) return fail(MH_ERR_OVERFLOW, "%s: rows of more than 2^30 elements, or more than 2^46 in all", what);
    return MH_OK;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_rms_norm_fwd(float* out, float* sum, const float* x, const float* residual, const float* w, int64_t rows, int64_t dim,
                    float eps) {
    MH_TRACE("mh_rms_norm_fwd");
    MH_TRY(norm_check("mh_rms_norm_fwd", rows, dim, eps));
    if (rows == 0) return MH_OK;
    if (!out || !x || !w) return fail(MH_ERR_NULL, "mh_rms_norm_fwd: null tensor");
    MH_TRY(require_init());
    NormArg a = {};
    a.x = x;
    a.residual = residual;
    a.w = w;
    a.out = out;
    a.sum = sum;
    a.rows = rows;
    a.dim = (int32_t)dim;
    a.eps = (double)eps;
    hipStream_t st = ctx().stream;
    if (dim > kNormRow) {
        const int64_t blocks = rows < 512 ? rows : 512;
        hipLaunchKernelGGL(k_norm_fwd_long, dim3((unsigned)blocks), dim3(1024), 0, st, a);
        return finish("mh_rms_norm_fwd");
    }
    // a workgroup for each round of rows, as many as a dispatch holds of 1024 threads: [16384, 4096] 174 us, 185 with 2048
    const int64_t group = norm_group(a.dim);
    int64_t blocks = (rows + group - 1) / group;
    if (blocks > max_grid_blocks(1024)) blocks = max_grid_blocks(1024);
#define MH_CALL(L, Q, T) hipLaunchKernelGGL((k_norm_fwd<L, Q, T>), dim3((unsigned)blocks), dim3(T), 0, st, a)
    MH_NORM(MH_CALL);
#undef MH_CALL
    return finish("mh_rms_norm_fwd");
}

int mh_rms_norm_bwd(float* grad_x, float* grad_w, const float* grad_out, const float* grad_sum, const float* h, const float* w,
                    int64_t rows, int64_t dim, float eps, int accumulate) {
    MH_TRACE("mh_rms_norm_bwd");
    MH_TRY(norm_check("mh_rms_norm_bwd", rows, dim, eps));
    if (!grad_x && !grad_w) return MH_OK;
    if (rows > 0 && (!grad_out || !h || !w)) return fail(MH_ERR_NULL, "mh_rms_norm_bwd: null tensor");
    if (rows == 0) return grad_w && !accumulate ? mh_zero(grad_w, dim) : MH_OK;
    MH_TRY(require_init());
    NormArg a = {};
    a.x = h;
    a.w = w;
    a.g = grad_out;
    a.gsum = grad_sum;
    a.gx = grad_x;
    a.rows = rows;
    a.dim = (int32_t)dim;
    a.accumulate = accumulate != 0;
    a.eps = (double)eps;
    hipStream_t st = ctx().stream;
    const bool lng = dim > kNormRow;
    const int64_t group = lng ? 1 : norm_group(a.dim);
    int64_t blocks = (rows + group - 1) / group;
    // as many workgroups as the chip holds at once, for few partials of grad_w: two of 256 threads a CU over rows of 1025 to
    // 4096 (512: 188 us with the partials' sum, 768: 189, 1536: 196, 256: 252, over [16384, 4096]), one of more, four of short rows
    const int64_t most = lng ? 64 : dim > 4096 ? 256 : dim > 1024 ? 512 : 1024;
    if (blocks > most) blocks = most;
    float* base = nullptr;
    const size_t part = grad_w ? (size_t)blocks * dim * 4 : 0, scales = lng ? (size_t)rows * sizeof(RowScale) : 0;
    if (part + scales) MH_TRY(scratch(scales + part, reinterpret_cast<void**>(&base)));
    if (grad_w) a.part = base + scales / 4;
    if (lng) {
        RowScale* sc = reinterpret_cast<RowScale*>(base);
        hipLaunchKernelGGL(k_norm_scales_long, dim3((unsigned)(rows < 512 ? rows : 512)), dim3(1024), 0, st, a, sc);
        hipLaunchKernelGGL(k_norm_bwd_long, dim3((unsigned)((dim + 4095) / 4096), (unsigned)blocks), dim3(256), 0, st, a, sc);
    } else {
#define MH_CALL(L, Q, T) hipLaunchKernelGGL((k_norm_bwd<L, Q, T>), dim3((unsigned)blocks), dim3(T), 0, st, a)
        MH_NORM(MH_CALL);
#undef MH_CALL
    }
    if (grad_w) {
        const int64_t cols = (dim + 31) / 32, fit = max_grid_blocks(256);
        hipLaunchKernelGGL(k_norm_grad_w, dim3((unsigned)(cols < fit ? cols : fit)), dim3(256), 0, st, a.part, (int32_t)blocks, a.dim,
                           grad_w, a.accumulate);
    }
    return finish("mh_rms_norm_bwd");
}

}  // extern "C"
