// mh_distill.hip -- distillation: the divergence of a student's softmax over all classes from a teacher's
// over its top k, and the gradient of the student's logits.
//
//   q = softmax(teacher / T) over a row's entries;  p = softmax(x / T);  lse = log sum_v exp(x_v / T)
//   loss = T^2 / n sum_rows sum_k q_k (log q_k - x_id / T + lse);  grad_v = ug T / n (p_v - sum_{id_k = v} q_k)
//
// The logits are all that is large: the floor is one read of x and one write of its gradient. One workgroup
// takes a row, holds a row of up to 32768 classes in registers between its statistics and its gradient, and
// reads a longer one twice, the second time from its end, where the caches still hold it. Where rows are
// fewer than CUs, a row is shared by several workgroups: their statistics, then the gradient.
// An exponential is a difference, a product with log2(e) / T and one instruction; sums are fp32 over at most C / 1024 elements a thread, then a tree.
#include "mh_internal.h"
#include "mh_math.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kMaxK = 1024;      // entries of a row: LDS holds their ids and weights
constexpr int kCountBlocks = 256;

struct DistillArg {
    const float* x;
    const int32_t* ids;
    const float* teacher;
    const float* ug;
    const float* lse_in;  // rows' log-sum-exp of the forward, or null
    float* grad;
    float* row_lse;   // or null
    float* row_loss;  // scratch
    const int32_t* kept;  // [kCountBlocks] partial counts of rows with an entry
    float* stat;      // [rows][splits][2] or null
    int64_t rows, classes;
    int32_t k, splits;
    int64_t span;     // classes of a split, a multiple of 4
    float inv_t, temperature;
};

__device__ __forceinline__ bool entry(int32_t id, float t) { return id >= 0 && t != -__builtin_inff(); }

// Rows with an entry, as partial counts: a wavefront a row.
__global__ __launch_bounds__(256) void k_distill_count(int32_t* part, const int32_t* ids, const float* teacher,
                                                       int64_t rows, int32_t k) {
    __shared__ int32_t red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t n = 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < rows; r += kCountBlocks * 4) {
        bool any = false;
        for (int32_t i = lane; i < k; i += 64) any = any || entry(ids[r * k + i], teacher[r * k + i]);
        n += __any(any) ? 1 : 0;
    }
    if (lane == 0) red[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// A row's entries in LDS: ids (-1: none) and q.
struct Entries {
    int32_t id[kMaxK];
    float q[kMaxK];
    float u[kMaxK];  // log q
};

// Fills e for row r. Returns 0 where the row has no entry, 2 where an id is past the classes, else 1.
template <int W>
__device__ int load_entries(const DistillArg& a, int64_t r, Entries& e, float* red) {
    const int tid = threadIdx.x;
    float best = -__builtin_inff();
    bool any = false, bad = false;
    for (int i = tid; i < a.k; i += W * 64) {
        const int32_t id = a.ids[r * a.k + i];
        const float t = a.teacher[r * a.k + i];
        const bool in = entry(id, t);
        any = any || in;
        bad = bad || (in && id >= a.classes);
        e.id[i] = in ? id : -1;
        e.u[i] = in ? t * a.inv_t : -__builtin_inff();
        if (in) best = __builtin_fmaxf(best, t * a.inv_t);
    }
    const int what = (__syncthreads_or(any) ? 1 : 0) | (__syncthreads_or(bad) ? 2 : 0);
    if (what != 1) return what ? 2 : 0;
    best = block_max<W>(best, red);
    float mass = 0.0f;
    for (int i = tid; i < a.k; i += W * 64) {
        const float v = e.id[i] >= 0 ? exp_neg(e.u[i] - best) : 0.0f;
        e.q[i] = v;
        mass += v;
    }
    mass = block_sum<W>(mass, red);
    const float lm = mlog(mass);
    for (int i = tid; i < a.k; i += W * 64) {
        e.q[i] = e.q[i] / mass;
        e.u[i] = e.u[i] - best - lm;
    }
    __syncthreads();
    return 1;
}

// The row's loss before T^2 / n from its entries and log-sum-exp.
template <int W>
__device__ float row_loss_of(const DistillArg& a, int64_t r, const Entries& e, float lse, float* red) {
    float s = 0.0f;
    for (int i = threadIdx.x; i < a.k; i += W * 64)
        if (e.id[i] >= 0 && e.q[i] != 0.0f) s += e.q[i] * (e.u[i] - (a.x[r * a.classes + e.id[i]] * a.inv_t - lse));
    return block_sum<W>(s, red);
}

// The entries' elements of the gradient, c0..c1 of row r: written after the dense part, each by the first
// entry of its class, which adds up those of the same class in their order.
template <int W, bool ACC>
__device__ __forceinline__ float entry_old(const DistillArg& a, int64_t at) { return ACC ? a.grad[at] : 0.0f; }

template <int W>
__device__ __forceinline__ bool entry_first(const DistillArg& a, const Entries& e, int i, int64_t c0, int64_t c1,
                                            float* q) {
    const int32_t id = e.id[i];
    if (id < c0 || id >= c1) return false;
    float s = 0.0f;
    for (int j = 0; j < a.k; ++j)
        if (e.id[j] == id) {
            if (j < i) return false;
            s += e.q[j];
        }
    *q = s;
    return true;
}

__device__ __forceinline__ int32_t kept_rows(const int32_t* part) {
    const int lane = threadIdx.x & 63;
    int32_t n = 0;
#pragma unroll
    for (int i = 0; i < kCountBlocks / 64; ++i) n += part[lane + 64 * i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    return n > 0 ? n : 1;
}

// Running maximum and sum of exponentials, in base 2: t = x log2(e) / T.
struct Run {
    float top, sum;
};
__device__ __forceinline__ void run_add(Run& r, vf4 v, float kf) {
    const float m = __builtin_fmaxf(__builtin_fmaxf(v.x, v.y), __builtin_fmaxf(v.z, v.w));
    if (m > r.top) {
        r.sum *= __builtin_amdgcn_exp2f((r.top - m) * kf);
        r.top = m;
    }
    // the difference first: log2(e) times the type's lowest value would be infinite
    const float b = r.top == -__builtin_inff() ? 0.0f : r.top;
    r.sum += (__builtin_amdgcn_exp2f((v.x - b) * kf) + __builtin_amdgcn_exp2f((v.y - b) * kf)) +
             (__builtin_amdgcn_exp2f((v.z - b) * kf) + __builtin_amdgcn_exp2f((v.w - b) * kf));
}
template <int W>
__device__ __forceinline__ Run run_join(Run r, float kf, float* red) {
    const float top = block_max<W>(r.top, red);
    const float s = r.top == -__builtin_inff() ? r.sum : r.sum * __builtin_amdgcn_exp2f((r.top - top) * kf);
    return {top, block_sum<W>(s, red)};
}

// A logit's probability from the row's maximum and sum, p = e^((x - top) / T) / sum, or from its log-sum-exp,
// p = e^(x / T - lse) with x / T - lse rounded once: where the logits are so large that the log-sum-exp's own
// rounding counts, the difference is held at 0, so that p stays below 1.
template <bool LSE>
struct Scale {
    float f, from, inv;  // 1 / T, lse; or log2(e) / T, top, 1 / sum
};
__device__ __forceinline__ float prob(const Scale<true>& s, float x) {
    const float d = __builtin_fmaf(x, s.f, -s.from);
    return __builtin_amdgcn_exp2f((d > 0.0f ? 0.0f : d) * kLog2e);
}
__device__ __forceinline__ float prob(const Scale<false>& s, float x) {
    return __builtin_amdgcn_exp2f((x - s.from) * s.f) * s.inv;
}
template <bool LSE>
__device__ __forceinline__ vf4 grad4(const Scale<LSE>& s, vf4 v, float c) {
    return {prob(s, v.x) * c, prob(s, v.y) * c, prob(s, v.z) * c, prob(s, v.w) * c};
}

// A row left out: its gradient is left alone, or zero.
template <int W, bool ACC>
__device__ void row_zero(const DistillArg& a, int64_t r, int64_t c0, int64_t c1) {
    if (ACC) return;
    float* g = a.grad + r * a.classes;
    const vf4 z = {0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t q1 = c0 + ((c1 - c0) & ~(int64_t)3);
    for (int64_t c = c0 + threadIdx.x * 4; c < q1; c += W * 256) st_ntu(g + c, z);
    if ((int64_t)threadIdx.x < c1 - q1) g[q1 + threadIdx.x] = 0.0f;
}

// Classes c0..c1 of row r's gradient.
template <int W, bool ACC, bool LSE>
__device__ void row_grad(const DistillArg& a, int64_t r, int64_t c0, int64_t c1, const Entries& e, const Scale<LSE>& s,
                         float c) {
    const float* x = a.x + r * a.classes;
    float* g = a.grad + r * a.classes;
    const int tid = threadIdx.x;
    // each thread's entries before the dense part writes over them; kMaxK / (W * 64) at most
    constexpr int NE = (kMaxK + W * 64 - 1) / (W * 64);
    float mine[NE];
    int32_t at[NE];
#pragma unroll
    for (int u = 0; u < NE; ++u) {
        const int i = tid + u * W * 64;
        float q = 0.0f;
        at[u] = -1;
        if (i < a.k && entry_first<W>(a, e, i, c0, c1, &q)) {
            at[u] = e.id[i];
            mine[u] = (prob(s, x[at[u]]) - q) * c;
            if (ACC) mine[u] = g[at[u]] + mine[u];
        }
    }
    __syncthreads();
    const int64_t nq = (c1 - c0) >> 2;
    const int tail = (int)((c1 - c0) & 3);
    for (int64_t q = nq - 1 - tid; q >= 0; q -= W * 64) {  // from the end, which was read last
        float* o = g + c0 + 4 * q;
        vf4 v = grad4(s, ld_ntu(x + c0 + 4 * q), c);
        if (ACC) {
            const vf4 old = ld_ntu(o);
            v = {old.x + v.x, old.y + v.y, old.z + v.z, old.w + v.w};
        }
        st_ntu(o, v);
    }
    if (tid < tail) {
        const int64_t p = c0 + 4 * nq + tid;
        const float v = prob(s, x[p]) * c;
        g[p] = ACC ? g[p] + v : v;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NE; ++u)
        if (at[u] >= 0) g[at[u]] = mine[u];
}

// A whole row a workgroup: statistics, loss and, with GRAD, the gradient.
template <int W, bool GRAD, bool ACC>
__global__ __launch_bounds__(W * 64) void k_distill_row(DistillArg a) {
    __shared__ Entries e;
    __shared__ float red[W];
    const int64_t r = blockIdx.x;
    const int what = load_entries<W>(a, r, e, red);
    if (what == 0) {
        if (threadIdx.x == 0) {
            a.row_loss[r] = 0.0f;
            if (a.row_lse) a.row_lse[r] = 0.0f;
        }
        if (GRAD) row_zero<W, ACC>(a, r, 0, a.classes);
        return;
    }
    const float kf = a.inv_t * kLog2e;
    const float* x = a.x + r * a.classes;
    Run run = {-__builtin_inff(), 0.0f};
    const int64_t nq = a.classes >> 2;
    for (int64_t q = threadIdx.x; q < nq; q += W * 64) run_add(run, *reinterpret_cast<const vf4u*>(x + 4 * q), kf);
    const int tail = (int)(a.classes & 3);
    if ((int)threadIdx.x < tail) {
        const float ninf = -__builtin_inff();
        run_add(run, vf4{x[4 * nq + threadIdx.x], ninf, ninf, ninf}, kf);
    }
    run = run_join<W>(run, kf, red);
    float lse = run.top * a.inv_t + mlog(run.sum);
    if (what == 2) lse = __builtin_nanf("");  // an id past the classes: shown in the loss and the gradient
    const float loss = what == 2 ? lse : row_loss_of<W>(a, r, e, lse, red);
    if (threadIdx.x == 0) {
        a.row_loss[r] = loss;
        if (a.row_lse) a.row_lse[r] = lse;
    }
    if (GRAD) {
        const float c = a.ug[0] * a.temperature / (float)kept_rows(a.kept);
        if (what == 2) {  // NaN all over the row, entries or not
            for (int i = threadIdx.x; i < a.k; i += W * 64) e.id[i] = -1;
            __syncthreads();
        }
        const Scale<false> s = {kf, run.top, 1.0f / (what == 2 ? lse : run.sum)};
        row_grad<W, ACC>(a, r, 0, a.classes, e, s, c);
    }
}

// A split of a row: its maximum and sum.
template <int W>
__global__ __launch_bounds__(W * 64) void k_distill_stat(DistillArg a) {
    __shared__ float red[W];
    const int64_t r = blockIdx.x / a.splits, sp = blockIdx.x % a.splits;
    const int64_t c0 = sp * a.span, c1 = c0 + a.span < a.classes ? c0 + a.span : a.classes;
    const float kf = a.inv_t * kLog2e;
    const float* x = a.x + r * a.classes;
    Run run = {-__builtin_inff(), 0.0f};
    const int64_t nq = (c1 - c0) >> 2;
    for (int64_t q = threadIdx.x; q < nq; q += W * 64) run_add(run, *reinterpret_cast<const vf4u*>(x + c0 + 4 * q), kf);
    const int tail = (int)((c1 - c0) & 3);
    if ((int)threadIdx.x < tail) {
        const float ninf = -__builtin_inff();
        run_add(run, vf4{x[c0 + 4 * nq + threadIdx.x], ninf, ninf, ninf}, kf);
    }
    run = run_join<W>(run, kf, red);
    if (threadIdx.x == 0) {
        a.stat[blockIdx.x * 2] = run.top;
        a.stat[blockIdx.x * 2 + 1] = run.sum;
    }
}

// A row's maximum and sum from its splits', in their order.
__device__ __forceinline__ Run join_splits(const DistillArg& a, int64_t r) {
    const float* st = a.stat + r * a.splits * 2;
    float top = -__builtin_inff(), sum = 0.0f;
    for (int i = 0; i < a.splits; ++i) top = __builtin_fmaxf(top, st[2 * i]);
    const float kf = a.inv_t * kLog2e;
    for (int i = 0; i < a.splits; ++i)
        sum += st[2 * i] == -__builtin_inff() ? st[2 * i + 1] : st[2 * i + 1] * __builtin_amdgcn_exp2f((st[2 * i] - top) * kf);
    return {top, sum};
}

// A split of a row's gradient, from the forward's log-sum-exp or the splits' statistics; with LOSS the first
// split writes the row's loss. GRAD off: the loss alone, a workgroup a row.
template <int W, bool LOSS, bool GRAD, bool ACC>
__global__ __launch_bounds__(W * 64) void k_distill_split(DistillArg a) {
    __shared__ Entries e;
    __shared__ float red[W];
    const int32_t per = GRAD ? a.splits : 1;
    const int64_t r = blockIdx.x / per, sp = blockIdx.x % per;
    const int64_t c0 = sp * a.span, c1 = c0 + a.span < a.classes ? c0 + a.span : a.classes;
    const int what = load_entries<W>(a, r, e, red);
    if (what == 0) {
        if (LOSS && sp == 0 && threadIdx.x == 0) {
            a.row_loss[r] = 0.0f;
            if (a.row_lse) a.row_lse[r] = 0.0f;
        }
        if (GRAD) row_zero<W, ACC>(a, r, c0, c1);
        return;
    }
    float lse;
    if (LOSS) {
        const Run run = join_splits(a, r);
        lse = run.top * a.inv_t + mlog(run.sum);
    } else {
        lse = a.lse_in[r];
    }
    if (what == 2) lse = __builtin_nanf("");
    if (LOSS && sp == 0) {
        const float loss = what == 2 ? lse : row_loss_of<W>(a, r, e, lse, red);
        if (threadIdx.x == 0) {
            a.row_loss[r] = loss;
            if (a.row_lse) a.row_lse[r] = lse;
        }
    }
    if (GRAD) {
        const float c = a.ug[0] * a.temperature / (float)kept_rows(a.kept);
        if (what == 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < a.k; i += W * 64) e.id[i] = -1;
            __syncthreads();
        }
        if (LOSS) {  // the splits' statistics are there
            const Run run = join_splits(a, r);
            const Scale<false> s = {a.inv_t * kLog2e, run.top, 1.0f / (what == 2 ? lse : run.sum)};
            row_grad<W, ACC>(a, r, c0, c1, e, s, c);
        } else {
            const Scale<true> s = {a.inv_t, lse, 1.0f};
            row_grad<W, ACC>(a, r, c0, c1, e, s, c);
        }
    }
}

// loss = T^2 / n sum of the rows' losses, in a fixed order.
__global__ __launch_bounds__(1024) void k_distill_loss(const float* row_loss, int64_t rows, const int32_t* kept,
                                                       float temperature, float* loss) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 4
    for (int64_t n = threadIdx.x; n < rows; n += 1024) s += (double)row_loss[n];
    s = block_sum<16>(s, red);
    const double n = kept_rows(kept);
    if (threadIdx.x == 0) loss[0] = (float)(s * ((double)temperature * temperature) / n);
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
struct DistillCall {
    const char* what;
    float *loss, *row_lse, *grad;
    const float* lse_in;
    const float* x;
    const int32_t* ids;
    const float* teacher;
    const float* ug;
    int64_t rows, classes, k;
    float temperature;
    bool accumulate;
};

int distill_check(const DistillCall& d) {
    if (d.rows < 0 || d.classes < 1 || d.k < 1 || d.k > kMaxK)
        return fail(MH_ERR_INVALID, "%s: needs rows >= 0, classes >= 1, 1 <= k <= %d (%lld, %lld, %lld)", d.what, kMaxK,
                    (long long)d.rows, (long long)d.classes, (long long)d.k);
    if (!(d.temperature >= 1.0e-6f && d.temperature <= 1.0e6f))
        return fail(MH_ERR_INVALID, "%s: the temperature must lie in 1e-6..1e6", d.what);
    if (d.classes > 0x7fffffff || d.rows > max_grid_blocks(1024))
        return fail(MH_ERR_OVERFLOW, "%s: more than 2^31 - 1 classes, or more rows than one dispatch holds", d.what);
    return MH_OK;
}

// Workgroups that share a row: one where rows fill the chip or are short, else up to what gives every CU two.
int row_splits(int64_t rows, int64_t classes) {
    const int64_t want = 2 * (int64_t)ctx().num_cus / (rows > 0 ? rows : 1);
    int64_t s = classes / 8192;
    if (s > want) s = want;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

int distill_run(const DistillCall& d) {
    DistillArg a = {};
    a.x = d.x;
    a.ids = d.ids;
    a.teacher = d.teacher;
    a.ug = d.ug;
    a.lse_in = d.lse_in;
    a.grad = d.grad;
    a.row_lse = d.row_lse;
    a.rows = d.rows;
    a.classes = d.classes;
    a.k = (int32_t)d.k;
    a.temperature = d.temperature;
    a.inv_t = 1.0f / d.temperature;
    a.splits = row_splits(d.rows, d.classes);
    a.span = ((d.classes + a.splits - 1) / a.splits + 3) & ~(int64_t)3;
    a.splits = (int32_t)((d.classes + a.span - 1) / a.span);
    const size_t n_kept = kCountBlocks * sizeof(int32_t);
    const size_t n_loss = ((size_t)d.rows * sizeof(float) + 255) & ~(size_t)255;
    char* base = nullptr;
    MH_TRY(scratch(n_kept + n_loss + (size_t)d.rows * a.splits * 2 * sizeof(float), reinterpret_cast<void**>(&base)));
    int32_t* kept = reinterpret_cast<int32_t*>(base);
    a.kept = kept;
    a.row_loss = reinterpret_cast<float*>(base + n_kept);
    a.stat = reinterpret_cast<float*>(base + n_kept + n_loss);
    hipStream_t st = ctx().stream;
    hipLaunchKernelGGL(k_distill_count, dim3(kCountBlocks), dim3(256), 0, st, kept, d.ids, d.teacher, d.rows, a.k);
    constexpr int W = 16;
    const dim3 rows((unsigned)d.rows), all((unsigned)(d.rows * a.splits)), t(W * 64);
    const bool grad = d.grad != nullptr;
    if (d.lse_in) {
        if (d.accumulate) hipLaunchKernelGGL((k_distill_split<W, false, true, true>), all, t, 0, st, a);
        else hipLaunchKernelGGL((k_distill_split<W, false, true, false>), all, t, 0, st, a);
    } else if (a.splits == 1) {
        if (!grad) hipLaunchKernelGGL((k_distill_row<W, false, false>), rows, t, 0, st, a);
        else if (d.accumulate) hipLaunchKernelGGL((k_distill_row<W, true, true>), rows, t, 0, st, a);
        else hipLaunchKernelGGL((k_distill_row<W, true, false>), rows, t, 0, st, a);
    } else {
        hipLaunchKernelGGL((k_distill_stat<W>), all, t, 0, st, a);
        if (!grad) hipLaunchKernelGGL((k_distill_split<W, true, false, false>), rows, t, 0, st, a);
        else if (d.accumulate) hipLaunchKernelGGL((k_distill_split<W, true, true, true>), all, t, 0, st, a);
        else hipLaunchKernelGGL((k_distill_split<W, true, true, false>), all, t, 0, st, a);
    }
    if (d.loss)
        hipLaunchKernelGGL(k_distill_loss, dim3(1), dim3(1024), 0, st, a.row_loss, d.rows, kept, d.temperature, d.loss);
    return finish(d.what);
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_distill_fwd(float* loss, float* row_lse, const float* x, const int32_t* ids, const float* teacher, int64_t rows,
                   int64_t classes, int64_t k, float temperature) {
    MH_TRACE("mh_distill_fwd");
    const DistillCall d = {"mh_distill_fwd", loss, row_lse, nullptr, nullptr, x, ids, teacher, nullptr, rows, classes, k,
                           temperature, false};
    MH_TRY(distill_check(d));
    if (!loss || (rows > 0 && (!x || !ids || !teacher))) return fail(MH_ERR_NULL, "%s: null tensor", d.what);
    MH_TRY(require_init());
    if (rows == 0) return mh_fill(loss, 0.0f, 1);
    return distill_run(d);
}

int mh_distill_bwd(float* grad_x, const float* x, const int32_t* ids, const float* teacher, const float* row_lse,
                   const float* ug, int64_t rows, int64_t classes, int64_t k, float temperature, int accumulate) {
    MH_TRACE("mh_distill_bwd");
    const DistillCall d = {"mh_distill_bwd", nullptr, nullptr, grad_x, row_lse, x, ids, teacher, ug, rows, classes, k,
                           temperature, accumulate != 0};
    MH_TRY(distill_check(d));
    if (rows == 0) return MH_OK;
    if (!grad_x || !x || !ids || !teacher || !row_lse || !ug) return fail(MH_ERR_NULL, "%s: null tensor", d.what);
    MH_TRY(require_init());
    return distill_run(d);
}

int mh_distill_step(float* loss, float* row_lse, float* grad_x, const float* x, const int32_t* ids,
                    const float* teacher, const float* ug, int64_t rows, int64_t classes, int64_t k, float temperature,
                    int accumulate) {
    MH_TRACE("mh_distill_step");
    const DistillCall d = {"mh_distill_step", loss, row_lse, grad_x, nullptr, x, ids, teacher, ug, rows, classes, k,
                           temperature, accumulate != 0};
    MH_TRY(distill_check(d));
    if (!loss || (rows > 0 && (!grad_x || !x || !ids || !teacher || !ug)))
        return fail(MH_ERR_NULL, "%s: null tensor", d.what);
    MH_TRY(require_init());
    if (rows == 0) return mh_fill(loss, 0.0f, 1);
    return distill_run(d);
}

}  // extern "C"
