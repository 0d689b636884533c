// mh_distill.hip -- distillation: the divergence of a student's softmax over all classes from a teacher's
// over its top k, and the gradient of the student's logits.
//
//   q = softmax(teacher / T) over a row's entries;  p = softmax(x / T);  lse = log sum_v exp(x_v / T)
//   loss = T^2 / n sum_rows sum_k q_k (log q_k - x_id / T + lse);  grad_v = ug T / n (p_v - sum_{id_k = v} q_k)
//
// The logits are all that is large: the floor is one read of x and one write of its gradient. A first kernel
// takes the entries, a wavefront a row: q, the logit at each id, entries of one class joined. A chain of loads
// that depend on each other, it would stand in the way of the stream (70 -> 64 us over [1025, 30011], 50
// entries). Then a workgroup takes a row: of up to 65536 classes it holds it in registers and reads it
// once; a longer one it reads twice, the second time from its end, where the caches still hold it. Where
// rows are fewer than CUs, several workgroups share a row: their statistics, then the gradient.
// An exponential is a difference, a product with log2(e) / T and one instruction; sums are fp32, of C / (64 W)
// elements a thread of a workgroup of W wavefronts (at most 16 of a row held by one, 32 by 4 to 16, 64 of more than
// 32768 classes; C / 1024 of rows that are not held), then a tree.
#include "mh_internal.h"
#include "mh_math.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kMaxK = 1024;       // entries of a row
constexpr int kEntryBlocks = 1024;  // workgroups of k_distill_entries at most
constexpr int kTicketStride = 32;   // counters in use lie in 128-byte lines of their own
constexpr int64_t kHeld = 65536;  // classes of a row that a CU holds

struct DistillArg {
    const float* x;
    const int32_t* ids;
    const float* teacher;
    const float* ug;
    const float* lse_in;  // rows' log-sum-exp of the forward, or null
    float* grad;
    float* row_lse;  // or null
    // of k_distill_entries
    int32_t* kept;    // rows with an entry
    uint32_t* tickets;  // their sum so far and the workgroups' arrivals: zero before and after
    int32_t* flag;    // [rows] 0: no entry, 1, 2: an id past the classes
    float* term;      // [rows] sum of q (log q - (x - base) / T)
    float* base;      // [rows] the largest of the entries' logits
    int32_t* ent_id;  // [rows][k] the class of its first entry, -1 at the others
    float* ent_q;     // the class's q
    float* ent_x;     // its logit
    float* row_loss;  // [rows]
    float* stat;      // [rows][splits][2]
    int64_t rows, classes;
    int32_t k, splits, slots;
    int64_t span;     // classes of a split, a multiple of 4
    float inv_t, temperature;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The rows' entries, a wavefront a row. Entries of one class meet in a hash table in LDS, of twice as many slots
// as entries at least: the first of them, by its place, takes the sum of their q in their order.
__global__ __launch_bounds__(1024) void k_distill_entries(DistillArg a) {
    extern __shared__ int32_t lds[];
    __shared__ int32_t red[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int32_t* key = lds + (size_t)wave * (3 * a.slots + 2 * a.k);  // a slot's class
    int32_t* first = key + a.slots;                                // its first entry
    int32_t* many = first + a.slots;                               // its entries
    int32_t* id = many + a.slots;
    float* q = reinterpret_cast<float*>(id + a.k);
    const float ninf = -__builtin_inff();
    int32_t kept = 0;
    for (int64_t r = (int64_t)blockIdx.x * waves + wave; r < a.rows; r += (int64_t)gridDim.x * waves) {
        const int64_t at = r * a.k;
        float best = ninf;
        bool any = false, bad = false;
        wave_sync();
        for (int i = lane; i < a.k; i += 64) {
            const int32_t c = a.ids[at + i];
            const float t = a.teacher[at + i];
            const bool in = c >= 0 && t != ninf;
            any = any || in;
            bad = bad || (in && c >= a.classes);
            id[i] = in ? c : -1;
            q[i] = t;
            if (in) best = __builtin_fmaxf(best, t);
        }
        any = __any(any);
        bad = __any(bad);
        kept += any;
        if (lane == 0) a.flag[r] = bad ? 2 : any ? 1 : 0;
        if (!any || bad) {
            for (int i = lane; i < a.k; i += 64) a.ent_id[at + i] = -1;
            if (lane == 0) a.term[r] = a.base[r] = 0.0f;
            continue;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) best = __builtin_fmaxf(best, __shfl_xor(best, o));
        for (int s = lane; s < a.slots; s += 64) {
            key[s] = -1;
            first[s] = 0x7fffffff;
            many[s] = 0;
        }
        float mass = 0.0f;
        for (int i = lane; i < a.k; i += 64) mass += id[i] >= 0 ? exp_neg((q[i] - best) * a.inv_t) : 0.0f;
        mass = wave_sum(mass);
        const float lm = mlog(mass), inv = 1.0f / mass;
        wave_sync();
        // sum q log q, and sum q (x - base) from the lane's own largest logit so far: the logits' common offset stays
        // out of the sums, where it would be rounded at its own size
        float term = 0.0f, part = 0.0f, weight = 0.0f, base = ninf;
        for (int i = lane; i < a.k; i += 64) {
            const int32_t c = id[i];
            if (c < 0) {
                q[i] = 0.0f;
                continue;
            }
            const float x = a.x[r * a.classes + c], u = (q[i] - best) * a.inv_t;
            const float v = exp_neg(u) * inv;
            a.ent_x[at + i] = x;
            q[i] = v;
            if (v != 0.0f) {  // 0 log 0 = 0
                term += v * (u - lm);
                if (x > base) {
                    part += weight > 0.0f ? weight * (base - x) : 0.0f;
                    base = x;
                }
                weight += v;
                part += v * (x == ninf ? ninf : x - base);
            }
            uint32_t s = ((uint32_t)c * 2654435761u) & (uint32_t)(a.slots - 1);
            for (;;) {  // ends: slots are more than entries
                const int32_t old = atomicCAS(&key[s], -1, c);
                if (old == -1 || old == c) break;
                s = (s + 1) & (uint32_t)(a.slots - 1);
            }
            atomicMin(&first[s], i);
            atomicAdd(&many[s], 1);
            a.ent_q[at + i] = __int_as_float((int)s);  // for the pass below
        }
        wave_sync();
        for (int i = lane; i < a.k; i += 64) {
            const int32_t c = id[i];
            bool mine = c >= 0;
            float v = q[i];
            if (mine) {
                const int s = __float_as_int(a.ent_q[at + i]);
                mine = first[s] == i;
                if (mine && many[s] > 1)
                    for (int j = i + 1; j < a.k; ++j) v += id[j] == c ? q[j] : 0.0f;
            }
            a.ent_id[at + i] = mine ? c : -1;
            a.ent_q[at + i] = v;
        }
        float top = base;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
        if (base > ninf && base < top) part += weight * (base - top);
        part = wave_sum(part);
        term = wave_sum(term) - part * a.inv_t;
        if (lane == 0) {
            a.term[r] = term;
            a.base[r] = top > ninf ? top : 0.0f;
        }
    }
    if (lane == 0) red[wave] = kept;
    __syncthreads();
    if (threadIdx.x == 0) {  // the last workgroup to arrive has the whole count
        uint32_t n = 0;
        for (int i = 0; i < waves; ++i) n += (uint32_t)red[i];
        uint32_t *sum = a.tickets, *arrived = a.tickets + kTicketStride;
        // the sum's answer is waited for before the arrival: an order for these two counters alone, where a
        // release would write the L2 back, once a workgroup
        const uint32_t before = __hip_atomic_fetch_add(sum, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::"v"(before) : "memory");
        if (__hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
            a.kept[0] = (int32_t)__hip_atomic_load(sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(sum, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// ug T / n over the n rows with an entry.
__device__ __forceinline__ float factor_of(const DistillArg& a) {
    return a.ug[0] * a.temperature / (float)(a.kept[0] > 0 ? a.kept[0] : 1);
}

// Running maximum and sum of exponentials, in base 2.
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
// Adds classes c0..c1 of a row, N loads in flight a thread.
template <int W>
__device__ __forceinline__ void run_row(Run& run, const float* x, int64_t c0, int64_t c1, float kf) {
    constexpr int N = 4;
    constexpr int64_t step = W * 64;
    const int64_t nq = (c1 - c0) >> 2;
    const float* p = x + c0;
    int64_t q = threadIdx.x;
    for (; q + (N - 1) * step < nq; q += N * step) {
        vf4 v[N];
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = *reinterpret_cast<const vf4u*>(p + 4 * (q + u * step));
#pragma unroll
        for (int u = 0; u < N; ++u) run_add(run, v[u], kf);
    }
    for (; q < nq; q += step) run_add(run, *reinterpret_cast<const vf4u*>(p + 4 * q), kf);
    if ((int64_t)threadIdx.x < (c1 - c0) - 4 * nq) {
        const float ninf = -__builtin_inff();
        run_add(run, vf4{p[4 * nq + threadIdx.x], ninf, ninf, ninf}, kf);
    }
}
template <int W>
__device__ __forceinline__ Run run_join(Run r, float kf, float* red) {
    const float top = block_max<W>(r.top, red);
    const float s = r.top == -__builtin_inff() ? r.sum : r.sum * __builtin_amdgcn_exp2f((r.top - top) * kf);
    return {top, block_sum<W>(s, red)};
}

// A logit's probability from the row's maximum and sum, p = e^((x - top) / T) / sum, or from its log-sum-exp,
// p = e^(x / T - lse) with x / T - lse rounded once, above 0 only by the log-sum-exp's rounding.
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
template <bool ACC>
__device__ __forceinline__ void grad_put(float* o, vf4 v) {
    if (ACC) {
        const vf4 old = ld_ntu(o);
        v = {old.x + v.x, old.y + v.y, old.z + v.z, old.w + v.w};
    }
    st_ntu(o, v);
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

// A row's loss before T^2 / n, its log-sum-exp, and the marks of a row without entries or with a bad id, from the
// largest logit and the sum of exponentials below it.
__device__ __forceinline__ void row_out(const DistillArg& a, int64_t r, int flag, float top, float sum) {
    if (threadIdx.x != 0) return;
    const float log_sum = mlog(sum);
    // the q sum to 1, so what the entries' sum left out comes in whole
    const float loss = a.term[r] + ((top - a.base[r]) * a.inv_t + log_sum);
    a.row_loss[r] = flag == 0 ? 0.0f : flag == 2 ? __builtin_nanf("") : loss;
    if (a.row_lse) a.row_lse[r] = flag == 0 ? 0.0f : flag == 2 ? __builtin_nanf("") : top * a.inv_t + log_sum;
}

// A thread's entries of classes c0..c1: with ACC what the gradient held there is read before the dense part
// writes over it; all are stored after it.
constexpr int entries_of(int W) { return kMaxK / (W * 64); }
template <int W, int N = entries_of(W)>
struct Mine {
    int32_t at[N];
    float old[N];
};
template <int W, bool ACC, int N>
__device__ __forceinline__ void entries_take(const DistillArg& a, int64_t r, int64_t c0, int64_t c1, Mine<W, N>& mine) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = threadIdx.x + u * W * 64;
        int32_t c = i < a.k ? a.ent_id[r * a.k + i] : -1;
        if (c < c0 || c >= c1) c = -1;
        mine.at[u] = c;
        mine.old[u] = ACC && c >= 0 ? a.grad[r * a.classes + c] : 0.0f;
    }
    if (ACC) __syncthreads();
}
template <int W, bool ACC, bool LSE, int N>
__device__ __forceinline__ void entries_put(const DistillArg& a, int64_t r, const Scale<LSE>& s, float c,
                                            const Mine<W, N>& mine) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < N; ++u) {
        if (mine.at[u] < 0) continue;
        const int64_t i = r * a.k + threadIdx.x + u * W * 64;
        const float v = (prob(s, a.ent_x[i]) - a.ent_q[i]) * c;
        a.grad[r * a.classes + mine.at[u]] = ACC ? mine.old[u] + v : v;
    }
}

// nq quads of a row's gradient, from the end, which was read last; N loads in flight a thread.
template <int W, bool ACC, bool LSE>
__device__ __forceinline__ void dense_grad(const float* x, float* g, int64_t nq, const Scale<LSE>& s, float c) {
    constexpr int N = 4;  // 8: 900 us where 4 take 871 over [4096, 131072]
    constexpr int64_t step = W * 64;
    int64_t q = nq - 1 - threadIdx.x;
    for (; q - (N - 1) * step >= 0; q -= N * step) {
        vf4 v[N];
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = ld_ntu(x + 4 * (q - u * step));
#pragma unroll
        for (int u = 0; u < N; ++u) grad_put<ACC>(g + 4 * (q - u * step), grad4(s, v[u], c));
    }
    for (; q >= 0; q -= step) grad_put<ACC>(g + 4 * q, grad4(s, ld_ntu(x + 4 * q), c));
}

// Classes c0..c1 of row r's gradient.
template <int W, bool ACC, bool LSE>
__device__ void row_grad(const DistillArg& a, int64_t r, int64_t c0, int64_t c1, const Scale<LSE>& s, float c) {
    const float* x = a.x + r * a.classes + c0;
    float* g = a.grad + r * a.classes + c0;
    const int tid = threadIdx.x;
    Mine<W> mine;
    entries_take<W, ACC>(a, r, c0, c1, mine);
    const int64_t nq = (c1 - c0) >> 2;
    dense_grad<W, ACC>(x, g, nq, s, c);
    if (tid < (int)((c1 - c0) & 3)) {
        const int64_t p = 4 * nq + tid;
        const float v = prob(s, x[p]) * c;
        g[p] = ACC ? g[p] + v : v;
    }
    entries_put<W, ACC>(a, r, s, c, mine);
}

// A whole row a workgroup, of any length: statistics, loss and, with GRAD, the gradient, for which the row is read
// again but for its last 32768 classes, which wait in LDS. That LDS also keeps a second workgroup off the CU:
// two rows a CU, 268 MB of [*, 131072] in use at a time, are more than the last cache holds.
template <int W, bool GRAD, bool ACC>
__global__ __launch_bounds__(W * 64) void k_distill_row(DistillArg a) {
    constexpr int NH = GRAD ? 8 : 1, step = W * 64;
    __shared__ float red[W];
    __shared__ vf4 held[GRAD ? NH * step : 1];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const int flag = a.flag[r];
    if (flag == 0) {
        row_out(a, r, 0, 0.0f, 1.0f);
        if (GRAD) row_zero<W, ACC>(a, r, 0, a.classes);
        return;
    }
    const float kf = a.inv_t * kLog2e;
    Run run = {-__builtin_inff(), 0.0f};
    const float* x = a.x + r * a.classes;
    const int64_t nq = a.classes >> 2, c_held = GRAD ? (nq - NH * step) * 4 : a.classes;
    run_row<W>(run, x, 0, c_held, kf);
    if (GRAD) {  // rows here are longer than what is held
        vf4 v[NH];
#pragma unroll
        for (int u = 0; u < NH; ++u) v[u] = ld_ntu(x + c_held + 4 * (u * step + tid));
#pragma unroll
        for (int u = 0; u < NH; ++u) {
            held[u * step + tid] = v[u];
            run_add(run, v[u], kf);
        }
        if (tid < (int)(a.classes & 3)) {
            const float ninf = -__builtin_inff();
            run_add(run, vf4{x[4 * nq + tid], ninf, ninf, ninf}, kf);
        }
    }
    run = run_join<W>(run, kf, red);
    row_out(a, r, flag, run.top, run.sum);
    if (GRAD) {  // an id past the classes: NaN all over the row
        const Scale<false> s = {kf, run.top, flag == 2 ? __builtin_nanf("") : 1.0f / run.sum};
        const float c = factor_of(a);
        float* g = a.grad + r * a.classes;
        Mine<W> mine;
        entries_take<W, ACC>(a, r, 0, a.classes, mine);
        if (tid < (int)(a.classes & 3)) {
            const int64_t p = 4 * nq + tid;
            const float v = prob(s, x[p]) * c;
            g[p] = ACC ? g[p] + v : v;
        }
#pragma unroll
        for (int u = 0; u < NH; ++u) grad_put<ACC>(g + c_held + 4 * (u * step + tid), grad4(s, held[u * step + tid], c));
        dense_grad<W, ACC>(x, g, c_held >> 2, s, c);
        entries_put<W, ACC>(a, r, s, c, mine);
    }
}

// The same with the row in registers, NQ quads a thread, and read once; a row's exponentials are taken once too.
// Up to 32768 classes two workgroups of 16 wavefronts share a CU at 64 registers, one loading while the other
// stores; at the 78 that the compiler took unbounded one workgroup ran alone (91 us against 69 over [1025,
// 30011]). Rows of up to 65536 have a CU to themselves: a workgroup ends with its stores under way and the next
// one's loads follow ([8192, 65536]: 787 us, 5.5 TB/s, against 846 read twice). Longer ones do not fit: 92
// registers of data leave too few of 128, and what spills costs more than reading twice (945 against 916 us
// over [4096, 131072]).
template <int W, int NQ, int NE, bool GRAD, bool ACC>
__global__ __launch_bounds__(W * 64, NQ > 8 ? 4 : 8) void k_distill_regs(DistillArg a) {
    __shared__ float red[W];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const float ninf = -__builtin_inff();
    const int flag = a.flag[r];
    if (flag == 0) {
        row_out(a, r, 0, 0.0f, 1.0f);
        if (GRAD) row_zero<W, ACC>(a, r, 0, a.classes);
        return;
    }
    const float* x = a.x + r * a.classes;
    const int nq = (int)(a.classes >> 2), tail = (int)(a.classes & 3);
    vf4 v[NQ];
    float top = ninf;
    auto max4 = [](vf4 q) { return __builtin_fmaxf(__builtin_fmaxf(q.x, q.y), __builtin_fmaxf(q.z, q.w)); };
    // Quad u of the thread: the row's address and u's in scalar registers, one offset in a vector register for
    // all of them (an address each is what spills). Bit 1 is the non-temporal path.
    const uint32_t off = (uint32_t)tid * 16;
    const auto row_of = [&](const float* p) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, nq * 16, 0x00020000);
    };
    const auto load = [&](__amdgpu_buffer_rsrc_t row, int u) {
        return __builtin_bit_cast(vf4, __builtin_amdgcn_raw_buffer_load_b128(row, off, u * W * 1024, 2));
    };
    const auto in_row = row_of(x);
    auto get = [&](int u) { return tid < nq - u * W * 64 ? load(in_row, u) : vf4{ninf, ninf, ninf, ninf}; };
#pragma unroll
    for (int u = 0; u < NQ; ++u) v[u] = get(u);
    float last = tid < tail ? x[4 * nq + tid] : ninf;
    const float kf = a.inv_t * kLog2e;
    top = __builtin_fmaxf(top, last);
#pragma unroll
    for (int u = 0; u < NQ; ++u) top = __builtin_fmaxf(top, max4(v[u]));
    top = block_max<W>(top, red);
    const float base = top == ninf ? 0.0f : top;
    const Scale<false> raw = {kf, base, 1.0f};
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        v[u] = grad4(raw, v[u], 1.0f);
        sum += (v[u].x + v[u].y) + (v[u].z + v[u].w);
    }
    last = prob(raw, last);
    sum = block_sum<W>(sum + last, red);
    row_out(a, r, flag, top, sum);
    if (GRAD) {
        const float c = factor_of(a);
        const Scale<false> s = {kf, base, flag == 2 ? __builtin_nanf("") : 1.0f / sum};
        Mine<W, NE> mine;
        entries_take<W, ACC>(a, r, 0, a.classes, mine);
        float* g = a.grad + r * a.classes;
        const auto out_row = row_of(g);
        auto put = [&](int u, vf4 e) {
            if (tid >= nq - u * W * 64) return;
            vf4 o = {e.x * s.inv * c, e.y * s.inv * c, e.z * s.inv * c, e.w * s.inv * c};
            if (ACC) {
                const vf4 old = load(out_row, u);
                o = {old.x + o.x, old.y + o.y, old.z + o.z, old.w + o.w};
            }
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), out_row, off, u * W * 1024, 2);
        };
#pragma unroll
        for (int u = 0; u < NQ; ++u) put(u, v[u]);
        if (tid < tail) {
            const float o = last * s.inv * c;
            g[4 * nq + tid] = ACC ? g[4 * nq + tid] + o : o;
        }
        entries_put<W, ACC>(a, r, s, c, mine);
    }
}

// A split of a row: its maximum and sum.
template <int W>
__global__ __launch_bounds__(W * 64) void k_distill_stat(DistillArg a) {
    __shared__ float red[W];
    const int64_t r = blockIdx.x / a.splits, sp = blockIdx.x % a.splits;
    if (a.flag[r] == 0) return;
    const int64_t c0 = sp * a.span, c1 = c0 + a.span < a.classes ? c0 + a.span : a.classes;
    const float kf = a.inv_t * kLog2e;
    Run run = {-__builtin_inff(), 0.0f};
    run_row<W>(run, a.x + r * a.classes, c0, c1, kf);
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

// The forward's log-sum-exp, rounded to fp32, scales a row's probabilities by its rounding: 2^-19 up to 64. Above,
// where an offset common to a row's logits is most of it, the backward alone takes the row's statistics again.
constexpr float kTrustedLse = 64.0f;

// A split of a row's gradient, from the forward's log-sum-exp (LOSS off) or the splits' statistics, of which the
// first split also writes the row's loss. GRAD off: the loss alone, a workgroup a row.
template <int W, bool LOSS, bool GRAD, bool ACC>
__global__ __launch_bounds__(W * 64) void k_distill_split(DistillArg a) {
    const int32_t per = GRAD ? a.splits : 1;
    const int64_t r = blockIdx.x / per, sp = blockIdx.x % per;
    const int64_t c0 = sp * a.span, c1 = c0 + a.span < a.classes ? c0 + a.span : a.classes;
    const int flag = a.flag[r];
    if (flag == 0) {
        if (LOSS && sp == 0) row_out(a, r, 0, 0.0f, 1.0f);
        if (GRAD) row_zero<W, ACC>(a, r, c0, c1);
        return;
    }
    if (LOSS) {
        const Run run = join_splits(a, r);
        if (sp == 0) row_out(a, r, flag, run.top, run.sum);
        if (GRAD) {
            const Scale<false> s = {a.inv_t * kLog2e, run.top, flag == 2 ? __builtin_nanf("") : 1.0f / run.sum};
            row_grad<W, ACC>(a, r, c0, c1, s, factor_of(a));
        }
    } else if (const float lse = a.lse_in[r]; __builtin_fabsf(lse) > kTrustedLse && flag != 2) {
        __shared__ float red[W];
        const float kf = a.inv_t * kLog2e;
        Run run = {-__builtin_inff(), 0.0f};
        run_row<W>(run, a.x + r * a.classes, 0, a.classes, kf);
        run = run_join<W>(run, kf, red);
        row_grad<W, ACC>(a, r, c0, c1, Scale<false>{kf, run.top, 1.0f / run.sum}, factor_of(a));
    } else {
        const Scale<true> s = {a.inv_t, flag == 2 ? __builtin_nanf("") : lse, 1.0f};
        row_grad<W, ACC>(a, r, c0, c1, s, factor_of(a));
    }
}

// loss = T^2 / n sum of the rows' losses, in a fixed order.
__global__ __launch_bounds__(1024) void k_distill_loss(DistillArg a, float* loss) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 4
    for (int64_t n = threadIdx.x; n < a.rows; n += 1024) s += (double)a.row_loss[n];
    s = block_sum<16>(s, red);
    const double n = a.kept[0] > 0 ? a.kept[0] : 1;
    if (threadIdx.x == 0) loss[0] = (float)(s * ((double)a.temperature * a.temperature) / n);
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
    a.slots = 64;
    while (a.slots < 2 * a.k) a.slots *= 2;
    // wavefronts of a workgroup of k_distill_entries by what LDS holds: 16 up to 128 entries a row, 2 at 1024
    const size_t row_lds = (3 * (size_t)a.slots + 2 * (size_t)a.k) * sizeof(int32_t);
    int waves = 16;
    while (waves > 1 && waves * row_lds > 65536) waves /= 2;
    while (waves > 4 && d.rows < (int64_t)waves * ctx().num_cus) waves /= 2;
    const int64_t blocks = (d.rows + waves - 1) / waves;
    const int64_t parts = blocks < kEntryBlocks ? blocks : kEntryBlocks;
    const size_t rows_b = ((size_t)d.rows * 4 + 255) & ~(size_t)255, ent_b = ((size_t)d.rows * a.k * 4 + 255) & ~(size_t)255;
    char* base = nullptr;
    MH_TRY(tickets(2 * kTicketStride, &a.tickets));
    MH_TRY(scratch(256 + 4 * rows_b + 3 * ent_b + (size_t)d.rows * a.splits * 8, reinterpret_cast<void**>(&base)));
    auto take = [&base](size_t bytes) {
        char* p = base;
        base += bytes;
        return p;
    };
    a.kept = reinterpret_cast<int32_t*>(take(256));
    a.flag = reinterpret_cast<int32_t*>(take(rows_b));
    a.term = reinterpret_cast<float*>(take(rows_b));
    a.base = reinterpret_cast<float*>(take(rows_b));
    a.row_loss = reinterpret_cast<float*>(take(rows_b));
    a.ent_id = reinterpret_cast<int32_t*>(take(ent_b));
    a.ent_q = reinterpret_cast<float*>(take(ent_b));
    a.ent_x = reinterpret_cast<float*>(take(ent_b));
    a.stat = reinterpret_cast<float*>(base);
    hipStream_t st = ctx().stream;
    hipLaunchKernelGGL(k_distill_entries, dim3((unsigned)parts), dim3(waves * 64), waves * row_lds, st, a);
    constexpr int W = 16;
    const dim3 rows((unsigned)d.rows), all((unsigned)(d.rows * a.splits)), t(W * 64);
    const bool grad = d.grad != nullptr;
    if (d.lse_in) {
        if (d.accumulate) hipLaunchKernelGGL((k_distill_split<W, false, true, true>), all, t, 0, st, a);
        else hipLaunchKernelGGL((k_distill_split<W, false, true, false>), all, t, 0, st, a);
    } else if (a.splits == 1 && a.classes <= kHeld && (grad || a.classes <= 32768)) {
#define MH_REGS(WW, NQ, NE)                                                                                                \
    do {                                                                                                              \
        const dim3 tt(WW * 64);                                                                                       \
        if (!grad) hipLaunchKernelGGL((k_distill_regs<WW, NQ, NE, false, false>), rows, tt, 0, st, a);                    \
        else if (d.accumulate) hipLaunchKernelGGL((k_distill_regs<WW, NQ, NE, true, true>), rows, tt, 0, st, a);          \
        else hipLaunchKernelGGL((k_distill_regs<WW, NQ, NE, true, false>), rows, tt, 0, st, a);                           \
    } while (0)
        // short rows with few entries: a wavefront each, with no barrier
        if (a.classes <= 1024 && a.k <= 128) MH_REGS(1, 4, 2);
        else if (a.classes <= 2048) MH_REGS(4, 2, 4);
        else if (a.classes <= 4096) MH_REGS(4, 4, 4);
        else if (a.classes <= 8192) MH_REGS(4, 8, 4);
        else if (a.classes <= 16384) MH_REGS(8, 8, 2);
        else if (a.classes <= 32768) MH_REGS(16, 8, 1);
        else MH_REGS(16, 16, 1);
#undef MH_REGS
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
        hipLaunchKernelGGL(k_distill_loss, dim3(1), dim3(1024), 0, st, a, d.loss);
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
