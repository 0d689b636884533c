// mh_group_router.hip -- routing to experts by sigmoid or softmax scores, with a bias for balance, groups of experts and
// a scale; the gradient of the logits; and the bias' step towards balance.
//
//   s = sigmoid(x) | softmax(x);  b = s + bias;  a group's score = the sum of its one or two largest b;
//   chosen = the k largest b in the keep_groups best groups;  weights = scale s_chosen, or scale q with q = s / sum s
//   With g the weights' gradient (0 where not chosen):
//     sigmoid:  grad_i = scale s_i (1 - s_i) g_i            normalised: scale q_i (1 - s_i) (g_i - sum g q)
//     softmax:  grad_j = scale p_j (g_j - sum g p)          normalised: scale q_i (g_i - sum g q)
//
// Scores decide a choice after a bias was added to them, so logits do not: experts whose biased scores agree to fp32 are
// not rare over a long batch, and which of them is chosen shows. What is compared is therefore meant in 64 bits.
// Choices are made in fp32 first, 8 at a time by sorted lists of the row, with a bound on its error; a row whose choice,
// or whose choice of groups, turns on less than twice that (one in a few hundred) is listed, and a second kernel chooses
// for it in 64 bits, a wavefront a row. That kernel alone takes short batches, whose rows it holds all at once. Weights
// are made in 64 bits and rounded once, by one formula in both, for a bias may choose among scores that fp32 does not hold; so are the
// gradients, but for the exponentials of a softmax of which every expert has one, to an ulp or so of fp32.
//
// L lanes hold a row in registers, V elements a lane in quads (element 4 (i L + lane) + c). Over [131072, 256], top 8 of 4 of
// 8 groups, the forward takes 92 us, where its read alone takes 24: 1200 vector instructions for a wavefront's 4 rows
// (scores, the groups' best, the sorted list, the check) fill three quarters of it. The listed rows take 11 us more, each k
// reductions that wait for each other, the counts 6, and the backward, which writes 134 MB and gathers the chosen's logits, 39 (with its
// scores made twice, in fp32, 46).
#include "mh_internal.h"
#include "mh_lanes.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kMaxGroups = 64;
constexpr int kRThreads = 256;
// Workgroups of a forward at most, and rows of its partial counts: its call over [131072, 256] 104 us, with 512 of them 116, 768 104,
// 1024 111, 1536 110; over [2^20, 16] 62.5, 83.5, 70.5, 62, 67.
constexpr int kRBlocks = 2048;
// Workgroups for listed rows: where every row is tied, a router of zeros, [131072, 256] takes 0.94 ms with 512, 2.5 with 128 and 0.76
// with 1024, which add 1 to 1.5 us to any call.
constexpr int64_t kRExactBlocks = 512;
// Workgroups that add up their counts by themselves: over 16 experts 64 rows (16 workgroups) 6.8 us instead of 8.5, 500 rows (125) 12.0
// instead of 8.6; over 256 experts 128 rows (32) 11.8 and 11.5, 500 rows 16.4 and 12.4.
constexpr int64_t kRArrivals = 32;
// Batches of up to this many rows go by wavefronts alone: over 256 experts 2048 rows take 13 us, by lists first 21; 4096 16.6 and 21,
// 8192 27 and 23, 131072 299 and 104.
constexpr int64_t kRExactRows = 2048;

struct GroupArg {
    const float* x;
    const float* bias;    // or null
    const int32_t* keep;  // or null: every row
    int64_t rows;
    int32_t experts, k;
    int32_t groups, each, open, best;  // each: experts of a group
    int32_t parts;                     // lanes that share a group, a power of two
    int32_t wave_parts;                // the same of a wavefront
    int32_t sigmoid, normalise, accumulate;
    float scale;
    FastDiv by_each;
    // forward
    float* weights;
    int32_t* chosen;
    int32_t* part_c;  // [blocks][experts]
    int32_t* todo;    // rows listed for the second kernel, or null: every row
    uint32_t* ntodo;
    uint32_t* arrived;  // of the second kernel's workgroups, or null: another kernel adds up
    int32_t* counts;
    // backward
    float* grad;
    const float* gw;
    const int32_t* sel;
};

// As group_red and others, of values of 64 bits.
template <int STEP>
__device__ __forceinline__ uint64_t other64(uint64_t v) {
    return (uint64_t)(uint32_t)other_lane<STEP>((int)(v >> 32)) << 32 | (uint32_t)other_lane<STEP>((int)v);
}
template <int L, int STEP = 1, typename T, typename Op>
__device__ __forceinline__ T group_red64(T v, Op op) {
    if constexpr (STEP < L)
        return group_red64<L, 2 * STEP>(op(v, __builtin_bit_cast(T, other64<STEP>(__builtin_bit_cast(uint64_t, v)))), op);
    return v;
}
template <int L>
__device__ __forceinline__ double group_sum64(double v) { return group_red64<L>(v, [](double p, double q) { return p + q; }); }
template <int L>
__device__ __forceinline__ float group_min(float v) { return -group_max<L>(-v); }

__device__ __forceinline__ double sigmoid64(float x) {
    const double e = exp64(-__builtin_fabs((double)x));
    return (x < 0.0f ? e : 1.0) / (1.0 + e);
}

// A constant in scalar registers, made where it stands: a loop's constants in vector registers cost a row's occupancy.
__device__ __forceinline__ double scalar(double c) {
    asm volatile("" : "+s"(c));
    return c;
}
// e^x for x <= 0 to 2^-31 of itself: what a score that is rounded to fp32 needs of 64 bits.
__device__ __forceinline__ double exp_short(double x) {
    x = x < -1000.0 ? -1000.0 : x;
    const double n = __builtin_rint(x * scalar(1.4426950408889634074));
    const double r = __builtin_fma(n, scalar(-0.69314718055994530942), x);
    double p = __builtin_fma(scalar(1.0 / 40320.0), r, scalar(1.0 / 5040.0));
    p = __builtin_fma(p, r, scalar(1.0 / 720.0));
    p = __builtin_fma(p, r, scalar(1.0 / 120.0));
    p = __builtin_fma(p, r, scalar(1.0 / 24.0));
    p = __builtin_fma(p, r, scalar(1.0 / 6.0));
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// e^x for x <= 0 to the exponential unit's own ulp and a quarter more of fp32: the exponent in 64 bits, its whole part taken off by a
// sum that has room for no other.
__device__ __forceinline__ float exp_rounded(double x) {
    x = x < -1000.0 ? -1000.0 : x;  // a NaN stays one
    const double t = x * scalar(1.4426950408889634074), whole = t + scalar(6755399441055744.0);
    return __builtin_ldexpf(__builtin_amdgcn_exp2f((float)(t - (whole - scalar(6755399441055744.0)))), __double2loint(whole));
}
// 1 / x of a positive normal x, to 2^-48 or so: a step of Newton's on the unit's own.
__device__ __forceinline__ double inverse(double x) {
    const double y = __builtin_amdgcn_rcp(x);
    return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}
// A weight's score; `top` and `by` are a softmax's largest logit and 1 / the sum of its exponentials.
__device__ __forceinline__ double weight_score(bool sigmoid, float v, float top, double by) {
    const double e = exp_short(sigmoid ? -__builtin_fabs((double)v) : (double)v - (double)top);
    return sigmoid ? (v < 0.0f ? e : 1.0) * inverse(1.0 + e) : e * by;
}
// A double as an integer of the same order; NaN below every number, -0 as +0; below them what may not be chosen.
constexpr int64_t kNever = INT64_MIN;
__device__ __forceinline__ int64_t sort_key64(double v) {
    const int64_t b = __double_as_longlong(v + 0.0);
    return v != v ? kNever + 1 : (b < 0 ? b ^ 0x7fffffffffffffffll : b);
}

// Whether the group of score c at index j comes before that of d at o: the larger, ties to the lower index, a NaN last.
template <typename T>
__device__ __forceinline__ bool before(T c, int j, T d, int o) {
    return c > d || (d != d && c == c) || (j < o && (c == d || (c != c && d != d)));
}

// The largest of a wavefront's, each lane's with the lanes' before it, then rows of 16 lanes and halves.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t larger(int64_t v) {
    const int lo = (int)v, hi = (int)(v >> 32);
    const int64_t w = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(hi, hi, CTRL, ROWS, 0xf, false) << 32 |
                                (uint32_t)__builtin_amdgcn_update_dpp(lo, lo, CTRL, ROWS, 0xf, false));
    return v > w ? v : w;
}
__device__ __forceinline__ int64_t wave_largest(int64_t v) {
    v = larger<0x111, 0xf>(v);
    v = larger<0x112, 0xf>(v);
    v = larger<0x114, 0xf>(v);
    v = larger<0x118, 0xf>(v);
    v = larger<0x142, 0xa>(v);
    v = larger<0x143, 0xc>(v);
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, 63));
}

// The choice of one row in 64 bits, by a wavefront: element 64 i + lane in the lane's i-th place. `row` holds C * 64
// doubles, `score` one a group. The experts go to `ids`, best first.
template <int C>
__device__ __forceinline__ void choose_exact(const GroupArg& a, const float* x, double* row, double* score, int32_t* ids, float& top,
                                             double& by) {
    const int lane = threadIdx.x & 63;
    double b[C];
    float plus[C];  // the bias, on its way with the logits
    top = -__builtin_inff();
    by = 0.0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int e = 64 * i + lane;
        b[i] = (double)(e < a.experts ? x[e] : -__builtin_inff());
        plus[i] = a.bias && e < a.experts ? a.bias[e] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) top = __builtin_fmaxf(top, (float)b[i]);
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < C; ++i) b[i] = sigmoid64((float)b[i]);
    } else {
        top = group_max<64>(top);
        double sum = 0.0, rough = 0.0;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            rough += exp_short(b[i] - (double)top);
            b[i] = exp64(b[i] - (double)top);
            sum += b[i];
        }
        sum = group_sum64<64>(sum);
        by = inverse(group_sum64<64>(rough));
#pragma unroll
        for (int i = 0; i < C; ++i) b[i] = b[i] / sum;
    }
    int64_t key[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int e = 64 * i + lane;
        if (a.bias) b[i] += (double)plus[i];
        key[i] = e < a.experts ? sort_key64(b[i]) : kNever;
    }
    if (a.groups > 1) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < C; ++i) row[64 * i + lane] = b[i];
        wave_sync();
        // the wavefront's lanes in as many parts of a group as there are lanes for
        const int parts = a.wave_parts, part = lane & (parts - 1), j = lane >> __builtin_ctz(parts);
        double first = -__builtin_inf(), second = first;
        int numbers = 0;  // a NaN comes behind them
        if (j < a.groups) {
            const double* v = row + j * a.each;
#pragma unroll 4
            for (int e = part; e < a.each; e += parts) {
                const double c = v[e], d = c == c ? c : -__builtin_inf();
                numbers += c == c;
                second = max_d(second, min_d(first, d));
                first = max_d(first, d);
            }
        }
        for (int o = 1; o < parts; o *= 2) {
            const double f = __shfl_xor(first, o), t = __shfl_xor(second, o);
            second = max_d(min_d(first, f), max_d(second, t));
            first = max_d(first, f);
            numbers += __shfl_xor(numbers, o);
        }
        if (numbers < 2) second = __builtin_nan("");
        if (numbers < 1) first = second;
        if (part == 0 && j < a.groups) score[j] = a.best == 2 && a.each > 1 ? first + second : first;
        wave_sync();
        bool open = false;
        if (lane < a.groups) {
            int n = 0;
#pragma unroll 8
            for (int o = 0; o < a.groups; ++o) n += before(score[o], o, score[lane], lane);
            open = n < a.open;
        }
        const uint64_t mask = __ballot(open);
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (!(mask >> (fdiv((uint32_t)(64 * i + lane), a.by_each) & 63) & 1)) key[i] = kNever;
    }
    for (int t = 0; t < a.k; ++t) {
        int64_t own = key[0];
        int in = 0;  // the lane's place of it, the first
#pragma unroll
        for (int i = 1; i < C; ++i) {
            in = key[i] > own ? i : in;
            own = key[i] > own ? key[i] : own;
        }
        const uint64_t has = __ballot(own == wave_largest(own));
        int at = __builtin_ctzll(has);
        at += 64 * __builtin_amdgcn_readlane(in, at);
        if (has & (has - 1)) {  // ties: the lowest index is that of the lowest place
            at = has >> lane & 1 ? 64 * in + lane : C * 64;
            at = group_red<64>(at, [](int p, int q) { return p < q ? p : q; });
            at = __builtin_amdgcn_readfirstlane(at);
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at == 64 * i + lane) key[i] = kNever;
        if (lane == 0) ids[t] = at;
    }
}

// A chosen row's results by L lanes, of which this is number l: its choices lie in `pick`. Their scores are 64-bit until the weight
// is rounded: a bias may choose among scores that fp32 does not hold.
template <int L>
__device__ __forceinline__ void put_choice(const GroupArg& a, const int32_t* pick, const float* x, int64_t r, int l, bool in, bool keep,
                                           float top, double by, int32_t* cnt) {
    double total = 0.0, s = 0.0;
    for (int t = l; keep && in && t < a.k; t += L) {
        s = weight_score(a.sigmoid != 0, x[pick[t]], top, by);
        total += s;
    }
    const double times = (double)a.scale * (a.normalise ? inverse(group_sum64<L>(total)) : 1.0);
    for (int t = l; in && t < a.k; t += L) {
        const int32_t id = keep ? pick[t] : 0;  // nothing is known of a padding row's
        if (L < kMaxChosen && a.k > L && keep) s = weight_score(a.sigmoid != 0, x[id], top, by);
        a.chosen[r * a.k + t] = keep ? id : -1;
        a.weights[r * a.k + t] = keep ? (float)(s * times) : 0.0f;
        if (keep) atomicAdd(&cnt[id], 1);
    }
}

// load_row, of rows that fill their lanes without a branch.
template <int L, int V>
__device__ __forceinline__ void load_next(const float* row, int E, int l, float* v) {
    if (E == L * V) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const vf4 q = *reinterpret_cast<const vf4u*>(row + 4 * (i * L + l));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = q[j];
        }
    } else {
        load_row<L, V>(row, E, l, v);
    }
}

template <int L, int V, bool SIGMOID>
__global__ __launch_bounds__(kRThreads, V == 16 ? 3 : 4) void k_group_router_fwd(GroupArg a) {
    constexpr int G = kRThreads / L;  // rows in flight in a workgroup
    constexpr int N = L * V < kMaxGroups ? L * V : kMaxGroups;
    __shared__ int32_t cnt[L * V];
    constexpr int K = L * V < kList ? kList : L * V < kMaxChosen ? L * V : kMaxChosen;
    __shared__ int32_t pick[G][K];
    __shared__ __attribute__((aligned(16))) float row[G][L * V], bias[L * V];
    __shared__ float of_group[G][N];
    const int tid = threadIdx.x, l = tid % L, g = tid / L;
    for (int e = tid; e < L * V; e += kRThreads) cnt[e] = 0;
    // the bias; past the experts minus infinity
    float most = 0.0f;
    for (int e = tid; e < L * V; e += kRThreads) bias[e] = e < a.experts ? (a.bias ? a.bias[e] : 0.0f) : -__builtin_inff();
    __syncthreads();
    for (int e = l; e < a.experts; e += L) {
        const float m = __builtin_fabsf(bias[e]);
        most = m < __builtin_inff() ? __builtin_fmaxf(most, m) : most;
    }
    most = group_max<L>(most);
    uint32_t gid[V / 4];  // the elements' groups, a byte each
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        gid[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) gid[i] |= (fdiv((uint32_t)(4 * (i * L + l) + j), a.by_each) & 63) << (8 * j);
    }
    const int64_t stride = (int64_t)gridDim.x * G;
    float next[V];
    {
        const int64_t n = (int64_t)blockIdx.x * G + g;
        load_next<L, V>(a.x + (n < a.rows ? n : 0) * a.experts, a.experts, l, next);
    }
    // every wavefront walks whole rounds, so that its lanes reduce together
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const int64_t r = r0 + g;
        const bool in = r < a.rows;
        const bool keep = in && (!a.keep || a.keep[r] != 0);
        const float* x = a.x + (in ? r : r0) * a.experts;
        float b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = next[i];
        {  // a round ahead
            const int64_t n = r + stride < a.rows ? r + stride : r0;
            load_next<L, V>(a.x + n * a.experts, a.experts, l, next);
        }
        // scores to within 2^-22 (of the largest, where softmax); past the experts the bias is minus infinity
        float unit = 1.0f, top = 0.0f;
        double by = 0.0;
        if (SIGMOID) {
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(b[i] * -kLog2e));
        } else {
            top = b[0];
#pragma unroll
            for (int i = 1; i < V; ++i) top = __builtin_fmaxf(top, b[i]);
            top = group_max<L>(top);
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double e = exp_short((double)b[i] - (double)top);
                sum += e;
                b[i] = (float)e;
            }
            by = inverse(group_sum64<L>(sum));
            unit = (float)by;
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] *= unit;
        }
        // with the bias, to LDS as well
        bool unsure = false;
        wave_sync();
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const vf4 q = *reinterpret_cast<const vf4*>(&bias[4 * (i * L + l)]) + vf4{b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]};
            *reinterpret_cast<vf4*>(&row[g][4 * (i * L + l)]) = q;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[4 * i + j] = q[j];
                unsure |= !(q[j] < __builtin_inff());
            }
        }
        wave_sync();
        // twice what two of them are off by together
        const float tell = unit * 0x1p-20f + most * 0x1p-22f;
        uint64_t mask = ~(uint64_t)0;
        if (a.groups > 1) {
            // a lane's share of a group, 4 experts at a time where they divide so
            const int part = l & (a.parts - 1);
            for (int j = l / a.parts; j < a.groups; j += L / a.parts) {
                const float* v = row[g] + j * a.each;
                float first = -__builtin_inff(), second = first;
                auto take = [&](float c) {
                    second = __builtin_amdgcn_fmed3f(first, second, c);
                    first = __builtin_fmaxf(first, c);
                };
                if ((a.each & 3) == 0) {
#pragma unroll 4
                    for (int e = 4 * part; e < a.each; e += 4 * a.parts) {
                        const vf4 q = *reinterpret_cast<const vf4*>(v + e);
                        take(q.x);
                        take(q.y);
                        take(q.z);
                        take(q.w);
                    }
                } else {
#pragma unroll 4
                    for (int e = part; e < a.each; e += a.parts) take(v[e]);
                }
                for (int o = 1; o < a.parts; o *= 2) {
                    const float f = __shfl_xor(first, o), t = __shfl_xor(second, o);
                    second = __builtin_fmaxf(__builtin_fminf(first, f), __builtin_fmaxf(second, t));
                    first = __builtin_fmaxf(first, f);
                }
                if (part == 0) of_group[g][j] = a.best == 2 && a.each > 1 ? first + second : first;
            }
            wave_sync();
            int lo = 0, hi = 0;  // halves of the open groups' bits
            float least = __builtin_inff(), best = -__builtin_inff();
            for (int j = l; j < a.groups; j += L) {
                const float c = of_group[g][j];
                int n = 0;
#pragma unroll 8
                for (int o = 0; o < a.groups; ++o) n += before(of_group[g][o], o, c, j);
                const bool open = n < a.open;
                least = open ? __builtin_fminf(least, c) : least;
                best = open ? best : __builtin_fmaxf(best, c);
                if (open) (j < 32 ? lo : hi) |= 1 << (j & 31);
            }
            lo = group_red<L>(lo, [](int p, int q) { return p | q; });
            hi = group_red<L>(hi, [](int p, int q) { return p | q; });
            mask = (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
            unsure |= !(group_min<L>(least) - group_max<L>(best) > 2.0f * tell);
        }
        if (a.groups > 1) {
            // a lane's elements in open groups, a bit each; a quad is of one group where they divide so
            int bits = 0;
            if ((a.each & 3) == 0) {
#pragma unroll
                for (int i = 0; i < V / 4; ++i) bits |= (mask >> (gid[i] & 255) & 1) != 0 ? 15 << (4 * i) : 0;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) bits |= (int)(mask >> (gid[i / 4] >> (8 * (i & 3)) & 255) & 1) << i;
            }
            wave_sync();
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                vf4 q;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int all = (bits << (31 - 4 * i - j)) >> 31, none = __float_as_int(-__builtin_inff());
                    b[4 * i + j] = q[j] = __int_as_float((__float_as_int(b[4 * i + j]) & all) | (none & ~all));
                }
                *reinterpret_cast<vf4*>(&row[g][4 * (i * L + l)]) = q;
            }
            wave_sync();
        }
        // 8 choices at a time, of what lies below the last. A double that begins with a float's bits has its order; the rest
        // holds the expert, whose order does not matter: a row with two of a value among its choices is not decided here.
        // Those chosen have to differ by more than what they are off by, and the last of them from the rest; what is closed or
        // past the experts is minus infinity, which none of them may be.
        float last = __builtin_inff(), gap = __builtin_inff(), was = __builtin_inff();
        for (int t0 = 0; t0 < a.k; t0 += kList) {
            double d[V < 8 ? 8 : V];
#pragma unroll
            for (int i = 0; i < (V < 8 ? 2 : V / 4); ++i) {
                vf4 q = vf4{0.0f, 0.0f, 0.0f, 0.0f};
                if (i < V / 4) q = *reinterpret_cast<const vf4*>(&row[g][4 * ((i < V / 4 ? i : 0) * L + l)]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    d[4 * i + j] = __hiloint2double(__float_as_int(i < V / 4 && q[j] < last ? q[j] : -__builtin_inff()), 4 * (i * L + l) + j);
            }
            list_rows<L, V>(d);
#pragma unroll
            for (int t = 0; t < kList; ++t) {
                const float v = __int_as_float(__double2hiint(d[t]));
                if (t0 + t < a.k) {
                    if (t0 + t > 0) gap = __builtin_fminf(gap, was - v);
                    last = was = v;
                    if (l == 0) pick[g][t0 + t] = __double2loint(d[t]);
                }
            }
        }
        int near = 0;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const vf4 q = *reinterpret_cast<const vf4*>(&row[g][4 * (i * L + l)]);
#pragma unroll
            for (int j = 0; j < 4; ++j) near += q[j] >= last - tell;
        }
        near = group_red<L>(near, [](int p, int q) { return p + q; });
        unsure = group_red<L>((int)unsure, [](int p, int q) { return p | q; }) != 0;
        unsure |= !(gap > tell) || near != a.k || !(last > -__builtin_inff());
        unsure &= keep;  // a padding row has nothing to choose
        if (l == 0 && unsure) {
            const uint32_t at = atomicAdd(a.ntodo, 1u);
            if (at < (uint64_t)a.rows) a.todo[at] = (int32_t)r;
        }
        wave_sync();
        put_choice<L>(a, pick[g], x, r, l, in && !unsure, keep, top, by, cnt);
    }
    __syncthreads();
    for (int e = tid; e < a.experts; e += kRThreads) a.part_c[(int64_t)blockIdx.x * a.experts + e] = cnt[e];
}

// Rows in 64 bits, a wavefront each: all of them, or those listed.
template <int C>
__global__ __launch_bounds__(kRThreads) void k_group_router_exact(GroupArg a) {
    __shared__ int32_t cnt[C * 64];
    __shared__ int32_t pick[kRThreads / 64][kMaxChosen];
    __shared__ double wide[kRThreads / 64][C * 64 + kMaxGroups];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    for (int e = tid; e < C * 64; e += kRThreads) cnt[e] = 0;
    __syncthreads();
    const int64_t listed = a.todo ? (int64_t)a.ntodo[0] : a.rows, rows = listed < a.rows ? listed : a.rows;
    for (int64_t i = (int64_t)blockIdx.x * (kRThreads / 64) + wave; i < rows; i += (int64_t)gridDim.x * (kRThreads / 64)) {
        const int64_t r = a.todo ? (int64_t)a.todo[i] : i;
        const bool keep = !a.keep || a.keep[r] != 0;
        const float* x = a.x + r * a.experts;
        float top = 0.0f;
        double by = 0.0;
        wave_sync();
        if (keep) choose_exact<C>(a, x, wide[wave], wide[wave] + C * 64, pick[wave], top, by);
        wave_sync();
        put_choice<64>(a, pick[wave], x, r, tid & 63, true, keep, top, by, cnt);
    }
    __syncthreads();
    if (!a.arrived) {
        for (int e = tid; e < a.experts; e += kRThreads) a.part_c[(int64_t)blockIdx.x * a.experts + e] = cnt[e];
        return;
    }
    // few workgroups: the last to arrive adds up. The stores are waited for, rather than the L2 written back.
    __shared__ int last;
    for (int e = tid; e < a.experts; e += kRThreads)
        __hip_atomic_store(&a.part_c[(int64_t)blockIdx.x * a.experts + e], cnt[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    for (int e = tid; e < a.experts; e += kRThreads) {
        int32_t s = 0;
#pragma unroll 8
        for (unsigned b = 0; b < gridDim.x; ++b)
            s += __hip_atomic_load(&a.part_c[(int64_t)b * a.experts + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.counts[e] = s;
    }
    if (tid == 0) __hip_atomic_store(a.arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The counts from the workgroups' partials: 32 experts and 32 shares of the partials a workgroup. The list of rows is
// done with.
__global__ __launch_bounds__(1024) void k_group_router_counts(const int32_t* part, int32_t blocks, int32_t experts, int32_t* counts,
                                                              uint32_t* ntodo) {
    __shared__ int32_t buf[1024];
    const int e = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
    int32_t s = 0;
    if (e < experts) {
#pragma unroll 8
        for (int b = share; b < blocks; b += 32) s += part[(int64_t)b * experts + e];
    }
    if (ntodo && blockIdx.x == 0 && threadIdx.x == 0) ntodo[0] = 0;
    buf[threadIdx.x] = s;
    __syncthreads();
    if (share != 0 || e >= experts) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) s += buf[32 * i + (threadIdx.x & 31)];
    counts[e] = s;
}

// What the chosen get goes to a row of LDS at their experts; a softmax's every expert gets its own part.
template <int L, int V>
__global__ __launch_bounds__(kRThreads) void k_group_router_bwd(GroupArg a) {
    constexpr int G = kRThreads / L;
    __shared__ __attribute__((aligned(16))) float mark[G][L * V];
    const int l = threadIdx.x % L, g = threadIdx.x / L;
    const int64_t stride = (int64_t)gridDim.x * G;
    const bool whole = !a.sigmoid && !a.normalise;  // every expert has a gradient
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += stride) {
        const int64_t r = r0 + g;
        const bool in = r < a.rows;
        const bool keep = in && (!a.keep || a.keep[r] != 0);
        const int64_t at = (in ? r : r0) * a.experts;
        // Scores and their sums are 64-bit, as the forward's: the chosen's may be less than fp32 holds, and a difference of gradients
        // keeps the bits that it leaves.
        float v[V], top = 0.0f;
        double by = 1.0;
        if (whole) {
            load_row<L, V>(a.x + at, a.experts, l, v);
            top = v[0];
#pragma unroll
            for (int i = 1; i < V; ++i) top = __builtin_fmaxf(top, v[i]);
            top = group_max<L>(top);
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = exp_rounded((double)v[i] - (double)top);
                sum += (double)v[i];
            }
            by = inverse(group_sum64<L>(sum));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = 0.0f;
            if (!a.sigmoid) {  // the chosen's maximum
                top = -__builtin_inff();
                if (keep)
                    for (int c = l; c < a.k; c += L) {
                        const int32_t id = a.sel[r * a.k + c];
                        if (id >= 0 && id < a.experts) top = __builtin_fmaxf(top, a.x[at + id]);
                    }
                top = group_max<L>(top);
            }
        }
        // an entry's expert, or -1; its score or exponential, what of a sigmoid its derivative leaves, and the weight's gradient
        double score = 0.0, rest = 1.0, gr = 0.0;
        auto entry = [&](int c) {
            const int32_t id = a.sel[r * a.k + c];
            if (id < 0 || id >= a.experts) return -1;
            const float x = a.x[at + id];
            gr = (double)a.gw[r * a.k + c];
            const double e = exp_short(a.sigmoid ? -__builtin_fabs((double)x) : (double)x - (double)top);
            score = e;
            if (a.sigmoid) {
                const double d = inverse(1.0 + e);
                rest = x < 0.0f ? d : e * d;
                score = x < 0.0f ? e * d : d;
            }
            return id;
        };
        int32_t id = -1;
        double all = 0.0, inner = 0.0;
        if (keep)
            for (int c = l; c < a.k; c += L) {
                id = entry(c);
                if (id < 0) continue;
                all += score;
                inner += score * gr;
            }
        all = group_sum64<L>(all);
        inner = group_sum64<L>(inner);
        if (a.normalise) by = inverse(all);
        inner *= by;
        by *= (double)a.scale;
        wave_sync();
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            vf4 q = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            *reinterpret_cast<vf4*>(&mark[g][4 * (i * L + l)]) = whole ? q * (float)(by * -inner) : q;
        }
        wave_sync();
        if (keep)
            for (int c = l; c < a.k; c += L) {
                if (L < kMaxChosen && a.k > L) id = entry(c);
                if (id >= 0) mark[g][id] = (float)(score * by * rest * (a.normalise || whole ? gr - inner : gr));
            }
        wave_sync();
        if (!in || (!keep && a.accumulate)) continue;  // a padding row: as it was, or zero
        float* o = a.grad + at;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const int c = 4 * (i * L + l);
            vf4 q = *reinterpret_cast<const vf4*>(&mark[g][c]);
            q = keep ? q : vf4{0.0f, 0.0f, 0.0f, 0.0f};
            if (c + 3 < a.experts) {
                if (a.accumulate) q = q + ld_ntu(o + c);
                st_ntu(o + c, q);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < a.experts) o[c + j] = a.accumulate ? o[c + j] + q[j] : q[j];
            }
        }
    }
}

__global__ __launch_bounds__(kRThreads) void k_router_bias(float* bias, const int32_t* counts, int64_t experts, float rate) {
    __shared__ int64_t red[kRThreads / 64];
    int64_t total = 0;
    for (int64_t e = threadIdx.x; e < experts; e += kRThreads) total += counts[e];
    total = block_sum<kRThreads / 64>(total, red);
    for (int64_t e = threadIdx.x; e < experts; e += kRThreads) {
        const int64_t c = counts[e] * experts;
        if (c < total) bias[e] += rate;
        if (c > total) bias[e] -= rate;
    }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
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

int router_check(const char* what, int64_t rows, int64_t experts, int64_t k, int scores, float scale) {
    if (rows < 0 || experts < 1 || experts > kMaxExperts || k < 1 || k > kMaxChosen || k > experts)
        return fail(MH_ERR_INVALID, "%s: needs rows >= 0, 1 <= experts <= %d, 1 <= k <= min(%d, experts) (%lld, %lld, %lld)",
                    what, kMaxExperts, kMaxChosen, (long long)rows, (long long)experts, (long long)k);
    if (scores != MH_SCORES_SOFTMAX && scores != MH_SCORES_SIGMOID) return fail(MH_ERR_INVALID, "%s: scores %d", what, scores);
    if (!(scale >= -3.4028234663852886e38f && scale <= 3.4028234663852886e38f))
        return fail(MH_ERR_INVALID, "%s: scale %g is not finite", what, (double)scale);
    if (rows > 0x7fffffff / k) return fail(MH_ERR_OVERFLOW, "%s: more than 2^31 - 1 choices", what);
    return MH_OK;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_group_router_fwd(float* weights, int32_t* chosen, int32_t* counts, const float* x, const float* bias,
                        const int32_t* keep, int64_t rows, int64_t experts, int64_t k, int64_t groups, int64_t keep_groups,
                        int group_best, int scores, int normalise, float scale) {
    MH_TRACE("mh_group_router_fwd");
    MH_TRY(router_check("mh_group_router_fwd", rows, experts, k, scores, scale));
    if (groups < 1 || groups > kMaxGroups || experts % groups != 0 || keep_groups < 1 || keep_groups > groups ||
        keep_groups * (experts / groups) < k || (group_best != 1 && group_best != 2))
        return fail(MH_ERR_INVALID,
                    "mh_group_router_fwd: needs 1 <= groups <= %d that divide %lld experts, 1 <= keep_groups <= groups with %lld "
                    "experts at least, group_best 1 or 2 (%lld, %lld, %d)",
                    kMaxGroups, (long long)experts, (long long)k, (long long)groups, (long long)keep_groups, group_best);
    if (!counts || (rows > 0 && (!weights || !chosen || !x))) return fail(MH_ERR_NULL, "mh_group_router_fwd: null tensor");
    MH_TRY(require_init());
    if (rows == 0) return mh_zero(reinterpret_cast<float*>(counts), experts);  // zero bits are the whole number 0 too
    GroupArg a = {};
    a.x = x;
    a.bias = bias;
    a.keep = keep;
    a.rows = rows;
    a.experts = (int32_t)experts;
    a.k = (int32_t)k;
    // where every group stays open there is nothing to sort out
    a.groups = keep_groups == groups ? 1 : (int32_t)groups;
    a.each = (int32_t)(experts / groups);
    a.open = (int32_t)keep_groups;
    a.best = group_best;
    a.by_each = make_fastdiv((uint32_t)a.each);
    a.sigmoid = scores == MH_SCORES_SIGMOID;
    a.normalise = normalise != 0;
    a.scale = scale;
    a.weights = weights;
    a.chosen = chosen;
    hipStream_t st = ctx().stream;
    const int64_t waves = kRThreads / 64, group = kRThreads / router_lanes(a.experts);
    const bool lists = rows > kRExactRows;
    a.parts = 1;
    while (2 * a.parts * a.groups <= router_lanes(a.experts)) a.parts *= 2;
    a.wave_parts = 1;
    while (2 * a.wave_parts * a.groups <= 64) a.wave_parts *= 2;
    int64_t blocks = lists ? (rows + group - 1) / group : 0;
    if (blocks > kRBlocks) blocks = (blocks + (blocks + kRBlocks - 1) / kRBlocks - 1) / ((blocks + kRBlocks - 1) / kRBlocks);  // equal rounds
    int64_t exact = lists ? kRExactBlocks : (rows + waves - 1) / waves;
    if (exact > kRBlocks) exact = kRBlocks;
    char* base = nullptr;
    const size_t list_bytes = lists ? (size_t)rows * 4 : 0, part_bytes = (size_t)(blocks + exact) * experts * 4;
    MH_TRY(scratch(list_bytes + part_bytes, reinterpret_cast<void**>(&base)));
    int32_t* part = reinterpret_cast<int32_t*>(base + list_bytes);
    a.part_c = part;
    if (lists) {
        MH_TRY(tickets(1, &a.ntodo));
        a.todo = reinterpret_cast<int32_t*>(base);
#define MH_CALL(L, V)                                                                                                             \
    do {                                                                                                                         \
        if (a.sigmoid) hipLaunchKernelGGL((k_group_router_fwd<L, V, true>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a);  \
        else hipLaunchKernelGGL((k_group_router_fwd<L, V, false>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a);           \
    } while (0)
        MH_ROUTER(MH_CALL);
#undef MH_CALL
        a.part_c += blocks * experts;
    }
    const bool alone = !lists && exact <= kRArrivals;
    if (alone) {
        MH_TRY(tickets(1, &a.arrived));
        a.counts = counts;
    }
    if (a.experts <= 64) hipLaunchKernelGGL(k_group_router_exact<1>, dim3((unsigned)exact), dim3(kRThreads), 0, st, a);
    else if (a.experts <= 256) hipLaunchKernelGGL(k_group_router_exact<4>, dim3((unsigned)exact), dim3(kRThreads), 0, st, a);
    else hipLaunchKernelGGL(k_group_router_exact<16>, dim3((unsigned)exact), dim3(kRThreads), 0, st, a);
    if (alone) return finish("mh_group_router_fwd");
    hipLaunchKernelGGL(k_group_router_counts, dim3((unsigned)((experts + 31) / 32)), dim3(1024), 0, st, part,
                       (int32_t)(blocks + exact), a.experts, counts, a.ntodo);
    return finish("mh_group_router_fwd");
}

int mh_group_router_bwd(float* grad_x, const float* x, const int32_t* keep, const int32_t* chosen, const float* grad_weights,
                        int64_t rows, int64_t experts, int64_t k, int scores, int normalise, float scale, int accumulate) {
    MH_TRACE("mh_group_router_bwd");
    MH_TRY(router_check("mh_group_router_bwd", rows, experts, k, scores, scale));
    if (rows == 0) return MH_OK;
    if (!grad_x || !x || !chosen || !grad_weights) return fail(MH_ERR_NULL, "mh_group_router_bwd: null tensor");
    MH_TRY(require_init());
    GroupArg a = {};
    a.x = x;
    a.keep = keep;
    a.rows = rows;
    a.experts = (int32_t)experts;
    a.k = (int32_t)k;
    a.sigmoid = scores == MH_SCORES_SIGMOID;
    a.normalise = normalise != 0;
    a.accumulate = accumulate != 0;
    a.scale = scale;
    a.grad = grad_x;
    a.gw = grad_weights;
    a.sel = chosen;
    const int64_t group = kRThreads / router_lanes(a.experts);
    int64_t blocks = (rows + group - 1) / group;
    if (blocks > 2048) blocks = 2048;
    hipStream_t st = ctx().stream;
#define MH_CALL(L, V) hipLaunchKernelGGL((k_group_router_bwd<L, V>), dim3((unsigned)blocks), dim3(kRThreads), 0, st, a)
    MH_ROUTER(MH_CALL);
#undef MH_CALL
    return finish("mh_group_router_bwd");
}

int mh_router_bias_update(float* bias, const int32_t* counts, int64_t experts, float rate) {
    MH_TRACE("mh_router_bias_update");
    if (experts < 1 || experts > kMaxExperts) return fail(MH_ERR_INVALID, "mh_router_bias_update: 1 <= experts <= %d (%lld)", kMaxExperts, (long long)experts);
    if (!(rate >= -3.4028234663852886e38f && rate <= 3.4028234663852886e38f))
        return fail(MH_ERR_INVALID, "mh_router_bias_update: rate %g is not finite", (double)rate);
    if (!bias || !counts) return fail(MH_ERR_NULL, "mh_router_bias_update: null tensor");
    MH_TRY(require_init());
    hipLaunchKernelGGL(k_router_bias, dim3(1), dim3(kRThreads), 0, ctx().stream, bias, counts, experts, rate);
    return finish("mh_router_bias_update");
}

}  // extern "C"
