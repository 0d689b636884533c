// mh_sample.hip -- a token for each row of logits from a uniform number, after temperature, top-k, top-p and min-p.
//
// The classes that top-k and top-p keep are a beginning of the row in the order of falling logits, ties by index: a
// threshold value t, the classes above it and the first few at it. Sums of probabilities decide where it ends, and a
// running sum in the order of the classes which one is drawn, so a class's mass e^((x - max) / T) is held as a whole
// number, 2^shift for the largest: sums are exact in any order, whatever the waves' or atomics' order, and every pass over
// a row sees the same ones. `shift` leaves room for all classes, 2^(62 - log2 classes).
//
// A workgroup takes a row. The threshold is found by the logits' bits, 8 at a time from the top: counts and masses by those bits
// in LDS, the digit where the count or the mass reaches what is kept, and on among the classes with that digit.
#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kSThreads = 1024;
constexpr int kSWaves = kSThreads / 64;
constexpr int64_t kMaxSampled = (int64_t)1 << 24;

struct SampleArg {
    const float* x;
    const float* u;
    const float* temperature;  // or null, as the next three
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* tokens;
    float* logprob;  // or null
    int64_t rows;
    int32_t classes;
    int32_t shift;
};

// A logit's order as a whole number, -0 as +0.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

// What a row's masses are made from.
struct Heat {
    float top;       // the largest logit
    float hi, lo;    // log2(e) / T in two parts
    float least;     // x - top below which min_p drops a class
    int shift;
};
// 2^shift e^((x - top) / T): the exponent in two parts, so that what rounds is the result.
__device__ __forceinline__ uint64_t mass_of(float x, const Heat& h) {
    if (x == h.top) return (uint64_t)1 << h.shift;
    const float d = x - h.top;
    const float t = d * h.hi;
    if (!(t > -63.0f)) return 0;
    const float n = __builtin_rintf(t);
    const float r = __builtin_fmaf(d, h.hi, -n) + d * h.lo;
    // 24 bits and the place they start at
    const float e = __builtin_amdgcn_exp2f(r);
    const double m = __builtin_ldexp((double)e, (int)n + h.shift);
    return (uint64_t)(m + 0.5);
}

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {  // sums up to and with each lane
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T w = __shfl_up(v, o);
        if ((int)(threadIdx.x & 63) >= o) v += w;
    }
    return v;
}

struct Threshold {
    uint32_t key;     // the value's order
    uint64_t ties;    // how many classes of it count
};

// The first classes of a row, by falling logits, whose count reaches `count`, or whose mass reaches `mass` (whichever is not
// 0), as a threshold; `sum` gets their mass. Both are known to be reached. hist_n and hist_m hold 256 each.
__device__ Threshold find(const float* x, int classes, const Heat& h, uint64_t count, uint64_t mass, uint32_t* hist_n,
                          unsigned long long* hist_m, uint64_t* sum, unsigned long long* said) {
    uint32_t prefix = 0, bits = 0;
    uint64_t above_n = 0, above_m = 0;
    for (int place = 24; place >= 0; place -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kSThreads) {
            hist_n[i] = 0;
            hist_m[i] = 0;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < classes; c += kSThreads) {
            const float v = x[c];
            const uint32_t k = order_of(v);
            if ((k & bits) != prefix) continue;
            atomicAdd(&hist_n[(k >> place) & 255], 1u);
            atomicAdd(&hist_m[(k >> place) & 255], (unsigned long long)mass_of(v, h));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t n = above_n, m = above_m;
            int b = 255;
            for (; b > 0; --b) {
                if (count ? n + hist_n[b] >= count : m + hist_m[b] >= mass) break;
                n += hist_n[b];
                m += hist_m[b];
            }
            said[0] = n;
            said[1] = m;
            said[2] = b;
            said[3] = hist_n[b];
        }
        __syncthreads();
        above_n = said[0];
        above_m = said[1];
        prefix |= (uint32_t)said[2] << place;
        bits |= 255u << place;
    }
    Threshold t;
    t.key = prefix;
    const uint64_t each = mass_of(of_order(prefix), h);
    const uint64_t here = said[3];
    if (count) t.ties = count - above_n;
    else t.ties = each ? (mass - above_m + each - 1) / each : here;
    if (t.ties > here) t.ties = here;
    *sum = above_m + t.ties * each;
    return t;
}

__global__ __launch_bounds__(kSThreads) void k_sample(SampleArg a) {
    __shared__ uint32_t hist_n[256];
    __shared__ unsigned long long hist_m[256], said[4], seg_m[kSWaves];
    __shared__ uint32_t seg_n[kSWaves];
    __shared__ float red_v[kSWaves];
    __shared__ int red_i[kSWaves], bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float* x = a.x + r * a.classes;
        // the largest logit, at its lowest index
        float best = -__builtin_inff();
        int at = 0x7fffffff;
        bool nan = false;
        __syncthreads();
        if (tid == 0) bad = 0;
        for (int c = tid; c < a.classes; c += kSThreads) {
            const float v = x[c];
            nan |= v != v;
            if (v > best) {
                best = v;
                at = c;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float v = __shfl_xor(best, o);
            const int i = __shfl_xor(at, o);
            if (v > best || (v == best && i < at)) {
                best = v;
                at = i;
            }
        }
        if (lane == 0) {
            red_v[wave] = best;
            red_i[wave] = at;
        }
        __syncthreads();
        if (nan) bad = 1;
#pragma unroll
        for (int i = 0; i < kSWaves; ++i)
            if (red_v[i] > best || (red_v[i] == best && red_i[i] < at)) {
                best = red_v[i];
                at = red_i[i];
            }
        __syncthreads();
        const float T = a.temperature ? a.temperature[r] : 1.0f;
        const bool none = bad != 0 || best == -__builtin_inff();
        if (none || !(T > 0.0f)) {
            if (tid == 0) {
                a.tokens[r] = none ? -1 : at;
                if (a.logprob) a.logprob[r] = none ? __builtin_nanf("") : 0.0f;
            }
            continue;
        }
        Heat h;
        h.top = best;
        const double per = 1.4426950408889634074 / (double)T;
        h.hi = (float)per;
        h.lo = (float)(per - (double)h.hi);
        h.shift = a.shift;
        h.least = -__builtin_inff();
        Threshold t = {0, 0};  // every class
        const int k = a.top_k ? a.top_k[r] : 0;
        const float p = a.top_p ? a.top_p[r] : 1.0f;
        const float mp = a.min_p ? a.min_p[r] : 0.0f;
        uint64_t sum = 0;
        bool cut = false;
        if (k > 0 && k < a.classes) {
            t = find(x, a.classes, h, (uint64_t)k, 0, hist_n, hist_m, &sum, said);
            cut = true;
        }
        if (p < 1.0f) {
            if (!cut) {
                uint64_t s = 0;
                for (int c = tid; c < a.classes; c += kSThreads) s += mass_of(x[c], h);
                sum = block_sum<kSWaves>((unsigned long long)s, seg_m);
            }
            const double part = (double)(p > 0.0f ? p : 0.0f) * (double)sum;
            uint64_t need = (uint64_t)__builtin_ceil(part);
            need = need < 1 ? 1 : (need > sum ? sum : need);
            t = find(x, a.classes, h, 0, need, hist_n, hist_m, &sum, said);
            cut = true;
        }
        // min_p on what is left
        const double limit = mp > 0.0f ? (mp >= 1.0f ? 0.0 : log((double)mp) * (double)T) : -__builtin_inf();
        auto stays = [&](float v) { return v == best || (double)v - (double)best >= limit; };
        // a wavefront's share of the classes in their order: the masses above the threshold, and how many are at it
        const int share = (a.classes + kSWaves - 1) / kSWaves;
        const int c0 = wave * share, c1 = c0 + share < a.classes ? c0 + share : a.classes;
        uint64_t m = 0;
        uint32_t n = 0;
        for (int c = c0 + lane; c < c1; c += 64) {
            const float v = x[c];
            const uint32_t o = order_of(v);
            if (!stays(v)) continue;
            if (!cut || o > t.key) m += mass_of(v, h);
            else n += o == t.key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            m += __shfl_xor((unsigned long long)m, o);
            n += __shfl_xor(n, o);
        }
        __syncthreads();
        if (lane == 0) {
            seg_m[wave] = m;
            seg_n[wave] = n;
        }
        __syncthreads();
        const uint64_t each = cut ? mass_of(of_order(t.key), h) : 0;
        uint64_t total = 0, before = 0, ties = 0;
        uint64_t ties_before = 0;
        for (int i = 0; i < kSWaves; ++i) {
            const uint64_t left = t.ties - ties;
            const uint64_t here = seg_n[i] < left ? seg_n[i] : left;
            if (i == wave) {
                before = total;
                ties_before = ties;
            }
            total += seg_m[i] + here * each;
            ties += here;
        }
        float u = a.u[r];
        u = u > 0.0f ? u : 0.0f;
        uint64_t goal = (uint64_t)((double)u * (double)total);
        goal = goal < total ? goal : total - 1;
        // the wavefront whose share holds it walks through it
        uint64_t mine = seg_m[wave];
        {
            const uint64_t left = t.ties - ties_before;
            mine += (seg_n[wave] < left ? seg_n[wave] : left) * each;
        }
        if (goal >= before && goal < before + mine) {
            for (int b = c0; b < c1; b += 64) {
                const int c = b + lane;
                const float v = c < c1 ? x[c] : -__builtin_inff();
                const uint32_t o = order_of(v);
                const bool in = c < c1 && stays(v);
                const bool tie = in && cut && o == t.key;
                const uint32_t at_tie = wave_scan((uint32_t)tie);
                uint64_t w = in && (!cut || o > t.key) ? mass_of(v, h) : 0;
                if (tie && ties_before + at_tie <= t.ties) w = each;
                const uint64_t upto = wave_scan((unsigned long long)w);
                const uint64_t hit = __ballot(before + upto > goal);
                if (hit) {
                    const int first = __builtin_ctzll(hit);
                    if (lane == first) {
                        a.tokens[r] = c;
                        if (a.logprob)
                            a.logprob[r] = (float)((v == best ? 0.0 : ((double)v - (double)best) / (double)T) -
                                                   log(__builtin_ldexp((double)total, -a.shift)));
                    }
                    break;
                }
                before += __shfl((unsigned long long)upto, 63);
                ties_before += __shfl(at_tie, 63);
            }
        }
    }
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_sample_tokens(int32_t* tokens, float* logprob, const float* x, const float* u, const float* temperature,
                     const int32_t* top_k, const float* top_p, const float* min_p, int64_t rows, int64_t classes) {
    MH_TRACE("mh_sample_tokens");
    if (rows < 0 || classes < 1) return fail(MH_ERR_INVALID, "mh_sample_tokens: needs rows >= 0 and classes >= 1 (%lld, %lld)", (long long)rows, (long long)classes);
    if (classes > kMaxSampled || rows > 0x7fffffff)
        return fail(MH_ERR_OVERFLOW, "mh_sample_tokens: more than 2^24 classes or 2^31 - 1 rows (%lld, %lld)", (long long)classes, (long long)rows);
    if (rows == 0) return MH_OK;
    if (!tokens || !x || !u) return fail(MH_ERR_NULL, "mh_sample_tokens: null tensor");
    MH_TRY(require_init());
    SampleArg a = {};
    a.x = x;
    a.u = u;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.tokens = tokens;
    a.logprob = logprob;
    a.rows = rows;
    a.classes = (int32_t)classes;
    a.shift = 62;
    while (((int64_t)1 << (62 - a.shift)) < classes) --a.shift;
    const int64_t blocks = rows < 4096 ? rows : 4096;
    hipLaunchKernelGGL(k_sample, dim3((unsigned)blocks), dim3(kSThreads), 0, ctx().stream, a);
    return finish("mh_sample_tokens");
}

}  // extern "C"
