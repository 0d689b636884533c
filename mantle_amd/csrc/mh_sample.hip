// mh_sample.hip -- a token for each row of logits from a uniform number, after temperature, top-k, top-p and min-p.
//
// What top-k, top-p and min-p keep is a beginning of the row in the order of falling logits, ties by index: it ends at one
// class, the cut. The token is the first class, by index, where the running sum of the kept masses e^((x - max) / T) exceeds u
// of their sum.
//
// A workgroup takes a row, a wavefront a run of its classes, of which each lane holds 4 Q logits in registers (the whole
// row up to 4 Q T classes; of a longer one the rest is read twice, the second time mostly from the caches):
//   1. the largest logit held, and bins of a power-of-two width below (and some above) it;
//   2. for top-k and top-p how many classes each bin has and their mass, both in one 64-bit LDS atomic: 20 bits of count above
//      44 of mass, a class 24 bits of its bin's largest. Whole numbers: the atomics' order does not show. A sum over the bins
//      then says in which of them a cut falls;
//   3. a second walk over the logits adds up what lies above those bins and lists what lies in them;
//   4. the list, a few hundred classes, is sorted, and the cuts are found in it by 64-bit sums;
//   5. the run of classes where the running sum passes u of the total is walked by the whole workgroup.
// Sums of step 3 to 5 are 64-bit floats in a fixed order. Masses are fp32: their rounding, 2^-22 of each and without a common
// sign, moves a border by some 2^-24 of the row.
//
// Rows for which bins do not work (a list of more than 2048 classes, as ties of thousands give, an infinite logit,
// temperatures beyond 1e30 or whose bins would span more than 16 powers of two, more than 2^19 classes) go by whole-number masses and a
// search over the logits' bits, 8 at a time: right for every row, and slower.
#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {
namespace {

constexpr int kBins = 4096;
constexpr int kAbove = 1024;  // of them above the largest logit that step 1 saw
constexpr int kList = 2048;
constexpr int kCountAt = 44;
constexpr int64_t kMaxBinned = (int64_t)1 << 19;
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
    int64_t row0;
    int32_t classes;
    int32_t shift;  // of the whole-number masses: 2^shift for the largest, room for all classes
};

// A row's settings.
struct Ask {
    int k;       // 0: all
    float p;     // 1: all
    double T;
    double limit;  // x - max below which min_p drops a class
    float u;
};

// A logit's order as a whole number, -0 as +0.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {  // sums up to and with each lane
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T w = __shfl_up(v, o);
        if ((int)(threadIdx.x & 63) >= o) v += w;
    }
    return v;
}

// log of the drawn class's share of the kept mass, `total` in units of the largest class's mass.
__device__ __forceinline__ float share_log(float v, float best, double T, double total) {
    return (float)((v == best ? 0.0 : ((double)v - (double)best) / T) - log(total));
}

// ---------------------------------------------------------------------------------------
// any row: whole-number masses
// ---------------------------------------------------------------------------------------
struct Heat {
    float top;     // the largest logit
    float hi, lo;  // log2(e) / T in two parts
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
    return (uint64_t)(__builtin_ldexp((double)__builtin_amdgcn_exp2f(r), (int)n + h.shift) + 0.5);
}

struct Threshold {
    uint32_t key;   // the value's order
    uint64_t ties;  // how many classes of it count
};

struct SlowLds {
    unsigned long long hist_m[256], said[4], seg_m[16];
    uint32_t hist_n[256], seg_n[16];
};

// The first classes of a row, by falling logits, whose count reaches `count`, or whose mass reaches `mass` (whichever is not
// 0), as a threshold; `sum` gets their mass. Both are known to be reached.
template <int T>
__device__ Threshold find(const float* x, int classes, const Heat& h, uint64_t count, uint64_t mass, SlowLds& s, uint64_t* sum) {
    uint32_t prefix = 0, bits = 0;
    uint64_t above_n = 0, above_m = 0;
    for (int place = 24; place >= 0; place -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += T) {
            s.hist_n[i] = 0;
            s.hist_m[i] = 0;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < classes; c += T) {
            const float v = x[c];
            const uint32_t k = order_of(v);
            if ((k & bits) != prefix) continue;
            atomicAdd(&s.hist_n[(k >> place) & 255], 1u);
            atomicAdd(&s.hist_m[(k >> place) & 255], (unsigned long long)mass_of(v, h));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t n = above_n, m = above_m;
            int b = 255;
            for (; b > 0; --b) {
                if (count ? n + s.hist_n[b] >= count : m + s.hist_m[b] >= mass) break;
                n += s.hist_n[b];
                m += s.hist_m[b];
            }
            s.said[0] = n;
            s.said[1] = m;
            s.said[2] = b;
            s.said[3] = s.hist_n[b];
        }
        __syncthreads();
        above_n = s.said[0];
        above_m = s.said[1];
        prefix |= (uint32_t)s.said[2] << place;
        bits |= 255u << place;
    }
    Threshold t;
    t.key = prefix;
    const uint64_t each = mass_of(of_order(prefix), h);
    const uint64_t here = s.said[3];
    if (count) t.ties = count - above_n;
    else t.ties = each ? (mass - above_m + each - 1) / each : here;
    if (t.ties > here) t.ties = here;
    *sum = above_m + t.ties * each;
    return t;
}

template <int T>
__device__ __attribute__((noinline)) void slow_row(const float* x, int classes, int shift, int32_t* token, float* logprob, float best,
                                                   Ask ask, SlowLds& s) {
    constexpr int W = T / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Heat h;
    h.top = best;
    const double per = 1.4426950408889634074 / ask.T;
    h.hi = (float)per;
    h.lo = (float)(per - (double)h.hi);
    h.shift = shift;
    Threshold t = {0, 0};
    uint64_t sum = 0;
    bool cut = false;
    if (ask.k > 0) {
        t = find<T>(x, classes, h, (uint64_t)ask.k, 0, s, &sum);
        cut = true;
    }
    if (ask.p < 1.0f) {
        if (!cut) {
            unsigned long long m = 0;
            for (int c = tid; c < classes; c += T) m += mass_of(x[c], h);
            sum = block_sum<W>(m, s.seg_m);
        }
        uint64_t need = (uint64_t)__builtin_ceil((double)ask.p * (double)sum);
        need = need < 1 ? 1 : (need > sum ? sum : need);
        t = find<T>(x, classes, h, 0, need, s, &sum);
        cut = true;
    }
    auto stays = [&](float v) { return v == best || (double)v - (double)best >= ask.limit; };
    // a wavefront's share of the classes in their order: the masses above the threshold, and how many are at it
    const int share = (classes + W - 1) / W;
    const int c0 = wave * share, c1 = c0 + share < classes ? c0 + share : classes;
    unsigned long long m = 0;
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
        m += __shfl_xor(m, o);
        n += __shfl_xor(n, o);
    }
    __syncthreads();
    if (lane == 0) {
        s.seg_m[wave] = m;
        s.seg_n[wave] = n;
    }
    __syncthreads();
    const uint64_t each = cut ? mass_of(of_order(t.key), h) : 0;
    uint64_t total = 0, before = 0, mine = 0, ties = 0, ties_before = 0;
    for (int i = 0; i < W; ++i) {
        const uint64_t left = t.ties - ties, here = s.seg_n[i] < left ? s.seg_n[i] : left;
        const uint64_t add = s.seg_m[i] + here * each;
        if (i == wave) {
            before = total;
            ties_before = ties;
            mine = add;
        }
        total += add;
        ties += here;
    }
    uint64_t goal = (uint64_t)((double)ask.u * (double)total);
    goal = goal < total ? goal : total - 1;
    // the wavefront whose share holds it walks through it
    if (goal < before || goal >= before + mine) return;
    for (int b = c0; b < c1; b += 64) {
        const int c = b + lane;
        const float v = c < c1 ? x[c] : -__builtin_inff();
        const uint32_t o = order_of(v);
        const bool in = c < c1 && stays(v);
        const bool tie = in && cut && o == t.key;
        const uint32_t at_tie = wave_scan((uint32_t)tie);
        unsigned long long w = in && (!cut || o > t.key) ? mass_of(v, h) : 0;
        if (tie && ties_before + at_tie <= t.ties) w = each;
        const unsigned long long upto = wave_scan(w);
        const uint64_t hit = __ballot(before + upto > goal);
        if (hit) {
            if (lane == __builtin_ctzll(hit)) {
                *token = c;
                if (logprob) *logprob = share_log(v, best, ask.T, __builtin_ldexp((double)total, -shift));
            }
            break;
        }
        before += __shfl(upto, 63);
        ties_before += __shfl(at_tie, 63);
    }
}

// ---------------------------------------------------------------------------------------
// rows that bins sort out
// ---------------------------------------------------------------------------------------
struct FastLds {
    union {
        unsigned long long hist[kBins];
        struct {
            uint64_t key[kList];  // order inverted, then the index: rising is the order that is kept
            double upto[kList];   // sums of masses
        } list;
    };
    double wave_d[16], seg[16];
    uint32_t wave_n[16];
    float wave_f[16];
    int wave_i[16];
    // what one thread found out for all
    uint32_t listed, k_bin, k_above_n, k_here, p_lo, p_hi;
    double k_above, k_in, p_above, all;
    int over, bad, first, last;
    uint64_t cut;
};

// Exclusive sums over the workgroup's threads of a count and a mass, and the totals; `after` is what each thread's own
// gives the next one, the same bits as its neighbour's.
template <int W>
__device__ __forceinline__ void block_scan(uint32_t n, double m, uint32_t& n0, double& m0, double& m1, uint32_t& n_all, double& m_all,
                                           FastLds& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t ni = wave_scan(n);
    const double mi = wave_scan(m);
    __syncthreads();
    if (lane == 63) {
        s.wave_n[wave] = ni;
        s.wave_d[wave] = mi;
    }
    __syncthreads();
    uint32_t nb = 0;
    double mb = 0.0;
    n_all = 0;
    m_all = 0.0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (i == wave) {
            nb = n_all;
            mb = m_all;
        }
        n_all += s.wave_n[i];
        m_all += s.wave_d[i];
    }
    const uint32_t np = __shfl_up(ni, 1);
    const double mp = __shfl_up(mi, 1);
    n0 = nb + (lane ? np : 0);
    m0 = lane ? mb + mp : mb;
    m1 = mb + mi;
}

// A row of logits as a buffer: reads past its end give 0 rather than branch.
typedef __amdgpu_buffer_rsrc_t Row;
__device__ __forceinline__ Row row_of(const float* x, int classes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(x), 0, 4 * classes, 0x00020000);
}
typedef uint32_t vu4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ vf4 logits(Row row, int c) {
    return __builtin_bit_cast(vf4, __builtin_amdgcn_raw_buffer_load_b128(row, 4 * c, 0, 0));
}
// What lies past a row's end as minus infinity.
__device__ __forceinline__ void close_row(vf4& v, int c, int classes) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < classes ? v[j] : -__builtin_inff();
}

// Where a logit falls: places of bin width below the reference, negative above it; past the last bin, and at minus
// infinity, the last.
__device__ __forceinline__ float place_of(float v, float ref, float per_bin) {
    return __builtin_fminf((ref - v) * per_bin, (float)(kBins - 1 - kAbove));
}

template <int T, int Q>
__global__ __launch_bounds__(T) void k_sample(SampleArg a) {
    constexpr int W = T / 64;
    constexpr int B = kBins / T;  // bins of a thread
    __shared__ union { FastLds f; SlowLds s; } lds;
    FastLds& s = lds.f;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // a wavefront's run of classes: whole rounds of 256
    const int run = (a.classes + 256 * W - 1) / (256 * W) * 256;
    const int w0 = wave * run, c0 = w0 + 4 * lane;
    const int quads = run / 256;
    const int64_t r = a.row0 + blockIdx.x;
    const float* x = a.x + r * a.classes;
    const Row row = row_of(x, a.classes);
    vf4 h[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) h[i] = logits(row, i < quads ? c0 + 256 * i : a.classes);
#pragma unroll
    for (int i = 0; i < Q; ++i)
        if (w0 + 256 * (i + 1) > a.classes || i >= quads) close_row(h[i], i < quads ? c0 + 256 * i : a.classes, a.classes);
    // every logit of the row: those held, then the others
    auto held = [&](auto&& f) {
        int at = c0;
        asm volatile("" : "+v"(at));  // or every walk shares 64 registers of indices
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if (i < quads) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = h[i][j];
                    asm volatile("" : "+v"(v));  // nothing made of it is kept from one walk to the next
                    f(v, at + 256 * i + j);
                }
                __builtin_amdgcn_sched_barrier(0);  // a quad's work at a time: all of them need 700 registers
            }
    };
    auto rest = [&](auto&& f) {
        if (quads <= Q) return;
        vf4 next = logits(row, c0 + 256 * Q);
        for (int i = Q; i < quads; ++i) {
            vf4 v = next;
            next = logits(row, i + 1 < quads ? c0 + 256 * (i + 1) : a.classes);
            if (w0 + 256 * (i + 1) > a.classes) close_row(v, c0 + 256 * i, a.classes);
#pragma unroll
            for (int j = 0; j < 4; ++j) f(v[j], c0 + 256 * i + j);
        }
    };
    const float T_ = a.temperature ? a.temperature[r] : 1.0f;
    Ask ask;
    ask.T = (double)T_;
    ask.k = a.top_k ? a.top_k[r] : 0;
    ask.p = a.top_p ? a.top_p[r] : 1.0f;
    if (!(ask.p < 1.0f)) ask.p = 1.0f;
    if (ask.p <= 0.0f) ask.k = 1, ask.p = 1.0f;  // the likeliest alone
    if (ask.k < 0 || ask.k >= a.classes) ask.k = 0;
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    ask.limit = mp > 0.0f ? (mp >= 1.0f ? 0.0 : log((double)mp) * ask.T) : -__builtin_inf();
    ask.u = a.u[r];
    ask.u = ask.u > 0.0f ? (ask.u < 1.0f ? ask.u : 0.999999940395355f) : 0.0f;
    const bool greedy = !(T_ > 0.0f);
    const bool cuts = !greedy && (ask.k > 0 || ask.p < 1.0f);
    // the largest logit held, and the least
    float top = -__builtin_inff(), low = __builtin_inff();
    bool nan = false;
    held([&](float v, int) {
        nan |= v != v;
        top = __builtin_fmaxf(top, v);
        low = v > -__builtin_inff() ? __builtin_fminf(low, v) : low;
    });
    auto block_top = [&](float& hi, float* lo) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            hi = __builtin_fmaxf(hi, __shfl_xor(hi, o));
            if (lo) *lo = __builtin_fminf(*lo, __shfl_xor(*lo, o));
        }
        __syncthreads();
        if (lane == 0) {
            s.wave_f[wave] = hi;
            if (lo) s.wave_d[wave] = (double)*lo;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) {
            hi = __builtin_fmaxf(hi, s.wave_f[i]);
            if (lo) *lo = __builtin_fminf(*lo, (float)s.wave_d[i]);
        }
    };
    if (tid == 0) s.bad = 0;
    block_top(top, &low);
    float best = top;
    // bins as narrow as the held logits' range allows, none wider than what e^-44 of the largest needs
    float width = 0.0f, per_bin = 0.0f, ref = top;
    bool binned = false;
    if (cuts && a.classes <= kMaxBinned && top > -__builtin_inff() && top < __builtin_inff()) {
        const float widest = __builtin_fmaxf(T_ * (1.0f / 64.0f), 1.0f / 128.0f);
        const float wish = __builtin_fminf(widest, (top - low) * (1.25f / (kBins - kAbove)));
        const int e = __builtin_amdgcn_frexp_expf(__builtin_fmaxf(wish, T_ * 1e-6f));
        width = __builtin_ldexpf(1.0f, e);
        per_bin = __builtin_ldexpf(1.0f, -e);
        binned = true;
    }
    double rate = 0.0;  // a bin's width over T, in powers of two
    bool wide = false;
    for (int turn = 0; binned; ++turn) {
        rate = (double)width * 1.4426950408889634074 / ask.T;
        if (turn == 3 || !(rate <= 16.0) || !(rate >= 1e-9)) {
            binned = false;
            break;
        }
        const float neg = -(float)rate;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < B; ++i) s.hist[i * T + tid] = 0;
        if (tid == 0) s.over = 0;
        __syncthreads();
        int over = 0;
        // what lies past the last bin has less than e^-44 of the largest's mass, or the bins are too narrow
        const float far = ref - 44.0f * T_;
        auto count = [&](float v, int c) {
            const float q = place_of(v, ref, per_bin);
            const float f = __builtin_floorf(q);
            const int b = (int)f + kAbove;
            uint32_t m = (uint32_t)__builtin_fmaf(__builtin_amdgcn_exp2f((q - f) * neg), 16777216.0f, 0.5f);
            const bool last = b == kBins - 1;
            over |= (b < 0) | (last && v > far ? 2 : 0);
            m = last ? 0 : m;
            if (c < a.classes) atomicAdd(&s.hist[b < 0 ? 0 : b], (unsigned long long)1 << kCountAt | m);
        };
        held(count);
        rest([&](float v, int c) {
            nan |= v != v;
            best = __builtin_fmaxf(best, v);
            count(v, c);
        });
        if (over) atomicOr(&s.over, over);
        if (quads > Q) block_top(best, nullptr);
        else __syncthreads();
        over = s.over;
        if (!over || best == __builtin_inff()) break;
        // a larger logit was among the others, or one far below: once more, from the largest, with wider bins
        ref = best;
        if ((over & 2) || wide) {
            const int e = __builtin_amdgcn_frexp_expf(__builtin_fmaxf(T_ * (1.0f / 64.0f), 1.0f / 128.0f));
            width = __builtin_ldexpf(1.0f, e);
            per_bin = __builtin_ldexpf(1.0f, -e);
            wide = true;
        }
    }
    if (!binned && quads > Q) {
        rest([&](float v, int) {
            nan |= v != v;
            best = __builtin_fmaxf(best, v);
        });
        block_top(best, nullptr);
    }
    if (nan) s.bad = 1;
    __syncthreads();
    const bool none = s.bad != 0 || best == -__builtin_inff();
    if (none || greedy) {  // the lowest index of the largest
        if (tid == 0) s.first = 0x7fffffff;
        __syncthreads();
        int at = 0x7fffffff;
        auto look = [&](float v, int c) { at = v == best && c < at ? c : at; };
        if (!none) {
            held(look);
            rest(look);
        }
        if (at != 0x7fffffff) atomicMin(&s.first, at);
        __syncthreads();
        if (tid == 0) {
            a.tokens[r] = none ? -1 : s.first;
            if (a.logprob) a.logprob[r] = none ? __builtin_nanf("") : 0.0f;
        }
        return;
    }
    bool slow = (cuts && !binned) || best == __builtin_inff() || !(T_ >= 1e-30f && T_ <= 1e30f);
    if (!slow && cuts) {
        // the bins' counts and masses, from the top down
        double M[B];
        uint32_t N[B], n = 0;
        double m = 0.0;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int b = tid * B + i;
            const uint64_t v = s.hist[b];
            N[i] = (uint32_t)(v >> kCountAt);
            M[i] = N[i] ? (double)(v & (((uint64_t)1 << kCountAt) - 1)) * exp2(-rate * (double)(b - kAbove)) * (1.0 / 16777216.0) : 0.0;
            n += N[i];
            m += M[i];
        }
        uint32_t n0, n_all;
        double m0, m1, m_all;
        block_scan<W>(n, m, n0, m0, m1, n_all, m_all, s);
        if (tid == 0) {
            s.listed = 0;
            s.k_bin = s.p_lo = s.p_hi = kBins;
        }
        __syncthreads();
        if (ask.k > 0 && n0 < (uint32_t)ask.k && n0 + n >= (uint32_t)ask.k) {
            uint32_t cn = n0;
            double cm = m0;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (cn < (uint32_t)ask.k && cn + N[i] >= (uint32_t)ask.k) {
                    s.k_bin = tid * B + i;
                    s.k_above_n = cn;
                    s.k_here = N[i];
                    s.k_above = cm;
                    s.k_in = M[i];
                }
                cn += N[i];
                cm += M[i];
            }
        }
        __syncthreads();
        const uint32_t k_bin = ask.k > 0 ? s.k_bin : kBins;
        if (ask.p < 1.0f) {
            // what top_p is a share of is known to within the bin where top_k ends
            const double lo = (double)ask.p * (ask.k > 0 ? s.k_above : m_all), hi = (double)ask.p * (ask.k > 0 ? s.k_above + s.k_in : m_all);
            double cm = m0;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const double to = i + 1 < B ? cm + M[i] : m1;
                if (N[i] > 0 && to >= lo) atomicMin(&s.p_lo, (uint32_t)(tid * B + i));
                if (N[i] > 0 && to >= hi) atomicMin(&s.p_hi, (uint32_t)(tid * B + i));
                cm += M[i];
            }
            __syncthreads();
            const uint32_t p_lo = s.p_lo < k_bin ? s.p_lo : k_bin;
            cm = m0;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if ((uint32_t)(tid * B + i) == p_lo) s.p_above = cm;
                cm += M[i];
            }
        }
        __syncthreads();
        const uint32_t p_hi = ask.p < 1.0f ? (s.p_hi < k_bin ? s.p_hi : k_bin) : k_bin;
        const uint32_t p_lo = ask.p < 1.0f ? (s.p_lo < p_hi ? s.p_lo : p_hi) : k_bin;
        // a cut among what has no mass in the bins
        slow = p_hi >= kBins - 1 || k_bin == kBins - 1;
        if (!slow) {
            // what lies in the bins of a cut is listed, what lies above is added up, a run each
            const float p_from = (float)((int)p_lo - kAbove), p_to = (float)((int)p_hi - kAbove), k_at = (float)((int)k_bin - kAbove);
            double sum = 0.0;
            const bool all_above = !(mp > 0.0f);
            const float rate_hi = (float)(1.4426950408889634074 / ask.T), rate_lo = (float)(1.4426950408889634074 / ask.T - (double)rate_hi);
            auto mass = [&](float v) {
                const float d = v - best;
                const float t = d * rate_hi;
                const float e = __builtin_amdgcn_exp2f(t);
                return __builtin_fmaf(e, (__builtin_fmaf(d, rate_hi, -t) + d * rate_lo) * 0.693147180559945f, e);
            };
            auto pick = [&](float v, int c) {
                const float f = __builtin_floorf(place_of(v, ref, per_bin));
                if (f < p_from) {
                    if (all_above || (double)v - (double)best >= ask.limit) sum += (double)mass(v);
                } else if ((f <= p_to || f == k_at) && c < a.classes) {
                    const uint32_t at = atomicAdd(&s.listed, 1u);
                    if (at < kList) s.list.key[at] = (uint64_t)(~order_of(v)) << 32 | (uint32_t)c;
                }
            };
            __syncthreads();  // the bins make room for the list
            held(pick);
            rest(pick);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
            if (lane == 0) s.seg[wave] = sum;
            __syncthreads();
            const int n_list = (int)s.listed;
            slow = n_list > kList;
            if (!slow) {
                int n2 = 2;
                while (n2 < n_list) n2 *= 2;
                for (int i = n_list + tid; i < n2; i += T) s.list.key[i] = ~(uint64_t)0;
                __syncthreads();
                for (int size = 2; size <= n2; size *= 2)
                    for (int step = size / 2; step > 0; step /= 2) {
                        for (int i = tid; i < n2 / 2; i += T) {
                            const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                            const bool up = (lo & size) == 0;
                            const uint64_t p = s.list.key[lo], q = s.list.key[hi];
                            if ((p > q) == up) {
                                s.list.key[lo] = q;
                                s.list.key[hi] = p;
                            }
                        }
                        __syncthreads();
                    }
                // their masses' running sums
                constexpr int E = kList / T;
                double own[E], sum_e = 0.0;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int at = tid * E + i;
                    own[i] = 0.0;
                    if (at < n_list) {
                        const float v = of_order(~(uint32_t)(s.list.key[at] >> 32));
                        own[i] = exp2(((double)v - (double)ref) * (1.4426950408889634074 / ask.T));
                    }
                    sum_e += own[i];
                }
                uint32_t unused0, unused1;
                double e0, e1, e_all;
                block_scan<W>(0, sum_e, unused0, e0, e1, unused1, e_all, s);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    e0 += own[i];
                    if (tid * E + i < n_list) s.list.upto[tid * E + i] = e0;
                }
                if (tid == 0) s.first = n_list - 1;
                __syncthreads();
                int last = n_list - 1;  // the last that is kept
                double need = 0.0;
                if (ask.k > 0) {
                    const int before = n_list - (int)s.k_here;  // above the bin where top_k ends
                    const int k_last = before + (ask.k - (int)s.k_above_n) - 1;
                    need = (double)ask.p * (s.k_above + s.list.upto[k_last] - (before > 0 ? s.list.upto[before - 1] : 0.0));
                    last = k_last;
                } else {
                    need = (double)ask.p * m_all;
                }
                if (ask.p < 1.0f) {
                    const int end = ask.k > 0 && k_bin > p_hi ? n_list - (int)s.k_here - 1 : last;
                    for (int i = tid; i <= end; i += T)
                        if (s.p_above + s.list.upto[i] >= need) {
                            atomicMin(&s.first, i);
                            break;
                        }
                    __syncthreads();
                    last = s.first < end ? s.first : end;
                }
                if (tid == 0) s.cut = s.list.key[last];
                // the kept of the list join their runs
                const int per = (n_list + 63) / 64;
                double add = 0.0;
                for (int i = lane * per; i < lane * per + per && i <= last; ++i) {
                    const uint64_t k = s.list.key[i];
                    const int c = (int)(uint32_t)k;
                    if (c / run != wave) continue;
                    const float v = of_order(~(uint32_t)(k >> 32));
                    if (all_above || (double)v - (double)best >= ask.limit) add += (double)mass(v);
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) add += __shfl_xor(add, o);
                if (lane == 0) s.seg[wave] += add;
                __syncthreads();
            }
        }
    } else if (!slow) {
        // nothing but min_p: every class counts
        const float rate_hi = (float)(1.4426950408889634074 / ask.T), rate_lo = (float)(1.4426950408889634074 / ask.T - (double)rate_hi);
        double sum = 0.0;
        auto add = [&](float v, int) {
            if (!((double)v - (double)best >= ask.limit)) return;
            const float d = v - best;
            const float t = d * rate_hi;
            if (!(t > -150.0f)) return;
            const float e = __builtin_amdgcn_exp2f(t);
            sum += (double)__builtin_fmaf(e, (__builtin_fmaf(d, rate_hi, -t) + d * rate_lo) * 0.693147180559945f, e);
        };
        held(add);
        rest(add);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) s.seg[wave] = sum;
        if (tid == 0) s.cut = ~(uint64_t)0;
        __syncthreads();
    }
    if (slow) {
        __syncthreads();
        slow_row<T>(x, a.classes, a.shift, a.tokens + r, a.logprob ? a.logprob + r : nullptr, best, ask, lds.s);
        return;
    }
    // the run where the running sum passes u of the total, and in it the class
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < W; ++i) total += s.seg[i];
    const double goal = (double)ask.u * total;
    double before = 0.0, from = 0.0;
    int seg = -1;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const double to = before + s.seg[i];
        if (s.seg[i] > 0.0 && (seg < 0 || from + s.seg[seg] <= goal)) {
            seg = i;
            from = before;
        }
        before = to;
    }
    const uint64_t cut = s.cut;
    if (tid == 0) {
        s.first = 0x7fffffff;
        s.last = -1;
    }
    const float rate_hi = (float)(1.4426950408889634074 / ask.T), rate_lo = (float)(1.4426950408889634074 / ask.T - (double)rate_hi);
    // parts of the run in turn, 4 classes a thread
    for (int p0 = seg * run; p0 < (seg + 1) * run; p0 += 4 * T) {
        const int c = p0 + 4 * tid;
        const vf4 v = logits(row, c < (seg + 1) * run ? c : a.classes);
        double w[4], own = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t k = (uint64_t)(~order_of(v[j])) << 32 | (uint32_t)(c + j);
            const float d = v[j] - best;
            const float t = d * rate_hi;
            w[j] = 0.0;
            if (c < (seg + 1) * run && c + j < a.classes && k <= cut && (double)v[j] - (double)best >= ask.limit && t > -150.0f) {
                const float e = __builtin_amdgcn_exp2f(t);
                w[j] = (double)__builtin_fmaf(e, (__builtin_fmaf(d, rate_hi, -t) + d * rate_lo) * 0.693147180559945f, e);
            }
            own += w[j];
        }
        uint32_t unused0, unused1;
        double w0, w1, w_all;
        block_scan<W>(0, own, unused0, w0, w1, unused1, w_all, s);
        double upto = from + w0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            upto += w[j];
            if (w[j] > 0.0) {
                if (upto > goal) atomicMin(&s.first, c + j);
                atomicMax(&s.last, c + j);
            }
        }
        __syncthreads();
        if (s.first != 0x7fffffff) break;
        from += w_all;
    }
    // a sum that rounding left short of the goal ends at the run's last
    __syncthreads();
    if (tid == 0) {
        const int at = s.first != 0x7fffffff ? s.first : s.last;
        a.tokens[r] = at;
        if (a.logprob) a.logprob[r] = share_log(x[at], best, ask.T, total);
    }
}

// A workgroup a row; several launches for more rows than a dispatch holds.
template <int T, int Q>
void launch_sample(SampleArg a, int64_t rows) {
    for (a.row0 = 0; a.row0 < rows; a.row0 += max_grid_blocks(T)) {
        const int64_t blocks = rows - a.row0 < max_grid_blocks(T) ? rows - a.row0 : max_grid_blocks(T);
        hipLaunchKernelGGL((k_sample<T, Q>), dim3((unsigned)blocks), dim3(T), 0, ctx().stream, a);
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
    a.classes = (int32_t)classes;
    a.shift = 62;
    while (((int64_t)1 << (62 - a.shift)) < classes) --a.shift;
    launch_sample<1024, 16>(a, rows);
    return finish("mh_sample_tokens");
}

}  // extern "C"
