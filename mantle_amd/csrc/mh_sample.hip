// mh_sample.hip -- a token for each row of logits from a uniform number, after temperature, top-k, top-p and min-p.
//
// What top-k, top-p and min-p keep is a beginning of the row in the order of falling logits, ties by index: it ends at one
// class, the cut. The token is the first class, by index, where the running sum of the kept masses e^((x - max) / T) exceeds u
// of their sum.
//
// A workgroup takes a row (64 threads of a short one where there are many, up to 1024), a wavefront a run of its classes,
// of which each lane holds 4 Q logits in registers (the whole row up to 4 Q T classes; of a longer one the rest is read
// as it is needed):
//   1. the largest logit held, the reference, and bins of a power-of-two width, T / 112 or 1 / 112 at least, around it;
//   2. for top-k and top-p how many classes each bin has and their mass, both in one 64-bit LDS atomic: 20 bits of count above
//      44 of mass, a class 24 bits of its bin's largest. Whole numbers: the atomics' order does not show. A scan of the bins
//      then says in which of them a cut falls;
//   3. a second walk, over the quads that reach those bins, adds up what lies above them and lists what lies in them. More
//      listed than there is room: from 2. on with narrower bins in the place of those;
//   4. the list is sorted, up to 512 keys by counting what comes before each (128 keys by the 28 steps of a sorting network,
//      each waiting for the last, take 11700 cycles; [33, 30011] takes 26.7 us instead of 29.9), and the cuts are found in
//      it by 64-bit sums;
//   5. the run of classes where the running sum passes u of the total is walked by the whole workgroup.
// Sums of steps 3 to 5 are 64-bit floats in a fixed order, of quads, which are added in fp32. Masses are fp32 too, for a walk is bound
// by its instructions: a class' is off by 2^-24 of itself for each T below the largest (the difference's rounding), three for the
// exponential and three for the quad's sum. That moves a border by as much as what is kept is off by together, where it has a common
// sign.
//
// Rows for which bins do not work (more than 256 to 2048 classes of one value at a cut, a cut 32 T below the largest, an
// infinite logit, temperatures outside 0.01 to 1e30, more than 2^19 classes) go by whole-number masses and a search over
// the logits' bits, 8 at a time: right for every row, and slower.
//
// The slowest row decides. Over [512, 131072] with settings of all kinds the call takes 124 us, where reading takes 41: two
// workgroups a CU, and of a row at a temperature of 1 or more, whose cut lies in the bulk, 80 thousand cycles of 280 are the
// counting (one LDS atomic and 20 instructions a class) and 83 the second walk (20 instructions a class). A single row of
// 32000 takes 18.5 us: some 42 thousand cycles, of which 13 count and 5 walk again, and the rest are short phases that each wait
// for a fetch, a barrier or 64-bit exponentials. Of Q 4 was taken (8 of 512 threads): 16 hold more of a row, and cost the
// short phases registers and code: [33, 30011] 26.8 us with 16, 24.8 to 25.5 with 4; [512, 131072] with 512 threads 124 with 8, 128 with 4.
#include "mh_internal.h"
#include "mh_rows.h"

namespace mh {
namespace {

// The most classes that bins count: a bin's count and mass share 64 bits.
constexpr int64_t kMaxBinned = (int64_t)1 << 19;
constexpr int kCountAt = 44;  // the first bit of the count
static_assert(kMaxBinned < (int64_t)1 << (64 - kCountAt) && kMaxBinned << 24 <= (int64_t)1 << (kCountAt - 1), "a bin holds every class");
// By the threads T of a workgroup: the bins, those of them above the reference at first, the classes a list holds, and
// those whose quads' largest logits are kept. Bins below the reference reach 32 T at least, whatever their power of two.
template <int T>
struct Sizes {
    static constexpr int kBins = T >= 512 ? 4096 : 8 * T, kAbove = kBins / 8, kList = kBins / 2, kTops = T >= 512 ? (int)kMaxBinned : 128 * T;
    static constexpr float kWidth = 1.0f / (T >= 512 ? 112 : T / 5);  // of T, at least
    static_assert(kTops <= kMaxBinned, "");
};
constexpr int kRanked = 512;  // the longest list that is sorted by ranks
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
    int32_t shift;  // of the whole-number masses: 2^shift for the largest, room for all of up to kMaxBinned classes
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

// Lanes' values moved within the wavefront; 0 where there is none to move (its bits are 0 in every type).
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) { return (uint32_t)moved<CTRL, ROWS>((int)v); }
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T moved(T v) {
    static_assert(sizeof(T) == 8, "");
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t m = (uint64_t)(uint32_t)moved<CTRL, ROWS>((int)(b >> 32)) << 32 | (uint32_t)moved<CTRL, ROWS>((int)b);
    return __builtin_bit_cast(T, m);
}
// Sums up to and with each lane of a row of 16 lanes, and of the wavefront.
template <typename T>
__device__ __forceinline__ T row_scan(T v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v = row_scan(v);
    v += moved<0x142, 0xa>(v);  // each row's last lane to the row behind it
    v += moved<0x143, 0xc>(v);  // the lower half's last lane to the upper half
    return v;
}
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                         (uint32_t)__builtin_amdgcn_readlane((int)b, lane));
    }
}
// The largest of a wavefront's numbers, in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_with(float v) {
    return __builtin_fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = max_with<0x111, 0xf>(v);
    v = max_with<0x112, 0xf>(v);
    v = max_with<0x114, 0xf>(v);
    v = max_with<0x118, 0xf>(v);
    v = max_with<0x142, 0xa>(v);
    v = max_with<0x143, 0xc>(v);
    return lane_value(v, 63);
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
__device__ __forceinline__ double scaled_mass(float x, const Heat& h) {
    if (x == h.top) return __builtin_ldexp(1.0, h.shift);
    const float d = x - h.top;
    const float t = d * h.hi;
    if (!(t > -63.0f)) return 0.0;
    const float n = __builtin_rintf(t);
    const float r = __builtin_fmaf(d, h.hi, -n) + d * h.lo;
    return __builtin_ldexp((double)__builtin_amdgcn_exp2f(r), (int)n + h.shift);
}
__device__ __forceinline__ uint64_t mass_of(float x, const Heat& h) { return (uint64_t)(scaled_mass(x, h) + 0.5); }

struct Threshold {
    uint32_t key;   // the value's order
    uint64_t ties;  // how many classes of it count
};

struct SlowLds {
    unsigned long long hist_m[256], said[4], seg_m[16];
    uint32_t hist_n[256], seg_n[16];
    double sum_d[16];
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
    // Room for every class at the largest's mass rounds n of them by n^2 2^-63 of it at most, 2^-25 over 2^19; more have room for what
    // they add up to, which they round by n 2^-63 of itself.
    if (classes > kMaxBinned) {
        h.shift = 0;
        double m = 0.0;
        for (int c = tid; c < classes; c += T) m += scaled_mass(x[c], h);
        h.shift = 62 - __builtin_amdgcn_frexp_exp(block_sum<W>(m, s.sum_d));
    }
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
                if (logprob) *logprob = share_log(v, best, ask.T, __builtin_ldexp((double)total, -h.shift));
            }
            break;
        }
        before += lane_value(upto, 63);
        ties_before += lane_value(at_tie, 63);
    }
}

// ---------------------------------------------------------------------------------------
// rows that bins sort out
// ---------------------------------------------------------------------------------------
// The least logit that `is` holds for; it holds for every larger one, infinity too. 64 at a time are looked at, 6 bits of
// their order. By whole wavefronts.
template <typename F>
__device__ __forceinline__ float least_of(F&& is) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t key = 0;  // the largest known for which it does not hold: a NaN's
#pragma unroll
    for (int place = 26; place >= -4; place -= 6) {
        const int p = place < 0 ? 0 : place;
        const uint32_t k = key + ((place < 0 ? lane & 3 : lane) << p);
        const bool no = k <= 0xff800000u && !is(of_order(k));
        key += (uint32_t)(__builtin_popcountll(__ballot(no && (place >= 0 || lane < 4))) - 1) << p;
    }
    return of_order(key + 1);
}

// What is known at once of a workgroup's sums.
struct Sums {
    double wave_d[16];
    uint32_t wave_n[16];
};
template <int T>
struct FastLds : Sums {
    union {
        unsigned long long hist[Sizes<T>::kBins];
        struct {
            uint64_t key[Sizes<T>::kList];  // order inverted, then the index: rising is the order that is kept
            double upto[Sizes<T>::kList];   // sums of masses
        } list;
    };
    float quad_top[Sizes<T>::kTops / 256];  // the largest of 256 classes
    double seg[16];
    float wave_f[16];
    // what one thread found out for all
    uint32_t listed, k_bin, k_above_n, k_here, p_lo, p_hi, p_above_n;
    double k_above, k_in, p_above;
    int bad, first, token;
};

// Exclusive sums over the workgroup's threads of a count and a mass, and the totals; m1 is the sum with the thread's own, the
// same bits as the next thread's m0. A sum over lanes is added in an order of its own for each, so the masses' need not
// rise.
template <int W>
__device__ __forceinline__ void block_scan(uint32_t n, double m, uint32_t& n0, double& m0, double& m1, uint32_t& n_all, double& m_all,
                                           Sums& s) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t ni = wave_scan(n);
    const double mi = wave_scan(m);
    __syncthreads();
    if (lane == 63) {
        s.wave_n[wave] = ni;
        s.wave_d[wave] = mi;
    }
    __syncthreads();
    const uint32_t nw = row_scan(lane < W ? s.wave_n[lane & 15] : 0u);
    const double mw = row_scan(lane < W ? s.wave_d[lane & 15] : 0.0);
    n_all = lane_value(nw, W - 1);
    m_all = lane_value(mw, W - 1);
    const uint32_t nb = wave ? lane_value(nw, wave - 1) : 0;
    const double mb = wave ? lane_value(mw, wave - 1) : 0.0;
    const double mp = moved<0x138, 0xf>(mi);  // the lane's before
    n0 = nb + ni - n;
    m0 = mb + mp;
    m1 = lane < 63 ? mb + mi : lane_value(mw, wave);
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

// What one class's mass is made from, in units of the largest's.
struct Mass {
    float best, hi, lo;  // the largest logit; log2(e) / T in two parts
    float least;         // the least logit that min_p keeps
    __device__ __forceinline__ Mass(float top, const Ask& ask) : best(top) {
        const double per = 1.4426950408889634074 / ask.T;
        hi = (float)per;
        lo = (float)(per - (double)hi);
        const double edge = (double)top + ask.limit;
        least = (float)edge;
        if ((double)least < edge) {  // the next one up
            const uint32_t b = __float_as_uint(least + 0.0f);
            least = __uint_as_float(b >> 31 ? b - 1 : b + 1);
        }
    }
    __device__ __forceinline__ float raw(float v) const {  // of a finite logit
        const float d = v - best;
        const float t = d * hi;
        const float e = __builtin_amdgcn_exp2f(t);
        return __builtin_fmaf(e, __builtin_fmaf(d, lo, __builtin_fmaf(d, hi, -t)) * 0.693147180559945f, e);
    }
    __device__ __forceinline__ float operator()(float v) const { return v >= least && (v - best) * hi > -150.0f ? raw(v) : 0.0f; }
};

template <int T, int Q>
__global__ __launch_bounds__(T, T == 256 ? 5 : 4) void k_sample(SampleArg a) {
    constexpr int W = T / 64;
    constexpr int kBins = Sizes<T>::kBins, kAbove = Sizes<T>::kAbove, kList = Sizes<T>::kList;
    constexpr int B = kBins / T;  // bins of a thread
    __shared__ union Lds {
        FastLds<T> f;
        SlowLds s;
        __device__ Lds() {}
    } lds;
    FastLds<T>& s = lds.f;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // a wavefront's run of classes: whole rounds of 256, of which the first Q are held
    const int run = (a.classes + 256 * W - 1) / (256 * W) * 256;
    const int w0 = wave * run, c0 = w0 + 4 * lane;
    const int quads = run / 256;
    const int64_t r = a.row0 + blockIdx.x;
    const float* x = a.x + r * a.classes;
    const Row row = row_of(x, a.classes);
    vf4 h[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) h[i] = logits(row, i < quads ? c0 + 256 * i : a.classes);
    // the settings: addresses that are there in any case, so that all are on their way at once
    float T_ = (a.temperature ? a.temperature : a.u)[r], mp = (a.min_p ? a.min_p : a.u)[r];
    Ask ask;
    ask.k = (a.top_k ? a.top_k : reinterpret_cast<const int32_t*>(a.u))[r];
    ask.p = (a.top_p ? a.top_p : a.u)[r];
    ask.u = a.u[r];
    T_ = a.temperature ? T_ : 1.0f;
    mp = a.min_p ? mp : 0.0f;
    ask.T = (double)T_;
    ask.k = a.top_k ? ask.k : 0;
    ask.p = a.top_p && ask.p < 1.0f ? ask.p : 1.0f;
    if (ask.p <= 0.0f) ask.k = 1, ask.p = 1.0f;  // the likeliest alone
    if (ask.k < 0 || ask.k >= a.classes) ask.k = 0;
    ask.limit = -__builtin_inf();
    if (mp > 0.0f) ask.limit = mp >= 1.0f ? 0.0 : log((double)mp) * ask.T;
    ask.u = ask.u > 0.0f ? (ask.u < 1.0f ? ask.u : 0.999999940395355f) : 0.0f;
    const bool greedy = !(T_ > 0.0f);
    const bool cuts = !greedy && (ask.k > 0 || ask.p < 1.0f);
    // the logits held: four at a time, or all of them at once need more registers than there are
    auto held = [&](auto&& f) {
        int at = c0;
        asm volatile("" : "+v"(at));  // or every walk shares the registers of all indices
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if (i < quads) {
                f(h[i], at + 256 * i, i);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    // quads of the run from memory: those of the 64 from `g` on that `which` has a bit for
    auto walk = [&](auto&& which, auto&& f) {
        for (int g = 0; g < quads; g += 64) {
            uint64_t m = which(g);
            m &= quads - g >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << (quads - g)) - 1;
            auto take = [&](int& i) {
                i = m ? g + __builtin_ctzll(m) : -1;
                m &= m - 1;
                return logits(row, i >= 0 ? c0 + 256 * i : a.classes);
            };
            int i0, i1, i2;
            vf4 v0 = take(i0), v1 = take(i1);
            while (i0 >= 0) {
                vf4 v = v0;
                const int i = i0;
                v0 = v1;
                i0 = i1;
                v1 = take(i2);
                i1 = i2;
                if (w0 + 256 * (i + 1) > a.classes) close_row(v, c0 + 256 * i, a.classes);
                f(v, c0 + 256 * i, i);
            }
        }
    };
    auto all = [](int) { return ~(uint64_t)0; };
    auto others = [](int g) { return g ? ~(uint64_t)0 : ~(uint64_t)0 << Q; };
    float top = -__builtin_inff();  // of what the wavefront has seen
    bool nan = false;
    const bool tops = a.classes <= Sizes<T>::kTops;
    auto look = [&](const vf4& v, int i) {
        nan |= __builtin_isunordered(v.x, v.y) | __builtin_isunordered(v.z, v.w);
        const float q = wave_max(__builtin_fmaxf(__builtin_fmaxf(v.x, v.y), __builtin_fmaxf(v.z, v.w)));
        top = __builtin_fmaxf(top, q);
        if (tops && lane == 0) s.quad_top[wave * quads + i] = q;
    };
    // the quads that reach a logit
    auto reach = [&](float v) {
        return [=, &s](int g) { return tops ? __ballot(s.quad_top[wave * quads + (g + lane < quads ? g + lane : 0)] >= v) : ~(uint64_t)0; };
    };
    auto block_top = [&]() {
        __syncthreads();
        if (lane == 0) s.wave_f[wave] = top;
        __syncthreads();
        return wave_max(s.wave_f[lane % W]);
    };
    // the largest logit held
#pragma unroll
    for (int i = 0; i < Q; ++i)
        if (w0 + 256 * (i + 1) > a.classes || i >= quads) close_row(h[i], i < quads ? c0 + 256 * i : a.classes, a.classes);
    held([&](const vf4& v, int, int i) { look(v, i); });
    if (tid == 0) {
        s.bad = 0;
        s.first = 0x7fffffff;
    }
    float best = block_top();
    float ref = best;
    // masses are e^((x - ref) / T) until the largest is known
    bool binned = cuts && tops && ref > -__builtin_inff() && ref < __builtin_inff() && T_ >= 0.01f && T_ <= 1e30f;
    // the bins: bin b holds what lies from b + start widths below ref on, a whole number of them. Every step there is exact
    // near the bins, so that narrower ones divide those before them, also where they begin above ref.
    float per_bin, start = -(float)kAbove;
    double width;
    {
        const int e = __builtin_amdgcn_frexp_expf(__builtin_fmaxf(T_, 1.0f) * Sizes<T>::kWidth);
        per_bin = __builtin_ldexpf(1.0f, -e);
        width = __builtin_ldexp(1.0, e);
    }
    auto bin_at = [&](float below) { return (int)__builtin_fminf(below - start, 1e6f); };  // of whole widths below ref
    uint32_t base_n = 0;  // what lies above the bins
    double base_m = 0.0, all_m = 0.0;
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < B; ++i) s.hist[i * T + tid] = 0;
        if (tid == 0) {
            s.listed = 0;
            s.k_bin = s.p_lo = s.p_hi = kBins;
        }
    };
    auto count = [&](const vf4& v) {
        const float neg = -(float)(width / ask.T * 1.4426950408889634074);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float q = (ref - v[j]) * per_bin;
            const float f = __builtin_floorf(q);
            const int b = bin_at(f);
            uint32_t m = 0;
            if (ask.p < 1.0f) m = (uint32_t)__builtin_fmaf(__builtin_amdgcn_exp2f((q - f) * neg), 16777216.0f, 0.5f);
            if ((uint32_t)b < (uint32_t)kBins) atomicAdd(&s.hist[b], (unsigned long long)1 << kCountAt | m);
        }
    };
    if (binned) {
        clear();
        __syncthreads();
        held([&](const vf4& v, int, int) { count(v); });
        walk(others, [&](const vf4& v, int, int i) {
            look(v, i);
            count(v);
        });
    } else if (quads > Q) {
        walk(others, [&](const vf4& v, int, int i) { look(v, i); });
    }
    if (nan) s.bad = 1;
    if (quads > Q || binned) best = block_top();
    else __syncthreads();
    const bool none = s.bad != 0 || best == -__builtin_inff();
    if (none || greedy) {  // the lowest index of the largest
        int at = 0x7fffffff;
        if (!none && top == best)
            walk(reach(best), [&](const vf4& v, int c, int) {
#pragma unroll
                for (int j = 0; j < 4; ++j) at = v[j] == best && c + j < at ? c + j : at;
            });
        if (at != 0x7fffffff) atomicMin(&s.first, at);
        __syncthreads();
        if (tid == 0) {
            a.tokens[r] = none ? -1 : s.first;
            if (a.logprob) a.logprob[r] = none ? __builtin_nanf("") : 0.0f;
        }
        return;
    }
    const Mass mass(best, ask);
    bool slow = (cuts && !binned) || best == __builtin_inff() || !(T_ >= 1e-30f && T_ <= 1e30f);
    // one of the others lies above the bins, or so far above ref that e^((best - ref) / T) is near a double's largest: at T =
    // 0.01 the bins reach 800 T above it, and exp64 700, of which a thread's first bin may take 87
    if (!slow && cuts && ((best - ref) * per_bin >= (float)kAbove || best - ref > 600.0f * T_)) {
        __syncthreads();
        clear();
        __syncthreads();
        ref = best;
        walk(all, [&](const vf4& v, int, int) { count(v); });
        __syncthreads();
    }
    uint64_t cut = ~(uint64_t)0;  // the last class that is kept, as the list's keys
    for (int turn = 0; !slow && cuts; ++turn) {
        // the bins' counts and masses, from the top down: each thread's B, then all before it
        const double rate = width / ask.T;
        // of a count of 1 at the top of the thread's first bin the mass, and what the next bin has of it
        double unit = 0.0, fall = 0.0;
        auto bin_mass = [&](uint64_t v, double e) { return v ? (double)(v & (((uint64_t)1 << kCountAt) - 1)) * e : 0.0; };
        uint32_t n = 0;
        double m = 0.0, each_m;
#pragma unroll
        for (int b = 0; b < B; ++b) n += (uint32_t)(s.hist[tid * B + b] >> kCountAt);
        if (n) {
            each_m = unit = exp64(-rate * ((double)start + (double)(tid * B))) * (1.0 / 16777216.0);
            fall = exp64(-rate);
#pragma nounroll
            for (int b = tid * B; b < tid * B + B; ++b, each_m *= fall) m += bin_mass(s.hist[b], each_m);
        }
        uint32_t n0, n_bins;
        double m0, m1, m_bins;
        block_scan<W>(n, m, n0, m0, m1, n_bins, m_bins, s);
        n0 += base_n;
        if (turn == 0) all_m = m_bins;
        // a cut lies in the bin whose sums pass it; where rounding lets none the row goes the slow way
        if (ask.k > 0 && n0 < (uint32_t)ask.k && n0 + n >= (uint32_t)ask.k) {
            uint32_t cn = n0;
            double cm = m0;
            each_m = unit;
#pragma nounroll
            for (int b = tid * B; b < tid * B + B; ++b, each_m *= fall) {
                const uint64_t v = s.hist[b];
                const uint32_t here = (uint32_t)(v >> kCountAt);
                const double in = bin_mass(v, each_m);
                if (cn + here >= (uint32_t)ask.k) {
                    s.k_bin = b;
                    s.k_above_n = cn;
                    s.k_here = here;
                    s.k_above = base_m + cm;
                    s.k_in = in;
                    break;
                }
                cn += here;
                cm += in;
            }
        }
        int p_bin = -1;  // where the thread finds top_p's border, and what lies above
        double p_above = 0.0;
        uint32_t p_above_n = 0;
        if (ask.p < 1.0f) {
            if (ask.k > 0) __syncthreads();
            // what top_p is a share of is known to within the bin where top_k ends
            const double hi = (double)ask.p * (ask.k > 0 ? s.k_above + s.k_in : all_m) - base_m;
            double lo = ask.k > 0 ? (double)ask.p * s.k_above - base_m : hi;
            lo = lo > 0.0 ? lo : 1e-300;
            // Sums round: they need not rise from thread to thread, nor m1 be what the thread's bins add up to. Of several threads
            // that find the border the first has it; a bin of none has none.
            if ((m0 < lo && m1 >= lo) || (m0 < hi && m1 >= hi)) {
                uint32_t cn = n0;
                double cm = m0;
                each_m = unit;
#pragma nounroll
                for (int b = tid * B; b < tid * B + B; ++b, each_m *= fall) {
                    const uint64_t v = s.hist[b];
                    const double to = b + 1 < tid * B + B ? cm + bin_mass(v, each_m) : m1;
                    if (v && cm < lo && to >= lo) {
                        p_bin = b;
                        p_above = base_m + cm;
                        p_above_n = cn;
                        atomicMin(&s.p_lo, (uint32_t)b);
                    }
                    if (ask.k > 0 && v && cm < hi && to >= hi) atomicMin(&s.p_hi, (uint32_t)b);
                    cn += (uint32_t)(v >> kCountAt);
                    cm = to;
                }
            }
        }
        __syncthreads();
        if (p_bin == (int)s.p_lo) {  // read behind the next barrier
            s.p_above = p_above;
            s.p_above_n = p_above_n;
        }
        const int k_bin = ask.k > 0 ? (int)s.k_bin : kBins;
        int p_lo = k_bin, p_hi = k_bin;
        if (ask.p < 1.0f) {
            p_lo = (int)s.p_lo;
            p_hi = ask.k == 0 ? p_lo : (int)s.p_hi < k_bin ? (int)s.p_hi : k_bin;
        }
        const int most = k_bin < kBins ? k_bin : p_hi;  // the last bin that is listed
        slow = p_lo > p_hi || most >= kBins || (ask.k > 0 && k_bin == kBins);
        if (slow) break;
        // what lies in the bins of a cut is listed, what lies above is added up, a run each
        auto bin_of = [&](float v) { return bin_at(__builtin_floorf((ref - v) * per_bin)); };
        const float v_list = least_of([&](float v) { return bin_of(v) <= most; });
        const float v_keep = least_of([&](float v) { return bin_of(v) < p_lo; });
        // no mass below e^-100 of the largest's; what min_p drops has none
        const float v_sum = __builtin_fmaxf(__builtin_fmaxf(v_keep, mass.least), (float)((double)best - 100.0 * ask.T));
        double sum = 0.0;
        __syncthreads();  // the bins make room for the list
        walk(
            reach(v_list),
            [&](const vf4& v, int c, int) {
                float q = 0.0f;
                bool some = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float e = mass.raw(v[j]);
                    q += v[j] >= v_sum ? e : 0.0f;
                    some |= v[j] >= v_list && !(v[j] >= v_keep);
                }
                sum += (double)q;
                if (some) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int b = bin_of(v[j]);
                        if (b < p_lo || (b > p_hi && b != k_bin)) continue;
                        const uint32_t at = atomicAdd(&s.listed, 1u);
                        if (at < kList) s.list.key[at] = (uint64_t)(~order_of(v[j])) << 32 | (uint32_t)(c + j);
                    }
                }
            });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) s.seg[wave] = sum;
        __syncthreads();
        const int n_list = (int)s.listed;
        if (n_list > kList) {
            // the bins of the cuts alone, as narrow as that makes them
            const int e = __builtin_amdgcn_frexp_expf((float)(most + 1 - p_lo) * (1.0f / kBins));
            slow = turn == 2 || e >= 0;
            if (slow) break;
            if (ask.p < 1.0f) {
                base_n = s.p_above_n;
                base_m = s.p_above;
            } else {
                base_n = s.k_above_n;
                base_m = s.k_above;
            }
            start = __builtin_ldexpf(start + (float)p_lo, -e);
            width = __builtin_ldexp(width, e);
            per_bin = __builtin_ldexpf(per_bin, -e);
            __syncthreads();
            clear();
            __syncthreads();
            walk(all, [&](const vf4& v, int, int) { count(v); });
            __syncthreads();
            continue;
        }
        if (n_list <= kRanked) {
            // each key's place is how many come before it: no step waits for another
            const int n8 = (n_list + 7) & ~7;
            for (int i = n_list + tid; i < n8; i += T) s.list.key[i] = ~(uint64_t)0;
            __syncthreads();
            for (int i = tid; i < n_list; i += T) {
                const uint64_t k = s.list.key[i];
                int at = 0;
#pragma unroll 8
                for (int o = 0; o < n8; ++o) at += s.list.key[o] < k;
                s.list.upto[at] = __longlong_as_double((long long)k);
            }
            __syncthreads();
            for (int i = tid; i < n_list; i += T) s.list.key[i] = (uint64_t)__double_as_longlong(s.list.upto[i]);
            __syncthreads();
        } else {
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
        }
        // their masses' running sums
        const int per = (n_list + T - 1) / T, i0 = tid * per, i1 = i0 + per < n_list ? i0 + per : n_list;
        auto in_bins = [&](int i) {  // as the bins have it
            return exp64(((double)of_order(~(uint32_t)(s.list.key[i] >> 32)) - (double)ref) / ask.T);
        };
        double own = 0.0;
#pragma nounroll
        for (int i = i0; i < i1; ++i) own += in_bins(i);
        uint32_t unused0, unused1;
        double e0, e1, e_all;
        block_scan<W>(0, own, unused0, e0, e1, unused1, e_all, s);
#pragma nounroll
        for (int i = i0; i < i1; ++i) s.list.upto[i] = e0 += in_bins(i);
        __syncthreads();
        int last = n_list - 1;  // the last that is kept
        double share = all_m;   // what top_p is a share of
        int end = last;         // of top_p's part of the list
        if (ask.k > 0) {
            const int before = n_list - (int)s.k_here;  // above the bin where top_k ends
            last = before + (ask.k - (int)s.k_above_n) - 1;
            share = s.k_above + s.list.upto[last] - (before > 0 ? s.list.upto[before - 1] : 0.0);
            end = k_bin > p_hi ? before - 1 : last;
        }
        if (ask.p < 1.0f) {
            const double least = (double)ask.p * share - s.p_above;
            for (int i = tid; i < end; i += T)
                if (s.list.upto[i] >= least && (i == 0 || s.list.upto[i - 1] < least)) atomicMin(&s.first, i);  // where sums fall again, the first
            __syncthreads();
            last = s.first < end ? s.first : end;
        }
        cut = s.list.key[last];
        // the kept of the list join their runs
        const int each = (n_list + 63) / 64;
        double add = 0.0;
        for (int i = lane * each; i < lane * each + each && i <= last; ++i) {
            const uint64_t k = s.list.key[i];
            const int c = (int)(uint32_t)k;
            if (c >= w0 && c < w0 + run) add += (double)mass(of_order(~(uint32_t)(k >> 32)));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) add += __shfl_xor(add, o);
        if (lane == 0) s.seg[wave] += add;
        __syncthreads();
        break;
    }
    if (!slow && !cuts) {  // nothing but min_p: every class counts
        double sum = 0.0;
        walk(reach(mass.least), [&](const vf4& v, int, int) {
            float q = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) q += mass(v[j]);
            sum += (double)q;
        });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) s.seg[wave] = sum;
        __syncthreads();
    }
    if (slow) {
        __syncthreads();
        slow_row<T>(x, a.classes, a.shift, a.tokens + r, a.logprob ? a.logprob + r : nullptr, best, ask, lds.s);
        return;
    }
    // The run where the running sum passes u of the total, and in it the class. Sums round, by the order that a scan adds them
    // in: where one begins need not be where the one before it ends, and what passes the goal may hold nothing. So the last run with any
    // mass that begins at the goal or before it is taken, of it the last such thread, and there is one of either.
    const double segs = row_scan(lane < W ? s.seg[lane & 15] : 0.0);
    const double total = lane_value(segs, W - 1), goal = (double)ask.u * total;
    const double ahead = moved<0x138, 0xf>(segs);
    const int seg = 63 - __builtin_clzll(__ballot(lane < W && s.seg[lane & 15] > 0.0 && ahead <= goal));
    double from = seg > 0 ? lane_value(segs, seg - 1) : 0.0;
    if (tid == 0) {
        s.first = -1;
        s.token = 0;
    }
    // the run in parts, each thread its own neighbouring quads of a part
    constexpr int P = Q < 8 ? Q : 8;
    const int stop = (seg + 1) * run < a.classes ? (seg + 1) * run : a.classes;
    for (int p0 = seg * run, id = tid; p0 < stop; p0 += 4 * P * T, id += T) {
        const int each = (stop - p0 + 4 * T - 1) / (4 * T) < P ? (stop - p0 + 4 * T - 1) / (4 * T) : P;
        const int c = p0 + 4 * each * tid;
        vf4 v[P];
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = logits(row, i < each ? c + 4 * i : a.classes);
        double own[P], m = 0.0;
        auto kept = [&](float x, int c) {
            const uint64_t k = (uint64_t)(~order_of(x)) << 32 | (uint32_t)c;
            return c < stop && k <= cut ? mass(x) : 0.0f;
        };
#pragma unroll
        for (int i = 0; i < P; ++i) {
            own[i] = 0.0;
            if (i < each) {
                float q = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) q += kept(v[i][j], c + 4 * i + j);
                own[i] = (double)q;
            }
            m += own[i];
        }
        uint32_t unused0, unused1;
        double m0, m1, part;
        block_scan<W>(0, m, unused0, m0, m1, unused1, part, s);
        const uint64_t begins = __ballot(m > 0.0 && from + m0 <= goal);
        if (begins && lane == 63 - __builtin_clzll(begins)) atomicMax(&s.first, id);
        __syncthreads();
        if (s.first == id) {
            // the quad, the first that passes the goal or else the last with any mass, and in it the class
            double upto = from + m0, to = upto;
            int at = c;
            vf4 quad = v[0];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (own[i] > 0.0 && to <= goal) {
                    upto = to;
                    at = c + 4 * i;
                    quad = v[i];
                }
                to += own[i];
            }
            int found = -1;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = kept(quad[j], at + j);
                if (e > 0.0f && (found < 0 || upto + (double)sum <= goal)) found = at + j;
                sum += e;
            }
            s.token = found;
        }
        from += part;
        if (goal < from) break;
    }
    __syncthreads();
    if (tid == 0) {
        const int at = s.token;
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

// Threads a row, by the microseconds of a row alone and of each row more that a CU has to take, with c thousand classes: of the
// slowest of rows with settings of all kinds, which a batch waits for. [4096, 500]: 21, 46, 107, 195 us with 64 to 1024 threads;
// [1024, 8000]: 79, 31, 43, 63; [512, 32000]: 58, 43, 50 with 256 to 1024; [128, 32000]: 51, 32, 28; [128, 500] 14.5, 14.5, 16, 16.
// (Many a row alone is not that slow, and has the same order: [1, 32000] 28, 18, 16.)
int sample_threads(int64_t rows, int64_t classes) {
    struct Form {
        int threads;
        double alone, alone_c, more, more_c;
        int64_t most;
    };
    const Form forms[] = {{64, 10.0, 6.6, 0.63, 0.27, Sizes<64>::kTops}, {256, 13.0, 1.1, 2.2, 0.21, Sizes<256>::kTops},
                          {512, 14.8, 0.5, 5.9, 0.21, kMaxSampled}, {1024, 15.4, 0.42, 11.2, 0.25, kMaxSampled}};
    const double c = 1e-3 * (double)classes, others = rows > 256 ? (double)rows / 256 - 1 : 0.0;
    int best = 1024;
    double least = 1e300;
    for (const Form& f : forms) {
        const double cost = f.alone + f.alone_c * c + others * (f.more + f.more_c * c);
        if (classes <= f.most && cost < least) {
            least = cost;
            best = f.threads;
        }
    }
    return best;
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
    switch (sample_threads(rows, classes)) {
        case 64: launch_sample<64, 4>(a, rows); break;
        case 256: launch_sample<256, 4>(a, rows); break;
        case 512: launch_sample<512, 8>(a, rows); break;
        default: launch_sample<1024, 4>(a, rows);
    }
    return finish("mh_sample_tokens");
}

}  // extern "C"
