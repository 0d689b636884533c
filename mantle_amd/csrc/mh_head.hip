// mh_head.hip -- softmax cross entropy of a vocabulary head, x [rows, dim] against w [classes, dim],
// without the logits as a tensor, and both gradients.
//
//   z = x w^T;  lse_n = log sum_v exp z_nv;  loss = mean over the kept rows of lse_n - z_n,label
//   G = (softmax(z) - onehot) ug / n;  grad_x = G w;  grad_w = G^T x
//
// Three products of 2 rows classes dim operations carry the time. The matrix instructions take fp32
// operands at a sixteenth of the fp16 rate, so every fp32 operand is held as two halves (hi, lo):
// v 2^e = hi + lo + r, |r| <= 2^-23 |v 2^e|, with a power of two e that puts the largest element into
// [2^14, 2^15). A product is hi hi + hi lo + lo hi, each exact in the fp32
// accumulator; what is dropped, lo lo, is below 2^-22 of |a b|. That is the error of fp32 operands within
// a factor of 4 for one term and below the rounding of an fp32 sum from some tens of terms on, at three
// fp16 instructions a product. fp16's least step, 2^-24, is lo's: elements below 2^-17 of the largest lose bits to
// it, and their absolute error stays below 2^-39 of the largest. For the logits e is a row's own in x, so that no
// row's result depends on another's size; a power of two a class of w as well cost 2 % of a forward (a different
// exponent for each sum at the product's end), and a logit's error, which is absolute, gains nothing from it while
// |x| |w| stays below 2^17. Both gradients contract over rows or classes: there e is the tensor's. lo times 2^11
// would hold 22 bits down to 2^-28, but its products need sums of their own, or a second pass over hi: 16.4 -> 18.4 ms
// a step over [4096, 2048] x [131072, 2048]. G is held the same way with e = 15 (|G| <= 1 before the factor ug / n,
// which the store applies).
//
// Operands lie in panels, the order the matrix instruction wants them: blocks of 32 rows x 16 of the
// contracted axis, hi then lo, 1 KB each, lane l's 16 bytes being 8 elements of row l % 32 from
// 8 (l / 32). A wavefront moves a block with one 16-byte load a lane, from memory straight to LDS, and
// reads it from there without bank conflicts. Panels are padded with zeros to whole tiles, so the loop
// over the contracted axis tests nothing.
//
// A step over [4096, 2048] x [131072, 2048] takes 16.2-17.0 ms by card: 14.2-14.9 in the three products (440-465
// TFLOP/s of fp32-exact products, three times that of fp16; torch's fp16 product of this shape reaches 1170-1220,
// its fp32 one 149), which run at 1.57 GHz with the matrix units busy in 80 % of the cycles: the card's power holds
// them. Tiles of 256 x 128 two a CU, or four wavefronts of 128 x 128 with a third less LDS traffic, take the same
// time. The rest is memory: G's panels 1.2 ms at 5.3 TB/s, w's 0.6, the scales 0.2.
#include "mh_internal.h"
#include "mh_math.h"
#include "mh_rows.h"

namespace mh {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kBlk = 2048;       // bytes of a panel block: 32 x 16 elements, hi and lo
constexpr int kGExp = 15;        // the power of two G is held with
constexpr int kAmaxBlocks = 1024;  // workgroups of k_amax for each of x and w

// What the kernels of one call share, in device memory.
struct HeadInfo {
    int32_t ex, ew;  // powers of two of all of x and of w
    int32_t kept;    // rows with a label
    int32_t pad;
};
static_assert(kAmaxBlocks == 4 * 256, "a workgroup of k_split reads four partials a thread");
struct alignas(16) HeadPart {  // k_amax's partials
    float ax[kAmaxBlocks], aw[kAmaxBlocks];
    int32_t kept[kAmaxBlocks];
};

// Blocks from one row block of a panel to the next, of kb in use: odd, so that the row blocks that workgroups
// read at the same time lie in different memory channels: 17.2 -> 16.5 ms a step over [4096, 2048] x
// [131072, 2048], 489 -> 450 us over [32768, 512] x [1000, 512], where powers of two were apart.
__host__ __device__ inline int64_t stride_of(int64_t kb) { return kb | 1; }
__host__ __device__ inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = __builtin_fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;  // NaN and infinity do not set the scale
}

// The power of two that puts a into [2^14, 2^15).
__device__ __forceinline__ int scale_exp(float a) {
    if (!(a > 0.0f)) return 0;
    int e;
    __builtin_frexpf(a, &e);  // a = f 2^e, f in [1/2, 1)
    return 15 - e;
}

// The largest finite magnitude of x's kept rows and of w, and the kept rows' count, as partials; each row's power of
// two.
__device__ __forceinline__ float amax4(float a, vf4 v) {
    return __builtin_fmaxf(__builtin_fmaxf(a, __builtin_fmaxf(finite_abs(v.x), finite_abs(v.y))),
                           __builtin_fmaxf(finite_abs(v.z), finite_abs(v.w)));
}
__global__ __launch_bounds__(256) void k_amax(HeadPart* part, int32_t* row_exp, const float* x, const float* w,
                                              const int32_t* labels, int64_t rows, int64_t dim, int64_t nw) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[4];
    __shared__ int32_t cnt[4];
    float a = 0.0f;
    int32_t kept = 0;
    const bool isx = blockIdx.x < kAmaxBlocks;
    const int b = isx ? blockIdx.x : blockIdx.x - kAmaxBlocks;
    if (isx) {
        // four rows at a time, so that their labels and their elements are under way together
        for (int64_t r0 = ((int64_t)b * 4 + wave) * 4; r0 < rows; r0 += kAmaxBlocks * 16) {
            bool in[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) in[u] = r0 + u < rows && labels[r0 + u < rows ? r0 + u : r0] >= 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) kept += in[u];  // a row left out may hold anything
            const float* row = x + r0 * dim;
            float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int64_t k = lane * 4; k + 3 < dim; k += 256) {
                vf4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = in[u] ? *reinterpret_cast<const vf4u*>(row + u * dim + k) : vf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 4; ++u) m[u] = amax4(m[u], v[u]);
            }
            if (lane < (dim & 3))
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (in[u]) m[u] = __builtin_fmaxf(m[u], finite_abs(row[u * dim + (dim & ~(int64_t)3) + lane]));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                m[u] = wave_max(m[u]);
                a = __builtin_fmaxf(a, m[u]);
            }
            const float mine = lane == 0 ? m[0] : lane == 1 ? m[1] : lane == 2 ? m[2] : m[3];
            if (lane < 4 && r0 + lane < rows) row_exp[r0 + lane] = scale_exp(mine);
        }
    } else {
        const int64_t nq = nw >> 2, step = kAmaxBlocks * 256;
        int64_t q = (int64_t)b * 256 + threadIdx.x;
        for (; q + 7 * step < nq; q += 8 * step) {  // eight loads in flight: 0.52 -> 0.2 ms a GB
            vf4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = ld_ntu(w + 4 * (q + u * step));
#pragma unroll
            for (int u = 0; u < 8; ++u) a = amax4(a, v[u]);
        }
        for (; q < nq; q += step) a = amax4(a, ld_ntu(w + 4 * q));
        if (b == 0 && threadIdx.x < (nw & 3)) a = __builtin_fmaxf(a, finite_abs(w[4 * nq + threadIdx.x]));
    }
    a = wave_max(a);
    if (lane == 0) {
        red[wave] = a;
        cnt[wave] = kept;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        a = __builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3]));
        if (isx) {
            part->ax[b] = a;
            part->kept[b] = cnt[0] + cnt[1] + cnt[2] + cnt[3];
        } else {
            part->aw[b] = a;
        }
    }
}

typedef float f32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void split8(f32x8 v, half8* hi, half8* lo) {
    *hi = __builtin_convertvector(v, half8);
    *lo = __builtin_convertvector(v - __builtin_convertvector(*hi, f32x8), half8);
}

constexpr int kSplitTile = 64;

// A [nr, nc] matrix into its row panels (contracted over columns) and, with colp, its column panels
// (contracted over rows), zero-padded: one 64 x 64 tile a workgroup. x's tiles come first, then w's.
struct SplitOne {
    const float* src;
    int64_t nr, nc;      // the matrix
    const int32_t* exps;  // its rows' powers of two, or null: one for all
    char* rowp;          // row blocks of rkb blocks, stride_of(rkb) apart; blocks at or past rkb are not stored
    char* colp;          // the same of ckb
    int64_t rkb, ckb;
    int64_t tiles_r, tiles_c;
    int64_t rb_end, cb_end;  // row blocks of rowp, of colp
};
__global__ __launch_bounds__(256) void k_split(SplitOne sx, SplitOne sw, const HeadPart* part, HeadInfo* info,
                                               const int32_t* labels) {
    // 68 floats a row: 16-byte accesses along a row and 4-byte ones along a column without bank conflicts
    __shared__ __attribute__((aligned(16))) float t[kSplitTile][kSplitTile + 4];
    __shared__ float red[4];
    __shared__ int32_t cnt[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t ntx = sx.tiles_r * sx.tiles_c;
    const bool isx = (int64_t)blockIdx.x < ntx;
    const SplitOne s = isx ? sx : sw;
    const int64_t tile = isx ? blockIdx.x : blockIdx.x - ntx;
    const int64_t r0 = tile / s.tiles_c * kSplitTile, c0 = tile % s.tiles_c * kSplitTile;
    float a = amax4(0.0f, reinterpret_cast<const vf4*>(isx ? part->ax : part->aw)[tid]);
    a = wave_max(a);
    if (lane == 0) red[wave] = a;
    // 16 threads a row, a quad each
    vf4 in[4];
    int er[2];
    if (s.exps)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t r = r0 + i * 32 + (lane & 31);
            er[i] = r < s.nr ? s.exps[r] : 0;
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + i * 16 + (tid >> 4), c = c0 + (tid & 15) * 4;
        in[i] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < s.nr && !(isx && labels[r] < 0)) {  // a row left out: zeros, whatever it holds
            const float* p = s.src + r * s.nc + c;
            if (c + 3 < s.nc) {
                in[i] = ld_ntu(p);
            } else {
                if (c < s.nc) in[i].x = p[0];
                if (c + 1 < s.nc) in[i].y = p[1];
                if (c + 2 < s.nc) in[i].z = p[2];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<vf4*>(&t[i * 16 + (tid >> 4)][(tid & 15) * 4]) = in[i];
    __syncthreads();
    const int e = scale_exp(__builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3])));
    if (!s.exps) er[0] = er[1] = e;
    const int r = lane & 31, k8 = (lane >> 5) * 8;
    // 2 row blocks x 4 blocks of the contracted axis each way: 8 blocks, two a wavefront
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rb = i, kb = wave;
        f32x8 v;
        half8 hi, lo;
        if (r0 / 32 + rb < s.rb_end && c0 / 16 + kb < s.rkb) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __builtin_ldexpf(t[rb * 32 + r][kb * 16 + k8 + j], er[rb]);
            split8(v, &hi, &lo);
            half8* p = reinterpret_cast<half8*>(s.rowp + ((r0 / 32 + rb) * stride_of(s.rkb) + c0 / 16 + kb) * kBlk);
            p[lane] = hi;
            p[64 + lane] = lo;
        }
        if (s.colp && c0 / 32 + rb < s.cb_end && r0 / 16 + kb < s.ckb) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __builtin_ldexpf(t[kb * 16 + k8 + j][rb * 32 + r], e);
            split8(v, &hi, &lo);
            half8* p = reinterpret_cast<half8*>(s.colp + ((c0 / 32 + rb) * stride_of(s.ckb) + r0 / 16 + kb) * kBlk);
            p[lane] = hi;
            p[64 + lane] = lo;
        }
    }
    if (blockIdx.x == 0) {  // the scales and the count, for the kernels behind
        float b = wave_max(amax4(0.0f, reinterpret_cast<const vf4*>(part->aw)[tid]));
        int32_t kept = part->kept[tid] + part->kept[tid + 256] + part->kept[tid + 512] + part->kept[tid + 768];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) kept += __shfl_xor(kept, o);
        __syncthreads();
        if (lane == 0) {
            red[wave] = b;
            cnt[wave] = kept;
        }
        __syncthreads();
        if (tid == 0) {
            info->ex = e;
            info->ew = scale_exp(__builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3])));
            info->kept = cnt[0] + cnt[1] + cnt[2] + cnt[3];
        }
    }
}

// ---------------------------------------------------------------------------------------
// the product of two panels
// ---------------------------------------------------------------------------------------
enum HeadEpi { EPI_LOGITS = 0, EPI_GRAD = 1 };

struct GemmArg {
    const char *a, *b;       // panels: M operand, N operand
    int64_t akb, bkb;        // blocks from one row block of each panel to the next
    int64_t kb;              // blocks contracted here, of one split: a multiple of 2
    int64_t kb_all;          // blocks contracted by all splits
    int32_t tiles_m, tiles_n, splits;
    const HeadInfo* info;
    // EPI_LOGITS: M is classes, N rows
    const int32_t* labels;   // at the first row of the panel; EPI_GRAD: rows to leave alone, or null
    int64_t rows, classes;   // of the operands; rows counted from the panel's first
    const int32_t* row_exp;  // the rows' powers of two, of all that the tiles hold
    float* stat;             // [64-class groups][2][stat_ld]: maximum, sum of exponentials
    int64_t stat_ld;
    float* target;           // [rows] the label's logit
    char* z;                 // the logits, in the blocks of G's row panels, or null
    int64_t zkb;
    // EPI_GRAD: out [m, n] += or = ug / kept * acc
    float* out;
    int64_t m, n;
    const float* ug;
    float* part;             // split sums [splits][tiles_m * TM][tiles_n * TN], or null
    int32_t exp_b;           // 0: x's power of two, 1: w's, 2: none
    int32_t accumulate;
};

// One or two products in a launch: the second starts with workgroup `first`, a multiple of 8.
struct GemmPair {
    GemmArg g[2];
    uint32_t first;
};

// ug / kept and the exponent that undoes the panels' scales, applied to one sum.
__device__ __forceinline__ float grad_value(float acc, float c, int e) { return c * __builtin_ldexpf(acc, e); }

// Waits until at most N of this wavefront's loads are under way and its LDS reads are done, then for the
// workgroup's other wavefronts. The compiler moves nothing across.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x70 | N);  // vmcnt N (below 16), lgkmcnt 0, expcnt as it is
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// Three stages of 16 of the contracted axis circle through LDS. In step s a wavefront waits for its loads of
// stage s + 1 and its reads of stage s, meets the others, and then, between the matrix instructions of
// stage s, which is in registers, reads stage s + 1 and loads stage s + 3 over stage s: neither the loads'
// latency nor LDS's stands before a matrix instruction.
template <int TM, int TN, int WM, int WN, int EPI>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_gemm(GemmPair pair) {
    const bool second = blockIdx.x >= pair.first;
    const GemmArg& g = pair.g[second];
    const uint32_t block = blockIdx.x - (second ? pair.first : 0);
    constexpr int kWaves = WM * WN, MI = TM / WM / 32, NI = TN / WN / 32;
    constexpr int kRows = (TM + TN) / 32;        // row blocks of a stage
    constexpr int kStage = kRows * kBlk;
    constexpr int kLoads = kRows * 2 / kWaves;   // 1 KB loads of a wavefront a stage
    static_assert(kRows % kWaves == 0 && 2 * kLoads < 16, "the waits' counts");
    __shared__ __attribute__((aligned(1024))) char lds[3 * kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // Workgroup b runs on XCD b % 8: each XCD takes a contiguous run of a split's tiles, in groups of 8 tile
    // rows, so that its L2 holds what its workgroups share, and as many as the others.
    const int64_t T = (int64_t)g.tiles_m * g.tiles_n, all = T * g.splits;
    const int64_t item = (int64_t)(block & 7) * ((all + 7) / 8) + (block >> 3);
    if ((int64_t)(block >> 3) >= (all + 7) / 8 || item >= all) return;
    const int64_t split = item / T, id = item - split * T;
    const int64_t gsz = (int64_t)8 * g.tiles_n, grp = id / gsz;
    const int gm = (int)(g.tiles_m - grp * 8 < 8 ? g.tiles_m - grp * 8 : 8);
    const int64_t tm = grp * 8 + (id - grp * gsz) % gm, tn = (id - grp * gsz) / gm;

    const int64_t k0 = split * g.kb;
    const int64_t kb = g.kb_all - k0 < g.kb ? g.kb_all - k0 : g.kb;
    const int S = (int)kb;  // even; 0 or less for a split past the end

    const char* src[kLoads / 2];  // the row blocks this wavefront brings
#pragma unroll
    for (int i = 0; i < kLoads / 2; ++i) {
        const int rb = wave * (kLoads / 2) + i;
        src[i] = (rb < TM / 32 ? g.a + ((tm * (TM / 32) + rb) * g.akb + k0) * kBlk
                               : g.b + ((tn * (TN / 32) + rb - TM / 32) * g.bkb + k0) * kBlk);
    }
    const uint32_t lane16 = lane * 16;
    // Part i of kLoads of a stage's loads, into the stage at `to`. Past the end: the last stage again, which no
    // one reads.
    auto load = [&](int s, int to, int i) {
        const int64_t at = (int64_t)(s < S ? s : S - 1) * kBlk;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(src[i >> 1] + at + (i & 1) * 1024 + lane16),
            (__attribute__((address_space(3))) void*)(lds + to + wave * (kLoads / 2) * kBlk + i * 1024), 16, 0, 0);
    };
    // Part i of kReads of the operands of the stage at `from`: N's first, both halves of each.
    constexpr int kReads = 2 * (MI + NI), kProducts = 3 * MI * NI;
    auto read = [&](int from, int i, half8(&a)[MI][2], half8(&b)[NI][2]) {
        const char* at = lds + from + lane16;
        if (i < 2 * NI) b[i >> 1][i & 1] = *reinterpret_cast<const half8*>(at + (TM / 32 + wn * NI) * kBlk + i * 1024);
        else a[(i - 2 * NI) >> 1][i & 1] = *reinterpret_cast<const half8*>(at + wm * MI * kBlk + (i - 2 * NI) * 1024);
    };

    f32x16 acc[MI][NI] = {};
    int here = 0;  // the stage in registers
    // The next stage's reads and loads go between the matrix instructions, one at a time: issued together at
    // the step's start they fill LDS's queue, and the wavefronts stand before it.
    auto step = [&](int s, half8(&a)[MI][2], half8(&b)[NI][2], half8(&an)[MI][2], half8(&bn)[NI][2]) {
        wait_and_meet<kLoads>();
        const int next = here == 2 * kStage ? 0 : here + kStage;
#pragma unroll
        for (int t = 0; t < kProducts; ++t) {
            constexpr int kEvery = kProducts / kReads;  // 2 in the large tiles, 1 in the small one
            if (t % kEvery == 0 && t / kEvery < kReads) read(next, t / kEvery, an, bn);
            if (t % (kProducts / kLoads) == kProducts / kLoads / 2) load(s + 3, here, t / (kProducts / kLoads));
            const int u = t / (MI * NI), i = t % (MI * NI) / NI, j = t % NI;  // the small terms first
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][u == 1], b[j][u == 0], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0x6);  // but address arithmetic
        }
        here = next;
    };
    if (S > 0) {
        half8 a0[MI][2], b0[NI][2], a1[MI][2], b1[NI][2];
#pragma unroll
        for (int i = 0; i < 3 * kLoads; ++i) load(i / kLoads, i / kLoads * kStage, i % kLoads);
        wait_and_meet<2 * kLoads>();
#pragma unroll
        for (int i = 0; i < kReads; ++i) read(0, i, a0, b0);
        for (int s = 0; s < S; s += 2) {
            step(s, a0, b0, a1, b1);
            step(s + 1, a1, b1, a0, b0);
        }
        wait_and_meet<0>();  // no load into LDS outlives the workgroup
    }

    // acc[i][j][r]: row (of M) 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4, column (of N) 32 j + lane % 32
    const int half = lane >> 5, col = lane & 31;
    if constexpr (EPI == EPI_LOGITS) {
        int e[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) e[j] = -(g.row_exp[tn * TN + (wn * NI + j) * 32 + col] + g.info->ew);
        const int64_t v0 = tm * TM + wm * MI * 32;  // the wavefront's first class
        // register r of tile i holds class v0 + 4 half + cls_of(i, r): compared with the label and the
        // last class relative to the first two terms
        const int64_t left = g.classes - v0 - 4 * half;
        const int last = left < 0 ? 0 : left < MI * 32 ? (int)left : MI * 32;
        auto cls_of = [](int i, int r) { return i * 32 + 8 * (r >> 2) + (r & 3); };
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int64_t n = tn * TN + (wn * NI + j) * 32 + col;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = __builtin_ldexpf(acc[i][j][r], e[j]);
            {
                const int64_t want = (n < g.rows ? (int64_t)g.labels[n] : -1) - v0 - 4 * half;
                if (want >= 0 && want < MI * 32) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (cls_of(i, r) == (int)want) g.target[n] = acc[i][j][r];
                }
                // the maximum and the sum of exponentials of each 64 classes, whatever the tile, so that the
                // sums' order does not depend on it: a difference, a product and one exp2 a logit; only the last
                // class's wavefront masks what lies past it
                const bool whole = g.classes - v0 >= MI * 32;
#pragma unroll
                for (int h = 0; h < MI / 2; ++h) {
                    float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
                    for (int i = 2 * h; i < 2 * h + 2; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (whole || cls_of(i, r) < last) top = __builtin_fmaxf(top, acc[i][j][r]);
                    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                    const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
                    for (int i = 2 * h; i < 2 * h + 2; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (whole || cls_of(i, r) < last)
                                sum += __builtin_amdgcn_exp2f((acc[i][j][r] - base) * kLog2e);
                    sum += __shfl_xor(sum, 32);  // a NaN among the logits is in the sum, whatever the maximum says
                    if (half == 0) {
                        const int64_t at = ((v0 >> 6) + h) * 2 * g.stat_ld + n;
                        g.stat[at] = top;
                        g.stat[at + g.stat_ld] = sum;
                    }
                }
            }
            if (g.z) {  // 4 consecutive classes a lane: 16 bytes of the block of (n / 32, v / 16)
                char* zb = g.z + (n >> 5) * g.zkb * kBlk;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int64_t vb = (v0 >> 4) + i * 2 + (q >> 1);
                        vf4 o = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                        *reinterpret_cast<vf4*>(zb + vb * kBlk + (col + 32 * (q & 1)) * 32 + half * 16) = o;
                    }
            }
        }
    } else {
        if (g.part) {
            const int64_t ld = (int64_t)g.tiles_n * TN;
            float* p = g.part + split * g.tiles_m * TM * ld;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int64_t m = tm * TM + (wm * MI + i) * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
                        p[m * ld + tn * TN + (wn * NI + j) * 32 + col] = acc[i][j][r];
                    }
            return;
        }
        const int e = -(kGExp + (g.exp_b == 2 ? 0 : g.exp_b ? g.info->ew : g.info->ex));
        const float c = g.ug[0] / (float)(g.info->kept > 0 ? g.info->kept : 1);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t m = tm * TM + (wm * MI + i) * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
                if (m >= g.m) continue;
                const bool out = g.labels && g.labels[m] < 0;  // a row left out: as it was, or zero
                if (out && g.accumulate) continue;
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const int64_t n = tn * TN + (wn * NI + j) * 32 + col;
                    if (n >= g.n) continue;
                    float* o = g.out + m * g.n + n;
                    const float v = out ? 0.0f : grad_value(acc[i][j][r], c, e);
                    *o = g.accumulate ? *o + v : v;
                }
            }
    }
}

// Joins the splits of the gradient products that have them, in their order. A product's rows of sums are
// tiles_n tiles of `tile` wide.
__global__ __launch_bounds__(256) void k_join(GemmPair pair, int32_t tile) {
    const bool second = blockIdx.x >= pair.first;
    const GemmArg& g = pair.g[second];
    const int64_t block = blockIdx.x - (second ? pair.first : 0), blocks = second ? gridDim.x - pair.first : pair.first;
    const int64_t ld = (int64_t)g.tiles_n * tile, plane = (int64_t)g.tiles_m * tile * ld;
    const int e = -(kGExp + (g.exp_b == 2 ? 0 : g.exp_b ? g.info->ew : g.info->ex));
    const float c = g.ug[0] / (float)(g.info->kept > 0 ? g.info->kept : 1);
    const int64_t total = g.m * g.n;
    for (int64_t i = block * 256 + threadIdx.x; i < total; i += blocks * 256) {
        const int64_t m = i / g.n, n = i - m * g.n;
        const bool out = g.labels && g.labels[m] < 0;
        if (out && g.accumulate) continue;
        float v = 0.0f;
        if (!out) {
            for (int s = 0; s < g.splits; ++s) v += g.part[s * plane + m * ld + n];
            v = grad_value(v, c, e);
        }
        g.out[i] = g.accumulate ? g.out[i] + v : v;
    }
}

// ---------------------------------------------------------------------------------------
// rows' statistics, the loss, and G's panels
// ---------------------------------------------------------------------------------------
// Each row's maximum and sum of exponentials from its class groups', its log-sum-exp, and the workgroup's sum of
// losses: 16 rows x 4 W
// threads, whose loads of a group's statistics are 64 bytes each. W = 16 wavefronts a workgroup, or 4 where the
// groups are few ([32768, 512] x [1000, 512]'s 16 groups: 17 and 9 us).
constexpr int kLseRows = 16;
struct Lse {
    float top, sum;
};
// What makes a row's probabilities of its logits: e^(z - top) inv. The log-sum-exp would not do: rounded to fp32
// it is off by up to 2^-24 of itself, and all of the row's probabilities with it, so that G's rows did not add up to 0.
struct RowScale {
    float top, inv;
};
// A sum that is not a number stays so; a group of logits at minus infinity adds nothing.
__device__ __forceinline__ void lse_join(Lse& a, float m, float s) {
    const float d = m > a.top ? a.top - m : m - a.top;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    if (m > a.top) {
        a.sum = a.sum * e + s;
        a.top = m;
    } else if (m > -__builtin_inff() || s != s) {
        a.sum += s * e;
    }
}
template <int W>
__global__ __launch_bounds__(W * 64) void k_rows_lse(const float* stat, int64_t groups, int64_t stat_ld,
                                                   const float* target, const int32_t* labels, int64_t rows,
                                                   int64_t classes, const float* row_lse_in, float* row_lse,
                                                   float* row_loss, double* block_loss, RowScale* row_scale) {
    __shared__ float sm[W][kLseRows], ss[W][kLseRows];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, p = wave * 4 + (lane >> 4);
    const int64_t n = (int64_t)blockIdx.x * kLseRows + r;
    Lse a = {-__builtin_inff(), 0.0f};
    for (int64_t gr = p; gr < groups; gr += 16 * W) {
        float m[4], s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t at = gr + u * 4 * W < groups ? gr + u * 4 * W : gr;
            m[u] = stat[at * 2 * stat_ld + n];
            s[u] = stat[(at * 2 + 1) * stat_ld + n];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (gr + u * 4 * W < groups) lse_join(a, m[u], s[u]);
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
        const float m = __shfl_xor(a.top, o), s = __shfl_xor(a.sum, o);
        lse_join(a, m, s);
    }
    if (lane < kLseRows) {
        sm[wave][r] = a.top;
        ss[wave][r] = a.sum;
    }
    __syncthreads();
    if (threadIdx.x >= kLseRows) return;
#pragma unroll
    for (int i = 1; i < W; ++i) lse_join(a, sm[i][r], ss[i][r]);
    float loss = 0.0f;
    if (n < rows) {
        const int32_t label = labels[n];
        float lse = a.top + mlog(a.sum);
        if (label >= classes) lse = __builtin_nanf("");  // no such class: shown in the loss and the gradients
        if (label < 0) lse = 0.0f;
        // the logits' common offset goes first
        loss = label < 0 ? 0.0f : label >= classes ? lse : (a.top - target[n]) + mlog(a.sum);
        if (row_lse) row_lse[n] = lse;
        if (row_loss) row_loss[n] = loss;
        if (row_scale) {
            const bool bad = label >= classes || (row_lse_in && row_lse_in[n] != row_lse_in[n]);
            row_scale[n] = {a.top, bad ? __builtin_nanf("") : 1.0f / a.sum};
        }
    }
    double total = loss;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) total += __shfl_xor(total, o);
    if (r == 0) block_loss[blockIdx.x] = total;
}

// loss = sum of the workgroups' losses / kept, by one workgroup of 256 threads and in a fixed order.
__device__ void rows_loss(const double* block_loss, int64_t blocks, const HeadInfo* info, float* loss, double* red) {
    double s = 0.0;
#pragma unroll 4
    for (int64_t n = threadIdx.x; n < blocks; n += 256) s += block_loss[n];
    s = block_sum<4>(s, red);
    if (threadIdx.x == 0) loss[0] = (float)(s / (double)(info->kept > 0 ? info->kept : 1));
}
__global__ __launch_bounds__(256) void k_rows_loss(const double* block_loss, int64_t blocks, const HeadInfo* info,
                                                   float* loss) {
    __shared__ double red[4];
    rows_loss(block_loss, blocks, info, loss, red);
}

// Logits to G's panels: a wavefront takes 32 rows x 32 classes (two blocks of logits, which become two
// blocks of the row panel in place) and writes the same elements to the column panel through LDS. With `loss`,
// `tiles` workgroups do that and one more adds up the loss.
__global__ __launch_bounds__(256) void k_to_g(char* z, int64_t zkb, char* gt, int64_t gtkb, int64_t gt_blocks, const RowScale* scale,
                                              const int32_t* labels, int64_t rows, int64_t classes, int64_t tiles_v,
                                              int64_t tiles, const double* block_loss, int64_t loss_blocks,
                                              const HeadInfo* info, float* loss) {
    __shared__ __attribute__((aligned(16))) _Float16 t[4][2][32][40];
    __shared__ double red[4];
    if (blockIdx.x >= tiles) {  // one workgroup more, behind the last chunk's: the loss
        rows_loss(block_loss, loss_blocks, info, loss, red);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t id = (int64_t)blockIdx.x * 4 + wave;
    const int64_t nb = id / tiles_v, vt = id % tiles_v;  // the grid covers whole workgroups of tiles
    const int64_t n = nb * 32 + (lane & 31);
    const int32_t label = n < rows ? labels[n] : -1;
    const RowScale sc = n < rows ? scale[n] : RowScale{0.0f, 0.0f};
    const int k8 = (lane >> 5) * 8;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        char* blk = z + (nb * zkb + vt * 2 + b) * kBlk;
        const vf4 q0 = reinterpret_cast<const vf4*>(blk)[lane * 2], q1 = reinterpret_cast<const vf4*>(blk)[lane * 2 + 1];
        f32x8 v = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t cls = vt * 32 + b * 16 + k8 + j;
            const float p = exp_neg(v[j] - sc.top) * sc.inv - (cls == label ? 1.0f : 0.0f);
            v[j] = label < 0 || cls >= classes ? 0.0f : p * (float)(1 << kGExp);
        }
        half8 hi, lo;
        split8(v, &hi, &lo);
        // every lane of the wavefront has its logits before the block is written over
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
        reinterpret_cast<half8*>(blk)[lane] = hi;
        reinterpret_cast<half8*>(blk)[64 + lane] = lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[wave][0][b * 16 + k8 + j][lane & 31] = hi[j];
            t[wave][1][b * 16 + k8 + j][lane & 31] = lo[j];
        }
    }
    __syncthreads();
    if (nb >= gt_blocks) return;  // rows that grad_w's product does not reach
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // rows n of 16 b .. 16 b + 15 as the contracted axis
        char* blk = gt + (vt * gtkb + nb * 2 + b) * kBlk;
#pragma unroll
        for (int p = 0; p < 2; ++p)
            reinterpret_cast<half8*>(blk)[64 * p + lane] =
                *reinterpret_cast<const half8*>(&t[wave][p][lane & 31][b * 16 + k8]);
    }
}

// ---------------------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------------------
// Up to 64 rows, or 128 without gradients, against a large w, whose bytes bound both products that read it: w
// goes to the matrix unit from memory, as it lies, split in registers. A power of two for all of it would take a
// pass of its own, so each element becomes three bf16 (hi, mid, lo: 24 bits at fp32's own exponents), and a
// product six instructions: all but mid lo, lo mid and lo lo, below 2^-24. [16, 4096] x [32000, 4096]: 433 ->
// 175 us forward (3 TB/s of w), 859 -> 495 with both gradients; torch's fp32 operations take 178 and 626. Of 128
// rows the forward gains, 429 -> 316 us, but k_few_dx would need 255 registers a thread: 1069 us a step, against
// 895 by panels.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr int kFewRows = 64, kFewRowsForward = 128, kFewBlk = 3 * 1024;  // bytes of a block of x: three planes of 32 rows x 16

struct Tri {
    bf16x8 h, m, l;
};
__device__ __forceinline__ Tri split3(f32x8 v) {
    Tri t;
    t.h = __builtin_convertvector(v, bf16x8);
    v -= __builtin_convertvector(t.h, f32x8);
    t.m = __builtin_convertvector(v, bf16x8);
    v -= __builtin_convertvector(t.m, f32x8);
    t.l = __builtin_convertvector(v, bf16x8);
    return t;
}
__device__ __forceinline__ f32x16 mul3(const Tri& a, const Tri& b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.l, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.h, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.h, c, 0, 0, 0);
}

struct FewArg {
    const float *x, *w;
    const int32_t* labels;
    int64_t rows, dim, classes, dkb;
    char* xp;        // x's blocks, [row blocks][dkb]
    float* stat;     // [32-class groups][2][stat_ld]
    int64_t stat_ld;
    float* target;
    char* z;         // as GemmArg's, or null; G's panel for k_few_dx
    int64_t zkb;
    float* part;     // [splits][rows of blocks][dim_p]
    int64_t dim_p, ckb, per;  // padded dims; 16-class blocks in all and of a split
};

// x to its three planes, a wavefront a block; a row left out becomes zeros, whatever it holds.
__global__ __launch_bounds__(64) void k_few_x(FewArg f) {
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x / f.dkb * 32 + (lane & 31), c = blockIdx.x % f.dkb * 16 + (lane >> 5) * 8;
    const bool in = r < f.rows && f.labels[r] >= 0;
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = in && c + j < f.dim ? f.x[r * f.dim + c + j] : 0.0f;
    const Tri t = split3(v);
    bf16x8* p = reinterpret_cast<bf16x8*>(f.xp + (int64_t)blockIdx.x * kFewBlk);
    p[lane] = t.h;
    p[64 + lane] = t.m;
    p[128 + lane] = t.l;
}

// Logits of 32 classes by all rows a workgroup: eight wavefronts take an eighth of the dims each, four 2 KB blocks of
// w under way a wavefront, and add up in LDS.
template <int NT>
__global__ __launch_bounds__(512) void k_few_logits(FewArg f) {
    __shared__ float sums[4][NT][16 * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int64_t v0 = (int64_t)blockIdx.x * 32, v = v0 + col;
    const int64_t per = (f.dkb + 7) / 8;
    const int64_t k1 = (wave + 1) * per < f.dkb ? (wave + 1) * per : f.dkb;
    const float* row = f.w + (v < f.classes ? v : 0) * f.dim;
    // a class past the last reads the first one's: its logits count nowhere
    auto whole = [&](int64_t kb) {
        const float* p = row + kb * 16 + half * 8;
        const vf4 a = *reinterpret_cast<const vf4u*>(p), b = *reinterpret_cast<const vf4u*>(p + 4);
        return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    };
    auto edge = [&](int64_t kb) {
        f32x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t c = kb * 16 + half * 8 + j;
            o[j] = c < f.dim ? row[c] : 0.0f;
        }
        return o;
    };
    f32x16 acc[NT] = {};
    for (int64_t k = wave * per; k < k1; k += 4) {
        f32x8 in[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) in[u] = (k + 4) * 16 <= f.dim ? whole(k + u) : edge(k + u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (k + u >= k1) break;
            const Tri a = split3(in[u]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bf16x8* p = reinterpret_cast<const bf16x8*>(f.xp + (t * f.dkb + k + u) * kFewBlk);
                acc[t] = mul3(a, Tri{p[lane], p[64 + lane], p[128 + lane]}, acc[t]);
            }
        }
    }
    // the second four wavefronts' sums go to the first four, and theirs to one a row block
    if (wave >= 4)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[wave - 4][t][r * 64 + lane] = acc[t][r];
    __syncthreads();
    if (wave < 4)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                acc[t][r] += sums[wave][t][r * 64 + lane];
                sums[wave][t][r * 64 + lane] = acc[t][r];
            }
    __syncthreads();
    if (wave >= NT) return;
    float z[16];
#pragma unroll
    for (int r = 0; r < 16; ++r)
        z[r] = (sums[0][wave][r * 64 + lane] + sums[1][wave][r * 64 + lane]) +
               (sums[2][wave][r * 64 + lane] + sums[3][wave][r * 64 + lane]);
    // register r: class v0 + 8 (r / 4) + 4 half + r % 4 of row n, as in k_gemm
    const int64_t n = wave * 32 + col;
    {
        const int64_t left = f.classes - v0 - 4 * half;
        const int64_t want = (n < f.rows ? (int64_t)f.labels[n] : -1) - v0 - 4 * half;
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int c = 8 * (r >> 2) + (r & 3);
            if (c == want && c < left) f.target[n] = z[r];
            if (c < left) top = __builtin_fmaxf(top, z[r]);
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) < left) sum += __builtin_amdgcn_exp2f((z[r] - base) * kLog2e);
        sum += __shfl_xor(sum, 32);
        if (half == 0) {
            f.stat[(int64_t)blockIdx.x * 2 * f.stat_ld + n] = top;
            f.stat[((int64_t)blockIdx.x * 2 + 1) * f.stat_ld + n] = sum;
        }
    }
    if (f.z) {
        char* zb = f.z + wave * f.zkb * kBlk;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<vf4*>(zb + ((v0 >> 4) + (q >> 1)) * kBlk + (col + 32 * (q & 1)) * 32 + half * 16) =
                vf4{z[4 * q], z[4 * q + 1], z[4 * q + 2], z[4 * q + 3]};
    }
}

// G w over a split of the classes, 32 dims by all rows a wavefront: its loads of w are 128 bytes of a class, 512 of
// four wavefronts, and four blocks' are under way.
template <int NT>
__global__ __launch_bounds__(256) void k_few_dx(FewArg f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int64_t d = ((int64_t)blockIdx.x * 4 + wave) * 32 + col;
    const int64_t k0 = blockIdx.y * f.per, k1 = k0 + f.per < f.ckb ? k0 + f.per : f.ckb;
    const float* wd = f.w + (d < f.dim ? d : 0);  // a dim past the last reads the first one's, for sums that no one reads
    f32x16 acc[NT] = {};
    for (int64_t k = k0; k < k1; k += 4) {
        f32x8 in[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t v = (k + u) * 16 + half * 8;
            if ((k + 4) * 16 <= f.classes) {
#pragma unroll
                for (int j = 0; j < 8; ++j) in[u][j] = wd[(v + j) * f.dim];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) in[u][j] = v + j < f.classes ? wd[(v + j) * f.dim] : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (k + u >= k1) break;
            const Tri b = split3(in[u]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const half8* p = reinterpret_cast<const half8*>(f.z + (t * f.zkb + k + u) * kBlk);
                const f32x8 g = __builtin_convertvector(p[lane], f32x8) + __builtin_convertvector(p[64 + lane], f32x8);
                acc[t] = mul3(split3(g), b, acc[t]);
            }
        }
    }
    float* o = f.part + blockIdx.y * (NT * 32) * f.dim_p;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[(t * 32 + 8 * (r >> 2) + 4 * half + (r & 3)) * f.dim_p + d] = acc[t][r];
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
// The logits of one chunk of rows and G's column panel take 8 bytes an element, a forward's statistics 8 bytes for 64;
// a chunk's rows keep them within this, 256 rows at least.
constexpr int64_t kChunkBytes = (int64_t)4 << 30;
constexpr int64_t kMaxChunk = 32768;
constexpr int64_t kFewElements = (int64_t)1 << 22;  // of w, from which its bytes and not launches count

struct Carve {
    size_t at = 0;
    size_t take(int64_t bytes) {
        const size_t o = at;
        at += (size_t)up(bytes, 1024);
        return o;
    }
};

// A product's tile and the splits of its contracted axis.
struct Form {
    int tile, splits;
};

// The least time, in units of one 128 x 128 x 16 block on a whole CU (0.23 us). A 256 x 256 tile takes four a
// block on a CU of its own and 24 blocks' time around them (its 256 KB store stands alone); of the 128 x 128
// ones up to three share a CU, which then works at 0.5, 0.78 or 0.82 of the large tile's rate, with 10 around
// them. Measured on either side: [4096, 1024] x [32000, 1024]'s logits take 625 us in large tiles and 670 in
// small ones; a step of [1023, 513] x [30011, 513] 491 us with its grad_x in 21 splits of large tiles or 12 of small
// ones. A split writes and reads its sums and costs one more launch. A gradient's sums run over at most 65536
// elements each, whatever that takes in splits: the matrix unit's fp32 sums drift by 4e-11 of themselves an element
// (8e-5 over 2^21 of them unsplit). A logit's sum is one, over all dims: 7e-4 of itself at 2^24 of them.
constexpr int64_t kMaxSplit = 64, kLongest = 4096;  // splits taken for speed at most, blocks of 16 of a split
Form form_of(int64_t m, int64_t n, int64_t kb, bool split) {
    static const double rate[4] = {1.0, 0.5, 0.78, 0.82};
    const int64_t cus = ctx().num_cus, least = split ? (kb + kLongest - 1) / kLongest : 1;
    Form best = {0, 0};
    double time = 0.0;
    for (const int T : {256, 128}) {
        const int64_t tiles = up(m, T) / T * (up(n, T) / T);
        for (int64_t s = least; s <= (least > kMaxSplit ? least : kMaxSplit); ++s) {
            const int64_t wg = tiles * s, steps = (kb + s - 1) / s;
            double t;
            if (T == 256) {
                t = (double)((wg + cus - 1) / cus) * 4.0 * (double)(steps + 24);
            } else {
                const int64_t w = (wg + cus - 1) / cus < 3 ? (wg + cus - 1) / cus : 3;
                const double rounds = (double)wg / (double)(cus * w) + 0.3;
                t = (rounds > 1.0 ? rounds : 1.0) * (double)w / rate[w] * (double)(steps + 10);
            }
            if (s > 1) t += (double)(s * m * n) * 8.0 / 5.0e6 / 0.23 + 20.0;
            if (best.tile == 0 || t < time) {
                time = t;
                best = {T, (int)s};
            }
            if (!split || steps <= 16) break;
        }
    }
    return best;
}

void set_form(GemmArg& g, int64_t m, int64_t n, const Form& f) {
    g.m = m;
    g.n = n;
    g.tiles_m = (int32_t)(up(m, f.tile) / f.tile);
    g.tiles_n = (int32_t)(up(n, f.tile) / f.tile);
    g.splits = f.splits;
    g.kb = up((g.kb_all + f.splits - 1) / f.splits, 2);
}
int64_t gemm_blocks(int64_t tiles, int64_t splits) { return 8 * ((tiles * splits + 7) / 8); }
uint32_t gemm_blocks(const GemmArg& g) { return (uint32_t)gemm_blocks((int64_t)g.tiles_m * g.tiles_n, g.splits); }
// `n` products of one tile in a launch.
template <int EPI>
void launch_gemm(const GemmArg* g, int n, int tile) {
    GemmPair p = {{g[0], g[n - 1]}, gemm_blocks(g[0])};
    const dim3 grid(p.first + (n > 1 ? gemm_blocks(g[1]) : 0));
    if (tile == 256) hipLaunchKernelGGL((k_gemm<256, 256, 2, 4, EPI>), grid, dim3(512), 0, ctx().stream, p);
    else hipLaunchKernelGGL((k_gemm<128, 128, 2, 2, EPI>), grid, dim3(256), 0, ctx().stream, p);
}

struct HeadCall {
    const char* what;
    float *loss, *row_loss, *row_lse_out;
    const float* row_lse_in;
    float *gx, *gw;
    const float *x, *w;
    const int32_t* labels;
    const float* ug;
    int64_t rows, dim, classes;
    bool train, accumulate;
};

// The gradient products, both in one launch where they take the same tile, and the joins of their splits.
void grad_products(GemmArg* g, const Form* f, int n) {
    if (n == 2 && f[0].tile != f[1].tile) {
        grad_products(g, f, 1);
        grad_products(g + 1, f + 1, 1);
        return;
    }
    launch_gemm<EPI_GRAD>(g, n, f[0].tile);
    GemmArg j[2];
    int nj = 0;
    uint32_t blocks[2] = {0, 0};
    for (int i = 0; i < n; ++i)
        if (g[i].splits > 1) {
            const int64_t b = grid_blocks(g[i].m * g[i].n, 256);
            blocks[nj] = (uint32_t)(b > 4096 ? 4096 : b);
            j[nj++] = g[i];
        }
    if (nj == 0) return;
    const GemmPair p = {{j[0], j[nj - 1]}, blocks[0]};
    hipLaunchKernelGGL(k_join, dim3(blocks[0] + blocks[1]), dim3(256), 0, ctx().stream, p, f[0].tile);
}

size_t part_bytes(int64_t m, int64_t n, const Form& f) {
    return f.splits > 1 ? (size_t)f.splits * up(m, f.tile) * up(n, f.tile) * sizeof(float) : 0;
}

// The forms of a chunk of nr rows. The contracted axes end at whole pairs of blocks; the rows behind nr and the
// classes behind the last are zeros in the panels.
struct Forms {
    Form logits, grad[2];  // of x, of w
    int64_t rows;          // padded to the tiles that read them
    size_t part[2];
};

// How a call's work is cut and where its workspace lies: known before anything is launched.
struct HeadPlan {
    int64_t rowsP, clsP, dkb;  // padded
    int64_t dim_x, dim_w;      // dims padded to the tiles that read x's and w's column panels
    int64_t chunk, groups;
    bool few;
    int nt;
    int64_t fdim, fkb, fsplits;
    Forms whole, last;  // of a chunk, of the last one
    size_t o_info, o_part, o_ex, o_xr, o_wr, o_xt, o_wt, o_stat, o_tgt, o_scale, o_rl, o_z, o_gt, o_sp, o_fx, bytes;
    int64_t items;  // work-items of the largest launch that grows with the sizes
};

Forms forms_of(HeadPlan& p, int64_t nr, int64_t dim, int64_t classes, bool gx, bool gw) {
    Forms f = {};
    auto launch = [](int64_t m, int64_t n, const Form& form) {
        const int64_t blocks = gemm_blocks(up(m, form.tile) / form.tile * (up(n, form.tile) / form.tile), form.splits);
        return blocks * (form.tile == 256 ? 512 : 256);
    };
    auto count = [&p](int64_t items) { p.items = items > p.items ? items : p.items; };
    f.logits = form_of(classes, nr, p.dkb, false);
    f.rows = up(nr, f.logits.tile);
    int64_t grads = 0;
    if (gx) {
        f.grad[0] = form_of(nr, dim, up(classes, 32) / 16, true);
        if (up(nr, f.grad[0].tile) > f.rows) f.rows = up(nr, f.grad[0].tile);
        f.part[0] = part_bytes(nr, dim, f.grad[0]);
        if (up(dim, f.grad[0].tile) > p.dim_w) p.dim_w = up(dim, f.grad[0].tile);
        if (!p.few) grads += launch(nr, dim, f.grad[0]);
    }
    if (gw) {
        f.grad[1] = form_of(classes, dim, up(nr, 32) / 16, true);
        f.part[1] = part_bytes(classes, dim, f.grad[1]);
        if (up(dim, f.grad[1].tile) > p.dim_x) p.dim_x = up(dim, f.grad[1].tile);
        grads += launch(classes, dim, f.grad[1]);
    }
    count(grads);
    if (!p.few) count(launch(p.clsP, f.rows, f.logits));
    if (gx || gw) count((f.rows / 32 * (p.clsP / 32) / 4 + 1) * 256);  // k_to_g
    return f;
}

HeadPlan plan_of(int64_t rows, int64_t dim, int64_t classes, bool gx, bool gw) {
    HeadPlan p = {};
    const bool train = gx || gw;
    p.rowsP = up(rows, 256);
    p.clsP = up(classes, 256);
    p.dkb = up(dim, 32) / 16;
    // w straight from memory where rows are few and w is large enough to bound the products, in rows long enough
    // for eight wavefronts each ([32, 64] x [100000, 64]: 178 us so, 146 by panels)
    p.few = rows <= (train ? kFewRows : kFewRowsForward) && dim >= 256 && classes * dim >= kFewElements;
    p.nt = rows > 64 ? 4 : rows > 32 ? 2 : 1;
    p.groups = p.few ? p.clsP / 32 : p.clsP / 64;
    p.chunk = (train ? kChunkBytes / (p.clsP * 8) : kChunkBytes / (p.groups * 8)) / 256 * 256;
    p.chunk = p.chunk < 256 ? 256 : p.chunk > kMaxChunk ? kMaxChunk : p.chunk;
    if (p.chunk > p.rowsP) p.chunk = p.rowsP;
    p.fdim = up(dim, 128);
    p.fkb = up(classes, 16) / 16;
    // splits of the classes that give every CU eight wavefronts or so, of 16 blocks at least
    p.fsplits = p.few ? (2 * ctx().num_cus + p.fdim / 128 - 1) / (p.fdim / 128) : 1;
    if (p.fsplits > p.fkb / 16) p.fsplits = p.fkb / 16;
    p.fsplits = p.fsplits < 1 ? 1 : p.fsplits > kMaxSplit ? kMaxSplit : p.fsplits;
    if (p.fsplits * kLongest < p.fkb) p.fsplits = (p.fkb + kLongest - 1) / kLongest;
    const int64_t behind = rows - (rows - 1) / p.chunk * p.chunk;  // rows of the last chunk
    p.whole = forms_of(p, rows < p.chunk ? rows : p.chunk, dim, classes, gx, gw);
    p.last = behind == p.chunk || rows < p.chunk ? p.whole : forms_of(p, behind, dim, classes, gx, gw);
    const int64_t most = p.dim_x > p.dim_w ? p.dim_x : p.dim_w, wide = most > up(dim, 64) ? most : up(dim, 64);
    const int64_t split = (p.rowsP / 64 + (p.few ? 0 : p.clsP / 64)) * (wide / 64) * 256, logits = p.few ? p.clsP / 32 * 512 : 0;
    p.items = split > p.items ? split : p.items;
    p.items = logits > p.items ? logits : p.items;

    Carve cv;
    p.o_info = cv.take(sizeof(HeadInfo));
    p.o_part = cv.take(sizeof(HeadPart));
    p.o_ex = cv.take(p.rowsP * 4);
    p.o_xr = cv.take(p.rowsP / 32 * stride_of(p.dkb) * kBlk);
    p.o_wr = p.few ? 0 : cv.take(p.clsP / 32 * stride_of(p.dkb) * kBlk);
    p.o_xt = gw ? cv.take(p.dim_x / 32 * stride_of(p.rowsP / 16) * kBlk) : 0;
    p.o_wt = gx && !p.few ? cv.take(p.dim_w / 32 * stride_of(p.clsP / 16) * kBlk) : 0;
    p.o_stat = cv.take(p.groups * 2 * p.chunk * 4);
    p.o_tgt = cv.take(p.chunk * 4);
    p.o_scale = cv.take(train ? p.chunk * (int64_t)sizeof(RowScale) : 0);
    p.o_rl = cv.take(p.rowsP / kLseRows * 8);
    if (train) {
        p.o_z = cv.take(p.chunk / 32 * stride_of(p.clsP / 16) * kBlk);
        p.o_gt = cv.take(p.clsP / 32 * stride_of(p.chunk / 16) * kBlk);
        size_t sp = p.few ? (size_t)(p.fsplits * p.nt * 32 * p.fdim) * sizeof(float) : 0;
        for (const Forms* f : {&p.whole, &p.last})
            if (f->part[0] + f->part[1] > sp) sp = f->part[0] + f->part[1];
        p.o_sp = cv.take((int64_t)sp);
    }
    p.o_fx = p.few ? cv.take(p.nt * p.dkb * kFewBlk) : 0;
    p.bytes = cv.at;
    return p;
}

int head_run(const HeadCall& h, const HeadPlan& pl) {
    const int64_t rows = h.rows, dim = h.dim, classes = h.classes;
    const int64_t rowsP = pl.rowsP, clsP = pl.clsP, dkb = pl.dkb, chunk = pl.chunk, groups = pl.groups;
    const int64_t fdim = pl.fdim, fkb = pl.fkb, fsplits = pl.fsplits;
    const bool few = pl.few;
    const int nt = pl.nt;
    char* base = nullptr;
    MH_TRY(scratch(pl.bytes, reinterpret_cast<void**>(&base)));
    hipStream_t st = ctx().stream;
    HeadInfo* info = reinterpret_cast<HeadInfo*>(base + pl.o_info);
    HeadPart* part = reinterpret_cast<HeadPart*>(base + pl.o_part);
    RowScale* scale = h.train ? reinterpret_cast<RowScale*>(base + pl.o_scale) : nullptr;
    double* block_loss = reinterpret_cast<double*>(base + pl.o_rl);
    float* target = reinterpret_cast<float*>(base + pl.o_tgt);

    int32_t* row_exp = reinterpret_cast<int32_t*>(base + pl.o_ex);
    hipLaunchKernelGGL(k_amax, dim3(few ? kAmaxBlocks : 2 * kAmaxBlocks), dim3(256), 0, st, part, row_exp, h.x, h.w, h.labels,
                       rows, dim, classes * dim);
    SplitOne sx = {h.x, rows, dim, row_exp, base + pl.o_xr, h.train && h.gw ? base + pl.o_xt : nullptr, dkb, rowsP / 16,
                   rowsP / 64, up(dim, 64) / 64, rowsP / 32, pl.dim_x / 32};
    SplitOne sw = {h.w, classes, dim, nullptr, base + pl.o_wr, h.train && h.gx ? base + pl.o_wt : nullptr, dkb, clsP / 16,
                   clsP / 64, up(dim, 64) / 64, clsP / 32, pl.dim_w / 32};
    if (sx.colp) sx.tiles_c = pl.dim_x / 64;
    if (sw.colp) sw.tiles_c = pl.dim_w / 64;
    const int64_t nsplit = sx.tiles_r * sx.tiles_c + (few ? 0 : sw.tiles_r * sw.tiles_c);
    hipLaunchKernelGGL(k_split, dim3((unsigned)nsplit), dim3(256), 0, st, sx, sw, part, info, h.labels);

    for (int64_t r0 = 0; r0 < rows; r0 += chunk) {
        const int64_t nr = rows - r0 < chunk ? rows - r0 : chunk;
        const Forms& f = nr < chunk && r0 > 0 ? pl.last : pl.whole;
        const int64_t nrP = f.rows, zkb = stride_of(clsP / 16), gtkb = stride_of(up(nr, 32) / 16);
        GemmArg g = {};
        g.a = base + pl.o_wr;
        g.b = base + pl.o_xr + r0 / 32 * stride_of(dkb) * kBlk;
        g.akb = g.bkb = stride_of(dkb);
        g.kb_all = dkb;
        g.info = info;
        g.labels = h.labels + r0;
        g.rows = nr;
        g.classes = classes;
        g.row_exp = row_exp + r0;
        g.stat = reinterpret_cast<float*>(base + pl.o_stat);
        g.stat_ld = chunk;
        g.target = target;
        g.z = h.train ? base + pl.o_z : nullptr;
        g.zkb = zkb;
        // every row and class that a gradient's tiles read gets its logits: the panels behind have no gaps
        set_form(g, clsP, nrP, f.logits);
        FewArg fa = {h.x, h.w, h.labels, rows, dim, classes, dkb, base + pl.o_fx, g.stat, g.stat_ld, target, g.z, zkb,
                     reinterpret_cast<float*>(base + pl.o_sp), fdim, fkb, (fkb + fsplits - 1) / fsplits};
        if (few) {
            hipLaunchKernelGGL(k_few_x, dim3((unsigned)(nt * dkb)), dim3(64), 0, st, fa);
            const dim3 grid((unsigned)(clsP / 32));
            if (nt == 1) hipLaunchKernelGGL((k_few_logits<1>), grid, dim3(512), 0, st, fa);
            else if (nt == 2) hipLaunchKernelGGL((k_few_logits<2>), grid, dim3(512), 0, st, fa);
            else hipLaunchKernelGGL((k_few_logits<4>), grid, dim3(512), 0, st, fa);
        } else {
            launch_gemm<EPI_LOGITS>(&g, 1, f.logits.tile);
        }
        const dim3 lse_grid((unsigned)((nr + kLseRows - 1) / kLseRows));
        float *lse = h.row_lse_out ? h.row_lse_out + r0 : nullptr, *rl = h.row_loss ? h.row_loss + r0 : nullptr;
        const float* lse_in = h.row_lse_in ? h.row_lse_in + r0 : nullptr;
        double* bl = block_loss + r0 / kLseRows;
        if (groups <= 32)
            hipLaunchKernelGGL((k_rows_lse<4>), lse_grid, dim3(256), 0, st, g.stat, groups, g.stat_ld, target,
                               h.labels + r0, nr, classes, lse_in, lse, rl, bl, scale);
        else
            hipLaunchKernelGGL((k_rows_lse<16>), lse_grid, dim3(1024), 0, st, g.stat, groups, g.stat_ld, target,
                               h.labels + r0, nr, classes, lse_in, lse, rl, bl, scale);
        if (!h.train) continue;
        const int64_t tiles_v = clsP / 32, tiles = nrP / 32 * tiles_v / 4;
        const bool with_loss = h.loss && r0 + chunk >= rows;
        hipLaunchKernelGGL(k_to_g, dim3((unsigned)(tiles + with_loss)), dim3(256), 0, st, base + pl.o_z, zkb,
                           base + pl.o_gt, gtkb, up(nr, 32) / 32, scale, h.labels + r0, nr,
                           classes, tiles_v, tiles, block_loss, (rows + kLseRows - 1) / kLseRows, info, h.loss);
        GemmArg d[2] = {};
        Form df[2];
        int nd = 0;
        float* sp = reinterpret_cast<float*>(base + pl.o_sp);
        if (h.gx) {
            GemmArg& p = d[nd];
            p.a = base + pl.o_z;
            p.akb = zkb;
            p.b = base + pl.o_wt;
            p.bkb = stride_of(clsP / 16);
            p.kb_all = up(classes, 32) / 16;
            p.exp_b = 1;
            p.labels = h.labels + r0;
            p.out = h.gx + r0 * dim;
            p.accumulate = h.accumulate;
            p.part = f.grad[0].splits > 1 ? sp : nullptr;
            set_form(p, nr, dim, f.grad[0]);
            df[nd++] = f.grad[0];
            if (few) {
                const dim3 grid((unsigned)(fdim / 128), (unsigned)fsplits);
                if (nt == 1) hipLaunchKernelGGL((k_few_dx<1>), grid, dim3(256), 0, st, fa);
                else hipLaunchKernelGGL((k_few_dx<2>), grid, dim3(256), 0, st, fa);
                p.info = info;
                p.ug = h.ug;
                p.exp_b = 2;
                p.part = fa.part;
                p.splits = (int32_t)fsplits;
                p.tiles_m = nt;
                p.tiles_n = (int32_t)(fdim / 32);
                const uint32_t blocks = (uint32_t)((rows * dim + 255) / 256);
                hipLaunchKernelGGL(k_join, dim3(blocks), dim3(256), 0, st, (GemmPair{{p, p}, blocks}), 32);
                d[--nd] = GemmArg{};
            }
        }
        if (h.gw) {
            GemmArg& p = d[nd];
            p.a = base + pl.o_gt;
            p.akb = gtkb;
            p.b = base + pl.o_xt + r0 / 16 * kBlk;
            p.bkb = stride_of(rowsP / 16);
            p.kb_all = up(nr, 32) / 16;
            p.out = h.gw;
            p.accumulate = h.accumulate || r0 > 0;
            // behind grad_x's sums; those of few rows are joined by then
            p.part = f.grad[1].splits > 1 ? sp + (few ? 0 : f.part[0] / sizeof(float)) : nullptr;
            set_form(p, classes, dim, f.grad[1]);
            df[nd++] = f.grad[1];
        }
        for (int i = 0; i < nd; ++i) {
            d[i].info = info;
            d[i].ug = h.ug;
        }
        if (nd) grad_products(d, df, nd);
    }
    if (!h.train)
        hipLaunchKernelGGL(k_rows_loss, dim3(1), dim3(256), 0, st, block_loss, (rows + kLseRows - 1) / kLseRows, info, h.loss);
    return finish(h.what);
}

int head_check(const char* what, int64_t rows, int64_t dim, int64_t classes, bool gx, bool gw, HeadPlan* p) {
    if (rows < 0 || dim < 1 || classes < 1)
        return fail(MH_ERR_INVALID, "%s: needs rows >= 0, dim >= 1, classes >= 1 (%lld, %lld, %lld)", what, (long long)rows,
                    (long long)dim, (long long)classes);
    if (classes > 0x7fffffff || dim > (1 << 24) || rows > 0x7fffffff)
        return fail(MH_ERR_OVERFLOW, "%s: more than 2^31 - 1 rows or classes, or 2^24 dims", what);
    // one workgroup a 64 x 64 tile of x and of w
    if ((up(rows, 256) / 64 + up(classes, 256) / 64) * (up(dim, 256) / 64) > max_grid_blocks(256))
        return fail(MH_ERR_OVERFLOW, "%s: operands of more than 2^36 elements, dims rounded up to 256", what);
    if (rows == 0) return MH_OK;
    *p = plan_of(rows, dim, classes, gx, gw);
    if (p->items > kMaxDispatchItems)
        return fail(MH_ERR_OVERFLOW, "%s: a launch of more than 2^32 work-items", what);
    return MH_OK;
}
int head_check(const HeadCall& h, HeadPlan* p) {
    return head_check(h.what, h.rows, h.dim, h.classes, h.gx != nullptr, h.gw != nullptr, p);
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_linear_cross_entropy_fwd(float* loss, float* row_loss, float* row_lse, const float* x, const float* w,
                                const int32_t* labels, int64_t rows, int64_t dim, int64_t classes) {
    MH_TRACE("mh_linear_cross_entropy_fwd");
    HeadCall h = {};
    h.what = "mh_linear_cross_entropy_fwd";
    h.loss = loss;
    h.row_loss = row_loss;
    h.row_lse_out = row_lse;
    h.x = x;
    h.w = w;
    h.labels = labels;
    h.rows = rows;
    h.dim = dim;
    h.classes = classes;
    HeadPlan p;
    MH_TRY(head_check(h, &p));
    if (!loss || !w || (rows > 0 && (!x || !labels))) return fail(MH_ERR_NULL, "%s: null tensor", h.what);
    MH_TRY(require_init());
    if (rows == 0) return mh_fill(loss, 0.0f, 1);
    return head_run(h, p);
}

int mh_linear_cross_entropy_bwd(float* grad_x, float* grad_w, const float* x, const float* w, const int32_t* labels,
                                const float* row_lse, const float* ug, int64_t rows, int64_t dim, int64_t classes,
                                int accumulate) {
    MH_TRACE("mh_linear_cross_entropy_bwd");
    HeadCall h = {};
    h.what = "mh_linear_cross_entropy_bwd";
    h.gx = grad_x;
    h.gw = grad_w;
    h.row_lse_in = row_lse;
    h.x = x;
    h.w = w;
    h.labels = labels;
    h.ug = ug;
    h.rows = rows;
    h.dim = dim;
    h.classes = classes;
    h.train = true;
    h.accumulate = accumulate != 0;
    HeadPlan p;
    MH_TRY(head_check(h, &p));
    if (!grad_x && !grad_w) return MH_OK;
    if (!w || !ug || (rows > 0 && (!x || !labels || !row_lse))) return fail(MH_ERR_NULL, "%s: null tensor", h.what);
    MH_TRY(require_init());
    if (rows == 0) return grad_w && !accumulate ? mh_zero(grad_w, classes * dim) : MH_OK;
    return head_run(h, p);
}

int mh_linear_cross_entropy_step(float* loss, float* row_lse, float* grad_x, float* grad_w, const float* x,
                                 const float* w, const int32_t* labels, const float* ug, int64_t rows, int64_t dim,
                                 int64_t classes, int accumulate) {
    MH_TRACE("mh_linear_cross_entropy_step");
    HeadCall h = {};
    h.what = "mh_linear_cross_entropy_step";
    h.loss = loss;
    h.row_lse_out = row_lse;
    h.gx = grad_x;
    h.gw = grad_w;
    h.x = x;
    h.w = w;
    h.labels = labels;
    h.ug = ug;
    h.rows = rows;
    h.dim = dim;
    h.classes = classes;
    h.train = grad_x || grad_w;
    h.accumulate = accumulate != 0;
    HeadPlan p;
    MH_TRY(head_check(h, &p));
    if (!loss || !w || (h.train && !ug) || (rows > 0 && (!x || !labels))) return fail(MH_ERR_NULL, "%s: null tensor", h.what);
    MH_TRY(require_init());
    if (rows == 0) {
        if (grad_w && !accumulate) MH_TRY(mh_zero(grad_w, classes * dim));
        return mh_fill(loss, 0.0f, 1);
    }
    return head_run(h, p);
}

int mh_plan_head(int64_t rows, int64_t dim, int64_t classes, int grad_x, int grad_w, mh_head_info* out) {
    if (!out) return fail(MH_ERR_NULL, "mh_plan_head: null");
    *out = mh_head_info{};
    HeadPlan p;
    MH_TRY(head_check("mh_plan_head", rows, dim, classes, grad_x != 0, grad_w != 0, &p));
    if (rows == 0) return MH_OK;
    out->rows_at_once = rows < p.chunk ? rows : p.chunk;
    out->scratch_bytes = (int64_t)p.bytes;
    out->largest_launch = p.items;
    return MH_OK;
}

}  // extern "C"
