// SPDX-License-Identifier: Apache-2.0
//
// The nearest orthogonal matrix of an update G, by Newton-Schulz products:
//
//   X = G / (|G|_F + eps);   per step (a, b, c):   A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// which applies the odd polynomial a s + b s^3 + c s^5 to every singular value.  X is taken with
// its shorter side p as rows (the transposed problem is the same one), q is the longer side.
//
// All the work is matrix products, 2 p^2 q + 2 p^3 + 2 p^2 q operations a step, half of the first two
// spared because A and A^2 are symmetric: only tiles on and below the diagonal are computed,
// and stored twice.
//
// Numerics.  The products run on fp16 MFMA with fp32 sums, on operands held as TWO fp16 terms,
// x = h + l, 22 bits in all: h h + h l + l h per product, as accurate as 32-bit products (the
// l l that is left out is 2^-22 of one) at three times the cost of one fp16 product instead of
// the ten times of fp32 MFMA.  One term is not enough: the iteration multiplies small singular values by a
// each step, and with them the rounding errors of the first steps, up to a^steps = 485 times;
// with a few strong directions over a floor of weak ones a single fp16 term ends 2 to 3 % off (bf16:
// 20 %), measured on spectra with a ratio of 1000.  Nor is it enough in the first steps alone, where B X is small beside
// a X if all singular values are small: where one row holds most of an update, one of them is near 1 from the start and B
// all but a single element, whose rounding nothing averages ([2560, 2560] fp32 1.5e-3 off, [768, 768] bf16 3.3e-3 instead of
// 1.6e-3).  The host, which launches the steps, does not see the spectrum: all products are of two terms, for
// results of every type.  (With one term in three or four of five steps [14336, 4096] bf16 took 5.4 ms instead of 10.2, [1024, 4096] bf16 265 us
// instead of 367.)
// fp16 rather than bf16 terms because the iterates are bounded: entries of X are at most about
// 1.2, they are held times a power of two near sqrt(p q) so that their typical size stays in the
// middle of fp16's range; A and B are held times powers of two likewise.  Where |G| is far below eps, or a step makes all singular values
// small, these powers follow a bound of the singular values from step to step, for each matrix by itself: see plan_kernel.
//
// Operand layout.  A matrix [R, K] that enters a product as rows x K is stored as blocks of 32
// rows x 16 k in the lane order of v_mfma_f32_32x32x16 (lane: row lane % 32, k = 8 (lane / 32) + 0..7), 1 KiB
// per block, blocks of one row of blocks adjacent, the second term a whole matrix behind the first.  Tiles go
// from memory to LDS with global_load_lds as they are, and from LDS to registers as
// conflict-free 16-byte reads.  Products run transposed (the second operand first), so that a
// lane holds four consecutive k of one row of the result seen as an operand: results go back to that
// layout in 8-byte stores, 512 contiguous bytes per instruction.  The transposed copy that the next product needs (X^T; the tile mirrored
// at the diagonal) is made in registers by an MFMA with the identity, which is exact.
// Sides are padded with zeros to whole tiles; products of zeros stay zeros, nothing is masked.

#include <errno.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fstx_gather_core.h"
#include "fstx_internal.h"
#include "fstx_overlap.h"
#include "fstx_update.h"

namespace {

#define FSTX_GLOBAL __attribute__((address_space(1)))
#define FSTX_LDS __attribute__((address_space(3)))
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 half_t;

constexpr uint32_t kBlk = 512;        // elements of one block (32 rows x 16 k) of one term
constexpr uint32_t kTerms = 2;
constexpr uint32_t kPadP = 256, kPadQ = 256; // sides are stored padded to these (the largest tile)
constexpr uint32_t kStepPad = 64;            // ... and summed over padded to this
constexpr uint32_t kMaxJobs = 20;
constexpr uint32_t kPartials = 1024;         // partial sums of squares per matrix
constexpr float kScaleA = 2048.0f;    // A is held times this

struct alignas(64) Job {
    const char *src;
    char *dst;
    half_t *x;        // [p, q]
    half_t *xt0, *xt1; // [q, p], the current one and the next in turn
    half_t *a, *b;    // [p, p]
    double *partials; // later the matrix's Plan
    uint64_t x_row, x_col;   // strides of G seen as X, elements
    uint64_t dst_pitch;      // bytes
    uint32_t p, q;
    uint32_t type, flipped;  // flipped: X is G transposed
    float scale;             // X is held times this
    uint32_t n_partials;
    uint64_t pad[2];
};
static_assert(sizeof(Job) == 128, "20 of them fit the kernel arguments");

struct Steps { // coefficients of a call, or of a run of steps
    float c[3 * 64];
    uint32_t n, first;
    float eps;
};

// What one step multiplies with: B = own A + product A A, X = own X + product B X, as they are held
struct StepPlan {
    float poly_own, poly_product, apply_own, apply_product;
};
// Per matrix, over its partial sums of squares once these are added
struct Plan {
    float factor;
    int32_t exponent; // X is G times factor 2^exponent
    uint32_t pad[2];
    StepPlan step[64];
};
static_assert(sizeof(Plan) <= kPartials * sizeof(double), "a plan takes the place of the partial sums");

struct Jobs {
    Job job[kMaxJobs];
    uint32_t first[kMaxJobs]; // first workgroup of each job; unused entries ~0
};

// How one product's tiles are dealt to workgroups (see Launcher::deal): the first `whole` tiles of a job
// take one workgroup each, the others `split` each, which leave partial sums.
struct Deal {
    uint32_t whole[kMaxJobs];
    uint32_t slot[kMaxJobs];   // where the job's partial sums begin, in tiles
    float *sums;
    uint32_t split, dies_log2;
};

// (by value: a conditional between two members is a conditional between their addresses)
template <typename T> __device__ __forceinline__ T pick(bool first, T a, T b) { return first ? a : b; }

// The whole job in two wide scalar loads: a copy, because conditional reads through a reference into the
// kernel's arguments end up as a copy of all of them in scratch memory.
__device__ __forceinline__ Job fetch_job(const Jobs &t, uint32_t ji) {
    typedef uint32_t v16u __attribute__((ext_vector_type(16)));
    const v16u *raw = reinterpret_cast<const v16u *>(&t.job[ji]);
    const v16u lo = raw[0], hi = raw[1];
    Job out;
    __builtin_memcpy(&out, &lo, 64);
    __builtin_memcpy(reinterpret_cast<char *>(&out) + 64, &hi, 64);
    return out;
}

__device__ __forceinline__ uint32_t job_of(const Jobs &t, uint32_t b) {
    uint32_t ji = 0;
#pragma unroll
    for (uint32_t i = 1; i < kMaxJobs; ++i) ji += b >= t.first[i];
    return ji;
}

__host__ __device__ inline uint32_t pad_to(uint32_t n, uint32_t to) { return (n + to - 1) / to * to; }

// N elements, those at(e) that are there(e), zeros else.  All loads go out together: the type is looked at once, and what
// is not there is read from the matrix's first element and dropped (a branch around each load would wait for one after the other: the first operands
// of a [14336, 4096] bf16 update 129 us instead of 186; 104 with the norm's sums added by plan_kernel).
template <uint32_t N, typename At, typename There>
__device__ __forceinline__ void load_elems(const char *src, uint32_t type, float (&x)[N], At at, There there) {
    if (type == FSTX_F32) {
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) x[e] = *(const FSTX_GLOBAL float *)(src + (there(e) ? at(e) : 0) * 4);
    } else {
        uint16_t raw[N];
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) raw[e] = *(const FSTX_GLOBAL uint16_t *)(src + (there(e) ? at(e) : 0) * 2);
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) x[e] = type == FSTX_BF16 ? __builtin_bit_cast(float, (uint32_t)raw[e] << 16) : (float)__builtin_bit_cast(half_t, raw[e]);
    }
#pragma unroll
    for (uint32_t e = 0; e < N; ++e) x[e] = there(e) ? x[e] : 0.0f;
}

// N consecutive elements, 16 bytes per load, as aligned as one element
template <uint32_t N> __device__ __forceinline__ void load_run(const char *src, uint64_t at, uint32_t type, float (&v)[N]) {
    typedef v4u by2 __attribute__((aligned(2)));
    typedef v4u by4 __attribute__((aligned(4)));
    if (type == FSTX_F32) {
#pragma unroll
        for (uint32_t k = 0; k < N; k += 4) {
            const v4u raw = *(const FSTX_GLOBAL by4 *)(src + (at + k) * 4);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t bits = raw[e];
                v[k + e] = __builtin_bit_cast(float, bits);
            }
        }
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < N; k += 8) {
        const v4u raw = *(const FSTX_GLOBAL by2 *)(src + (at + k) * 2);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t lo = raw[e] << 16, hi = raw[e] & 0xffff0000u;
            if (type == FSTX_BF16) {
                v[k + 2 * e] = __builtin_bit_cast(float, lo);
                v[k + 2 * e + 1] = __builtin_bit_cast(float, hi);
            } else {
                v[k + 2 * e] = (float)__builtin_bit_cast(half_t, (uint16_t)(lo >> 16));
                v[k + 2 * e + 1] = (float)__builtin_bit_cast(half_t, (uint16_t)(hi >> 16));
            }
        }
    }
}

// ------------------------------------------------------------ |G|_F and the first operands

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// G seen with the side along which memory runs as columns, whichever of X's sides that is
struct View {
    uint64_t row_stride, col_stride;
    uint32_t rows, cols;
    bool x_cols; // the columns are X's columns
};
__device__ __forceinline__ View view_of(const Job &job) {
    if (job.x_col <= job.x_row) return View{job.x_row, job.x_col, job.p, job.q, true};
    return View{job.x_col, job.x_row, job.q, job.p, false};
}

// Partial sums of squares in 64 bits, each workgroup its own rows in a fixed order: the sum does
// not depend on which workgroup ends first, and squares of the largest floats do not overflow.
__global__ __launch_bounds__(256) void sum_squares_kernel(const Jobs t) {
    __shared__ double part[4];
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job job = fetch_job(t, ji);
    const View g = view_of(job);
    const uint32_t me = blockIdx.x - t.first[ji];
    // the matrix as one run of eights of a row, dealt out to all threads in turn
    const uint32_t eights = (g.cols + 7) / 8;
    const uint64_t first = (uint64_t)me * 256 + threadIdx.x, stride = (uint64_t)job.n_partials * 256;
    const uint64_t rows_on = stride / eights;
    const uint32_t eights_on = (uint32_t)(stride - rows_on * eights);
    uint64_t row = first / eights;
    uint32_t nth = (uint32_t)(first - row * eights);
    auto next = [&]() {
        row += rows_on;
        nth += eights_on;
        if (nth >= eights) {
            nth -= eights;
            ++row;
        }
    };
    double sum = 0;
    auto add = [&](const float (&v)[8]) {
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) sum += (double)v[k] * (double)v[k];
    };
    if (g.col_stride == 1 && g.cols % 8 == 0) {
        while (row < g.rows) { // four at a time: those behind the end are read from the beginning and dropped
            float v[4][8];
            bool there[4];
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n) {
                there[n] = row < g.rows;
                load_run<8>(job.src, there[n] ? row * g.row_stride + nth * 8 : 0, job.type, v[n]);
                next();
            }
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n) {
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) v[n][k] = there[n] ? v[n][k] : 0.0f;
                add(v[n]);
            }
        }
    } else {
        for (; row < g.rows; next()) {
            float v[8];
            load_elems<8>(job.src, job.type, v, [&](uint32_t k) { return row * g.row_stride + (uint64_t)(nth * 8 + k) * g.col_stride; },
                          [&](uint32_t k) { return nth * 8 + k < g.cols; });
            add(v);
        }
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) job.partials[me] = part[0] + part[1] + part[2] + part[3];
}

// The powers of two that a matrix's operands are held times, from a bound s of its singular values: |G| / (|G| + eps)
// at first, |a| s + |b| s^3 + |c| s^5 behind a step.  X is held times scale 2^e, s 2^e being just below 1 (e = 0 from s = 1/2 on), A times
// kScaleA 2^(2 e), and B times the power of two up to which 4 |b| + 16 |c|, its largest entry for s = 2, stays below fp16's
// largest, and for e > 0 another 2^g that puts the bound |b| s^2 + |c| s^4 there.  Held times fixed powers of two instead, an
// update of |G| = 10^-6 eps came out 1.7 % off, with its digits in fp16's denormals, and one of 10^-8 eps as zero.
// One wavefront per matrix; its partial sums are all read before the plan is written over them.
__global__ __launch_bounds__(64) void plan_kernel(const Jobs t, const Steps steps) {
    const Job job = fetch_job(t, blockIdx.x);
    double sum = 0;
    for (uint32_t i = threadIdx.x; i < job.n_partials; i += 64 * 16) { // (all loads at once: one after the other they take 4 us)
        double part[16];
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) part[k] = job.partials[i + 64 * k < job.n_partials ? i + 64 * k : 0];
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) sum += i + 64 * k < job.n_partials ? part[k] : 0.0;
    }
    const double norm = sqrt(wave_sum(sum)), whole = norm + (double)steps.eps;
    if (threadIdx.x) return;
    auto exponent_of = [](double bound) { return bound > 0 && bound < 1 ? -ilogb(bound) - 1 : 0; };
    FSTX_GLOBAL Plan *plan = (FSTX_GLOBAL Plan *)reinterpret_cast<Plan *>(job.partials);
    double s = norm / whole; // (NaN, like what follows from it, where G holds infinities or NaN or |G| + eps is zero)
    int e = exponent_of(s), shift = 0;
    const double mantissa = frexp(whole, &shift); // 1 / (|G| + eps) may lie outside of what 32 bits hold, its mantissa and exponent do not
    plan->factor = (float)((double)job.scale / mantissa);
    plan->exponent = whole < HUGE_VAL ? e - shift : 0;
    for (uint32_t k = 0; k < steps.n; ++k) {
        const double a = steps.c[3 * k], b = steps.c[3 * k + 1], c = steps.c[3 * k + 2];
        const bool linear = b == 0 && c == 0; // (B is zero)
        const double top = linear ? 1.0 : 4.0 * fabs(b) + 16.0 * fabs(c);
        const int held = ilogb(60000.0 / top);
        int g = 0;
        if (e > 0 && !linear) { // (exponents, because s^4 may be smaller than what 64 bits hold)
            const double small = fmax(log2(fabs(b)) + 2.0 * log2(s), log2(fabs(c)) + 4.0 * log2(s));
            g = (int)fmin(fmax(floor(log2(top) - 2.0 - small), 0.0), 4096.0);
        }
        const double next = s * (fabs(a) + s * s * (fabs(b) + s * s * fabs(c)));
        const bool last = k + 1 == steps.n;
        const int to = last ? -ilogb((double)job.scale) : exponent_of(next); // the result itself is not scaled
        FSTX_GLOBAL StepPlan &p = plan->step[k];
        p.poly_own = (float)ldexp(b / (double)kScaleA, held + g - 2 * e);
        p.poly_product = (float)ldexp(c / ((double)kScaleA * (double)kScaleA), held + g - 4 * e);
        p.apply_own = (float)ldexp(a, to - e);
        p.apply_product = (float)ldexp(1.0, to - e - g - held);
        s = next;
        e = to;
    }
}

// ------------------------------------------------------------ the products

// Waits until at most `left` of this wavefront's global loads are on their way and none of its LDS
// reads, then for the other wavefronts.  (The empty statements keep the compiler from moving memory accesses
// across; the wait is the builtin, which it takes into account when it places its own.)
template <uint32_t left> __device__ __forceinline__ void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (left & 15) | (left >> 4) << 14);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// C = P Q^T over whole tiles: TR x TC per workgroup of four wavefronts (2 x 2), k in stages.  While one stage is
// multiplied from registers the next one is read from LDS into other registers and two more are on
// their way from memory to LDS; reads and loads are issued in between the products.
//
// What bounds it.  B X of a [14336, 4096] update, three products of 0.48 * 10^12 operations each in fp16: 1.07 to
// 1.2 ms with 256 x 256 tiles, 1.2 to 1.35 PFLOP/s; the library's 8192^3 fp16 product does 1.3 to 1.5 on the same cards
// with the matrix cores busy 94 % of the time at 1.43 GHz -- the power limit -- and this one 80 % at 1.6 GHz.
// Steps on the way, same product: 1.45 ms with 128 x 128 tiles, 32 k per
// stage and one stage ahead; 1.3 with 16 k and two ahead; 1.15 with 256 x 128 tiles; 1.07 with 256 x 256, reads between the
// products and the ends' loads put before their stores.  More stages ahead, raised wave priority around the
// products, and reads gathered into the first half of a stage changed nothing or cost 1 to 10 %.
template <uint32_t TR, uint32_t TC> struct Product {
    static constexpr uint32_t kKb = TR == 64 ? 2 : 1;                         // k blocks per stage
    // Stages in LDS: one computed on, the others on their way.  Small tiles run where few workgroups wait for
    // each other's results from memory: four, [768, 768] fp32 157 us instead of 176, [1024, 1024] bf16 187 instead of 204 (five: the same).
    static constexpr uint32_t kBufs = TR == 64 ? 4 : 3;
    static constexpr uint32_t kHalfP = TR / 32 * kKb * kTerms;                 // blocks of either operand per stage
    static constexpr uint32_t kHalfQ = TC / 32 * kKb * kTerms;
    static constexpr uint32_t kStage = (kHalfP + kHalfQ) * kBlk;              // elements per stage
    static constexpr uint32_t kLoads = (kHalfP + kHalfQ) / 4;                 // per wavefront and stage
    static constexpr uint32_t kWaves = TR * TC > 256 * 128 ? 1 : 2;           // wavefronts per SIMD the registers are divided for
    static constexpr uint32_t kNR = TR / 64, kNC = TC / 64;                   // 32-blocks per wavefront
    static_assert(kHalfP % 4 == 0 && kHalfQ % 4 == 0, "a load instruction of four wavefronts stays within one operand");

    // `Swap`: lanes hold rows of P (four consecutive rows of Q each); else rows of Q
    template <bool Swap>
    static __device__ __forceinline__ void run(const half_t *p, const half_t *q, uint64_t p_plane, uint64_t q_plane, uint32_t k_blocks_stored, uint32_t stages,
                                               half_t *lds, v16f (&acc)[kNR][kNC]) {
        const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wr = wave >> 1, wc = wave & 1;
        const uint64_t row_step = (uint64_t)k_blocks_stored * kBlk;
        auto load_part = [&](uint32_t kb0, uint32_t buf, uint32_t n) {
            const uint32_t at = n * 4 + wave;
            const bool second = n * 4 >= kHalfP;
            const uint32_t in = second ? at - kHalfP : at;
            const uint32_t rb = in / (kKb * kTerms), rest = in % (kKb * kTerms);
            const half_t *from = (second ? q : p) + rb * row_step + (uint64_t)(kb0 + rest / kTerms) * kBlk + (rest % kTerms ? pick(second, q_plane, p_plane) : 0) + lane * 8;
            __builtin_amdgcn_global_load_lds((const FSTX_GLOBAL void *)from, (FSTX_LDS void *)(lds + buf * kStage + at * kBlk), 16, 0, 0);
        };
        auto load_stage = [&](uint32_t kb0, uint32_t buf) {
#pragma unroll
            for (uint32_t n = 0; n < kLoads; ++n) load_part(kb0, buf, n);
        };
        struct Fragments {
            v8h p[kKb][kNR][kTerms], q[kKb][kNC][kTerms];
        };
        // A stage's LDS reads and its products, numbered: reads in the order in which products want them
        constexpr uint32_t kReads = kKb * kTerms * (kNR + kNC), kPerKb = 3 * kNR * kNC, kProducts = kKb * kPerKb;
        auto read = [&](const half_t *base, Fragments &f, uint32_t r) {
            const uint32_t kb = r / (kTerms * (kNR + kNC)), m = r / (kNR + kNC) % kTerms, i = r % (kNR + kNC);
            if (i < kNR) f.p[kb][i][m] = *(const v8h *)(base + (((wr * kNR + i) * kKb + kb) * kTerms + m) * kBlk);
            else f.q[kb][i - kNR][m] = *(const v8h *)(base + (kHalfP + ((wc * kNC + i - kNR) * kKb + kb) * kTerms + m) * kBlk);
        };
        auto product = [&](const Fragments &f, uint32_t n) {
            const uint32_t kb = n / kPerKb, kind = n % kPerKb / (kNR * kNC), i = n / kNC % kNR, j = n % kNC;
            const uint32_t mp = kind == 2, mq = kind == 1; // h h, h l, l h
            acc[i][j] = Swap ? __builtin_amdgcn_mfma_f32_32x32x16_f16(f.q[kb][j][mq], f.p[kb][i][mp], acc[i][j], 0, 0, 0)
                             : __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[kb][i][mp], f.q[kb][j][mq], acc[i][j], 0, 0, 0);
        };
        auto fetch = [&](uint32_t buf, Fragments &f) {
            const half_t *base = lds + buf * kStage + lane * 8;
#pragma unroll
            for (uint32_t r = 0; r < kReads; ++r) read(base, f, r);
        };
        auto multiply = [&](const Fragments &f) {
#pragma unroll
            for (uint32_t n = 0; n < kProducts; ++n) product(f, n);
        };
        auto after = [&](uint32_t buf) { return buf + 1 == kBufs ? 0 : buf + 1; };
        for (uint32_t s = 0; s < kBufs && s < stages; ++s) load_stage(s * kKb, s);
        Fragments even, odd;
        if (stages < kBufs) wait_and_meet<0>();
        else wait_and_meet<(kBufs - 1) * kLoads>();
        fetch(0, even);
        uint32_t buf = 0; // of the stage in registers
        // One turn: the stage in `now` is multiplied while the next one is read from LDS into `next` and the
        // one kBufs further on its way to where the stage in `now` was.  Before that, this wavefront's loads of
        // the next stage have landed (kBufs - 2 later ones may be on their way) and its reads of `now` are done; behind
        // the barrier that holds for all four.
        auto turn = [&](uint32_t s, const Fragments &now, Fragments &next) {
            wait_and_meet<(kBufs - 2) * kLoads>();
            const half_t *base = lds + after(buf) * kStage + lane * 8;
#pragma unroll
            for (uint32_t r = 0; r < kReads; ++r) { // reads and loads in between the products
                read(base, next, r);
                if (r * kLoads / kReads != (r + 1) * kLoads / kReads) load_part((s + kBufs) * kKb, buf, r * kLoads / kReads);
#pragma unroll
                for (uint32_t n = r * kProducts / kReads; n < (r + 1) * kProducts / kReads; ++n) product(now, n);
                __builtin_amdgcn_sched_barrier(0); // left alone, the compiler gathers the reads behind the products
            }
            buf = after(buf);
        };
        uint32_t s = 0;
        for (; s + kBufs + 1 < stages; s += 2) {
            turn(s, even, odd);
            turn(s + 1, odd, even);
        }
        for (;; ++s) { // the last stages: at most kBufs + 1 of them, the registers changing hands by copy
            if (s + 1 == stages) break;
            wait_and_meet<0>();
            fetch(after(buf), odd);
            if (s + kBufs < stages) load_stage((s + kBufs) * kKb, buf);
            __builtin_amdgcn_sched_barrier(0);
            multiply(even);
            buf = after(buf);
            even = odd;
        }
        multiply(even);
    }
};

// Elements of one term of a matrix of so many blocks of 16 rows and columns
__device__ __forceinline__ uint64_t plane_of(uint32_t row_blocks, uint32_t col_blocks) { return (uint64_t)row_blocks * col_blocks * 256; }

// Where a lane's four values 4g..4g+3 of a 32 x 32 block lie in an operand: row block `rb`, columns 32 cb + 8g + 4 (lane / 32)..+3
__device__ __forceinline__ uint64_t quad_at(uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t g, uint32_t lane) {
    return ((uint64_t)rb * k_blocks_stored + 2 * cb + (g >> 1)) * kBlk + ((g & 1) * 32 + (lane & 31)) * 8 + 4 * (lane >> 5);
}

// What a lane holds of a 32 x 32 block as it is stored, and its value
struct RawBlock {
    v4h h[4], l[4];
};
__device__ __forceinline__ RawBlock load_block(const half_t *m, uint64_t plane, uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t lane) {
    RawBlock out;
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g) {
        const half_t *at = m + quad_at(rb, cb, k_blocks_stored, g, lane);
        out.h[g] = *(const FSTX_GLOBAL v4h *)at;
        out.l[g] = *(const FSTX_GLOBAL v4h *)(at + plane);
    }
    return out;
}
__device__ __forceinline__ v16f value_of(const RawBlock &b) {
    v16f out;
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) out[r] = (float)b.h[r / 4][r % 4] + (float)b.l[r / 4][r % 4];
    return out;
}

__device__ __forceinline__ void store_block(half_t *m, uint64_t plane, uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t lane, const half_t (&h)[16],
                                            const half_t (&l)[16]) {
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g) {
        half_t *at = m + quad_at(rb, cb, k_blocks_stored, g, lane);
        v4h vh, vl;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            vh[e] = h[4 * g + e];
            vl[e] = l[4 * g + e];
        }
        *(FSTX_GLOBAL v4h *)at = vh;
        *(FSTX_GLOBAL v4h *)(at + plane) = vl;
    }
}

__device__ __forceinline__ void split(const v16f &v, half_t (&h)[16], half_t (&l)[16]) {
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) {
        // One value for both terms: folded into the product before it, as the compiler otherwise may for one of them, the
        // conversion rounds the unrounded product, now and then to the neighbour of the h that l is the rest of
        // ([129, 129] fp32 2e-5 off instead of 1.2e-6).
        float x = v[r];
        asm("" : "+v"(x));
        h[r] = (half_t)x;
        l[r] = (half_t)(x - (float)h[r]);
    }
}

// The block with rows and columns exchanged between the lanes: a product with the identity whose
// k order is that of the values a lane holds (k slot e of half s is column 16 s + 8 (e / 4) + 4 (lane / 32) + e % 4).
__device__ __forceinline__ void exchange(const half_t (&in)[16], half_t (&out)[16], uint32_t lane) {
    v16f d = {};
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        v8h x, one;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            x[e] = in[8 * s + e];
            one[e] = (lane & 31) == 16 * s + 8 * (e / 4) + 4 * (lane >> 5) + e % 4 ? (half_t)1.0f : (half_t)0.0f;
        }
        d = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, one, d, 0, 0, 0);
    }
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) out[r] = (half_t)d[r];
}

// X and X^T from G: a wavefront takes a 32 x 32 block, its lanes along the side along which memory runs.
__global__ __launch_bounds__(256) void first_operands_kernel(const Jobs t) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job job = fetch_job(t, ji);
    const uint32_t lane = threadIdx.x & 63;
    const View g = view_of(job);
    const uint32_t p_blocks = pad_to(job.p, kPadP) / 16, q_blocks = pad_to(job.q, kPadQ) / 16;
    const uint32_t across = (g.x_cols ? q_blocks : p_blocks) / 2, down = (g.x_cols ? p_blocks : q_blocks) / 2;
    const uint32_t blk = (blockIdx.x - t.first[ji]) * 4 + threadIdx.x / 64;
    if (blk >= across * down) return;
    const uint32_t rb = blk / across, cb = blk - rb * across;
    const uint32_t col = cb * 32 + (lane & 31);
    auto row_of = [&](uint32_t r) { return rb * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4; };
    float x[16];
    load_elems<16>(job.src, job.type, x, [&](uint32_t r) { return (uint64_t)row_of(r) * g.row_stride + (uint64_t)col * g.col_stride; },
                   [&](uint32_t r) { return row_of(r) < g.rows && col < g.cols; });
    const FSTX_GLOBAL Plan *plan = (const FSTX_GLOBAL Plan *)reinterpret_cast<const Plan *>(job.partials);
    const float factor = plan->factor;
    const int exponent = plan->exponent;
    v16f v;
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) v[r] = __builtin_ldexpf(x[r], exponent) * factor;
    half_t h[16], l[16], ht[16], lt[16];
    split(v, h, l);
    exchange(h, ht, lane);
    exchange(l, lt, lane);
    const uint64_t plane = plane_of(p_blocks, q_blocks);
    if (g.x_cols) {
        store_block(job.xt0, plane, cb, rb, p_blocks, lane, h, l);
        store_block(job.x, plane, rb, cb, q_blocks, lane, ht, lt);
    } else {
        store_block(job.x, plane, cb, rb, q_blocks, lane, h, l);
        store_block(job.xt0, plane, rb, cb, p_blocks, lane, ht, lt);
    }
}

enum Phase : uint32_t { kGram, kPoly, kApply, kLast };

struct At {
    uint32_t step;
    __device__ uint32_t current() const { return step & 1; } // which of xt0, xt1 is the current one
};

// result = own * (what is there) + product * (sum of the products)
struct Coefficients {
    float own, product;
};
template <uint32_t kPhase> __device__ __forceinline__ Coefficients coefficients_of(const Job &job, const At &at) {
    if constexpr (kPhase == kGram) {
        return Coefficients{0.0f, kScaleA / (job.scale * job.scale)};
    } else {
        const FSTX_GLOBAL StepPlan &p = ((const FSTX_GLOBAL Plan *)reinterpret_cast<const Plan *>(job.partials))->step[at.step];
        return kPhase == kPoly ? Coefficients{p.poly_own, p.poly_product} : Coefficients{p.apply_own, p.apply_product};
    }
}

// Tiles of a symmetric matrix that reach on or below the diagonal, row by row: row i has kAspect (i + 1) of
// them, a tile being kAspect times as high as wide.
template <uint32_t kAspect> __host__ __device__ inline uint32_t triangle_tiles(uint32_t rows) { return kAspect * (rows * (rows + 1) / 2); }
template <uint32_t kAspect> __device__ __forceinline__ void triangle(uint32_t t, uint32_t &i, uint32_t &j) {
    i = (uint32_t)((sqrtf(8.0f * (float)(t / kAspect) + 1.0f) - 1.0f) * 0.5f);
    while (triangle_tiles<kAspect>(i) > t) --i;
    while (triangle_tiles<kAspect>(i + 1) <= t) ++i;
    j = t - triangle_tiles<kAspect>(i);
}

// own x + product v to rows first + 0..3, 8..11, 16..19, 24..27 of the destination, one column per lane
template <typename T>
__device__ __forceinline__ void store_rows(char *at, uint32_t col, uint64_t pitch, uint32_t first, uint32_t rows, const v16f &x, const v16f &v, float own,
                                           float product) {
    FSTX_GLOBAL char *to = (FSTX_GLOBAL char *)at + (uint64_t)col * sizeof(T);
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) {
        const uint32_t row = 8 * (r / 4) + r % 4;
        if (first + row < rows) *(FSTX_GLOBAL T *)(to + row * pitch) = (T)(own * x[r] + product * v[r]);
    }
}

// What is there already where block (rb, cb) of a product goes: A's block, or X's
template <uint32_t kPhase>
__device__ __forceinline__ RawBlock own_block(const Job &job, const At &step, uint32_t rb, uint32_t cb, uint32_t lane) {
    const uint32_t p_blocks = pad_to(job.p, kPadP) / 16, q_blocks = pad_to(job.q, kPadQ) / 16; // as stored
    if constexpr (kPhase == kGram) {
        return RawBlock{};
    } else if constexpr (kPhase == kLast) {
        const bool flipped = job.flipped;
        return load_block(pick<const half_t *>(flipped, job.x, pick(step.current(), job.xt1, job.xt0)), plane_of(p_blocks, q_blocks), pick(flipped, rb, cb), pick(flipped, cb, rb),
                          pick(flipped, q_blocks, p_blocks), lane);
    } else {
        return load_block(kPhase == kPoly ? job.a : job.x, plane_of(p_blocks, kPhase == kPoly ? p_blocks : q_blocks), rb, cb,
                          kPhase == kPoly ? p_blocks : q_blocks, lane);
    }
}

// What becomes of one 32 x 32 block of a product. `v` is laid out with lanes along rows (the transposed
// product), in the last step of a matrix that is not flipped with lanes along columns.
template <uint32_t kPhase>
__device__ __forceinline__ void finish_block(const Job &job, const At &step, const Coefficients &c, uint32_t rb, uint32_t cb, v16f v, const RawBlock &there, uint32_t lane) {
    const uint32_t p_blocks = pad_to(job.p, kPadP) / 16, q_blocks = pad_to(job.q, kPadQ) / 16;
    if constexpr (kPhase == kLast) {
        // lanes run along the contiguous side of the destination: 64 or 128 contiguous bytes per row
        const bool flipped = job.flipped;
        const uint32_t along = pick(flipped, rb, cb) * 32 + (lane & 31), first = pick(flipped, cb, rb) * 32 + 4 * (lane >> 5);
        const uint32_t rows = pick(flipped, job.q, job.p), cols = pick(flipped, job.p, job.q);
        if (along >= cols) return;
        const v16f x = value_of(there);
        char *at = job.dst + (uint64_t)first * job.dst_pitch;
        if (job.type == FSTX_F32) store_rows<float>(at, along, job.dst_pitch, first, rows, x, v, c.own, c.product);
        else if (job.type == FSTX_BF16) store_rows<__bf16>(at, along, job.dst_pitch, first, rows, x, v, c.own, c.product);
        else store_rows<half_t>(at, along, job.dst_pitch, first, rows, x, v, c.own, c.product);
    } else {
        if constexpr (kPhase == kGram) {
            v *= c.product;
        } else {
            const v16f own = value_of(there);
#pragma unroll
            for (uint32_t r = 0; r < 16; ++r) v[r] = c.own * own[r] + c.product * v[r];
        }
        half_t h[16], l[16], ht[16], lt[16];
        split(v, h, l);
        half_t *to = kPhase == kGram ? job.a : kPhase == kPoly ? job.b : job.x;
        const uint64_t plane = plane_of(p_blocks, kPhase == kApply ? q_blocks : p_blocks);
        store_block(to, plane, rb, cb, kPhase == kApply ? q_blocks : p_blocks, lane, h, l);
        if (kPhase == kApply || cb != rb) {
            exchange(h, ht, lane);
            exchange(l, lt, lane);
            store_block(kPhase == kApply ? pick(step.current(), job.xt0, job.xt1) : to, plane, cb, rb, p_blocks, lane, ht, lt);
        }
    }
}

template <uint32_t kPhase> __host__ __device__ constexpr bool symmetric() { return kPhase == kGram || kPhase == kPoly; }

template <uint32_t kPhase, uint32_t TR, uint32_t TC> __host__ __device__ inline uint32_t tiles_of(uint32_t p, uint32_t q) {
    const uint32_t pt = (p + TR - 1) / TR, qt = (q + TC - 1) / TC;
    return symmetric<kPhase>() ? triangle_tiles<TR / TC>(pt) : pt * qt;
}

template <uint32_t kPhase, uint32_t TR, uint32_t TC>
__device__ __forceinline__ void place_of(const Job &job, uint32_t tile, uint32_t &ti, uint32_t &tj) {
    if constexpr (symmetric<kPhase>()) {
        triangle<TR / TC>(tile, ti, tj);
    } else { // columns of up to eight tiles, so that the tiles at work share both operands
        const uint32_t pt = (job.p + TR - 1) / TR, qt = (job.q + TC - 1) / TC;
        const uint32_t group = tile / (8 * qt), first = group * 8, height = pt - first < 8 ? pt - first : 8;
        const uint32_t in = tile - group * 8 * qt;
        ti = first + in % height;
        tj = in / height;
    }
}

template <uint32_t kPhase, uint32_t TR, uint32_t TC>
__global__ __launch_bounds__(256, (Product<TR, TC>::kWaves)) void newton_schulz_kernel(const Jobs t, const Deal deal, const At step) {
    typedef Product<TR, TC> Prod;
    constexpr uint32_t kNR = Prod::kNR, kNC = Prod::kNC;
    __shared__ __attribute__((aligned(1024))) half_t lds[Prod::kBufs * Prod::kStage];
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job job = fetch_job(t, ji);
    const uint32_t lb = blockIdx.x - t.first[ji], whole = deal.whole[ji];
    const uint32_t whole_wgs = (whole + (1u << deal.dies_log2) - 1) >> deal.dies_log2 << deal.dies_log2;
    uint32_t tile, piece = 0, part = 0;
    const bool partial = lb >= whole_wgs;
    if (!partial) {
        if (!fstx_gather::tile_for_die(lb, whole, deal.dies_log2, tile)) return;
    } else {
        piece = lb - whole_wgs;
        tile = whole + piece / deal.split;
        part = piece % deal.split;
    }
    uint32_t ti, tj;
    place_of<kPhase, TR, TC>(job, tile, ti, tj);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    // the operands' tiles, and the k that are summed here
    const uint32_t stored = (kPhase == kGram ? pad_to(job.q, kPadQ) : pad_to(job.p, kPadP)) / 16;
    const uint32_t stages = pad_to(kPhase == kGram ? job.q : job.p, kStepPad) / 16 / Prod::kKb;
    const uint32_t from = partial ? (uint32_t)((uint64_t)stages * part / deal.split) : 0;
    const uint32_t to = partial ? (uint32_t)((uint64_t)stages * (part + 1) / deal.split) : stages;
    const half_t *left = kPhase == kGram ? job.x : kPhase == kPoly ? job.a : job.b;
    const half_t *right = kPhase == kGram ? job.x : kPhase == kPoly ? job.a : pick(step.current(), job.xt1, job.xt0);
    const uint64_t row = (uint64_t)stored * kBlk, k0 = (uint64_t)from * Prod::kKb * kBlk;
    const uint32_t p_blocks = pad_to(job.p, kPadP) / 16, q_blocks = pad_to(job.q, kPadQ) / 16;
    const uint64_t left_plane = plane_of(p_blocks, kPhase == kGram ? q_blocks : p_blocks);
    const uint64_t right_plane = plane_of(p_blocks, kPhase == kPoly ? p_blocks : q_blocks);
    left += ti * (TR / 32) * row + k0;
    right += tj * (TC / 32) * row + k0;
    v16f acc[kNR][kNC] = {};
    if (kPhase == kLast && !job.flipped) Prod::template run<false>(left, right, left_plane, right_plane, stored, to - from, lds, acc);
    else Prod::template run<true>(left, right, left_plane, right_plane, stored, to - from, lds, acc);

    if (partial) {
        float *out = deal.sums + ((uint64_t)deal.slot[ji] + piece) * (TR * TC) + wave * (kNR * kNC * 1024) + lane * 4;
#pragma unroll
        for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
            for (uint32_t j = 0; j < kNC; ++j)
#pragma unroll
                for (uint32_t g = 0; g < 4; ++g)
                    *(FSTX_GLOBAL v4f *)(out + (i * kNC + j) * 1024 + g * 256) =
                        v4f{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        return;
    }
    // The blocks of one row of blocks: what is there already is read for the row after it before anything is
    // written (a load behind a store would wait its turn), so that its latency is paid once.
    const uint32_t rb0 = ti * (TR / 32) + (wave >> 1) * kNR, cb0 = tj * (TC / 32) + (wave & 1) * kNC;
    RawBlock there[2][kNC];
    auto fetch_row = [&](uint32_t i) {
#pragma unroll
        for (uint32_t j = 0; j < kNC; ++j)
            if (!symmetric<kPhase>() || cb0 + j <= rb0 + i) there[i % 2][j] = own_block<kPhase>(job, step, rb0 + i, cb0 + j, lane);
    };
    fetch_row(0);
    const Coefficients c = coefficients_of<kPhase>(job, step);
#pragma unroll
    for (uint32_t i = 0; i < kNR; ++i) {
        if (i + 1 < kNR) fetch_row(i + 1);
#pragma unroll
        for (uint32_t j = 0; j < kNC; ++j)
            if (!symmetric<kPhase>() || cb0 + j <= rb0 + i) // above the diagonal: written as the mirror of (cb, rb)
                finish_block<kPhase>(job, step, c, rb0 + i, cb0 + j, acc[i][j], there[i % 2][j], lane);
    }
}

// The tiles whose sums came in pieces: a wavefront per 32 x 32 block adds them in order.
template <uint32_t kPhase, uint32_t TR, uint32_t TC>
__global__ __launch_bounds__(64) void join_pieces_kernel(const Jobs t, const Deal deal, const At step) {
    typedef Product<TR, TC> Prod;
    constexpr uint32_t kBlocks = TR / 32 * (TC / 32);
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job job = fetch_job(t, ji);
    const uint32_t lb = blockIdx.x - t.first[ji], in = lb % kBlocks, nth = lb / kBlocks;
    uint32_t ti, tj;
    place_of<kPhase, TR, TC>(job, deal.whole[ji] + nth, ti, tj);
    const uint32_t ri = in / (TC / 32), ci = in % (TC / 32), rb = ti * (TR / 32) + ri, cb = tj * (TC / 32) + ci;
    if (symmetric<kPhase>() && cb > rb) return;
    const uint32_t wave = ri / Prod::kNR * 2 + ci / Prod::kNC, i = ri % Prod::kNR, j = ci % Prod::kNC;
    const float *at = deal.sums + ((uint64_t)deal.slot[ji] + (uint64_t)nth * deal.split) * (TR * TC) +
                      ((wave * Prod::kNR + i) * Prod::kNC + j) * 1024 + threadIdx.x * 4;
    const RawBlock there = own_block<kPhase>(job, step, rb, cb, threadIdx.x);
    const Coefficients c = coefficients_of<kPhase>(job, step);
    v16f v = {};
#pragma unroll 4
    for (uint32_t s = 0; s < deal.split; ++s, at += TR * TC)
#pragma unroll
        for (uint32_t g = 0; g < 4; ++g) {
            const v4f part = *(const FSTX_GLOBAL v4f *)(at + g * 256);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[4 * g + e] += part[e];
        }
    finish_block<kPhase>(job, step, c, rb, cb, v, there, threadIdx.x);
}

// ------------------------------------------------------------ slim matrices
//
// Up to 32 rows the whole iteration fits one workgroup when it is done on the Gram matrix M = G G^T in 64 bits: X is Q G with
// Q a polynomial of M, so that a step is P = a I + b A + c A^2, Q <- P Q, A <- P A P, which all commute.  Squaring the
// singular values costs half of the digits, which 64 bits have to spare and two fp16 terms have not: of a [1, 1] fp32
// update they got 1.6e-6 of the value wrong, and this 4e-8.
//
// P A P loses that A is X X^T, whose eigenvalues are never negative: what rounding leaves of an eigenvalue of zero, +-2^-53,
// grows by a^2 a step like that of any small direction, but a negative one without end (rank 1 and twenty steps of a = 3.4445: 1e40).
// So steps are taken in runs in which a direction grows by kSlimGrowth at most, 2^26 times 2^-53 of an eigenvalue; between two runs
// X = Q X is made, in 64 bits, and A taken from it anew.  The nine steps of a polar factor are one run; fourteen steps of a = 15/8
// too (a [32, 4096] fp32 update 45 us), fifteen are two (67 us), sixty-four five (197 us).
//
// A run is three launches and reads the update twice: with five steps a [1, 700] fp32 update takes 23 us instead of 101, [32, 4096] 32 instead of 119 and
// [32, 28672] 50 instead of 287.  At 64 rows one workgroup's products would take as long as the launches they save.
// The partial sums of M are added in a fixed order.

constexpr uint32_t kSlim = 32;      // rows at most
constexpr uint32_t kSlimJobs = 32;
constexpr uint32_t kSlimParts = 128; // workgroups that share the columns of one matrix
constexpr double kSlimGrowth = 8192.0;

struct alignas(32) SlimJob {
    const char *src;
    char *dst;
    double *grams; // n_parts of kSlim x kSlim
    double *q;     // kSlim x kSlim
    double *x;     // p x q_cols, what the runs before have made of X (more than one run only)
    uint64_t x_row, x_col, dst_pitch; // elements, elements, bytes
    uint32_t p, q_cols, type, flipped, n_parts, pad;
};
struct SlimJobs {
    SlimJob job[kSlimJobs];
    uint32_t first[kSlimJobs];
};
static_assert(sizeof(SlimJobs) <= 3328, "fits the kernel arguments");

__device__ __forceinline__ uint32_t slim_job_of(const SlimJobs &t, uint32_t b) {
    uint32_t ji = 0;
#pragma unroll
    for (uint32_t i = 1; i < kSlimJobs; ++i) ji += b >= t.first[i];
    return ji;
}

// v_mfma_f64_16x16x4: lane l holds A[l % 16][l / 16] and B[l / 16][l % 16], and D[4 r + l / 16][l % 16] in element r.
using f64x4 = __attribute__((__vector_size__(4 * sizeof(double)))) double;
__device__ __forceinline__ f64x4 mfma64(double a, double b, f64x4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

// Elements of X: in the first run those of G, in the type they have, later 64-bit ones
template <bool kFirst> struct SlimElem { typedef float type; };
template <> struct SlimElem<false> { typedef double type; };
template <bool kFirst, uint32_t N, typename Row, typename Col>
__device__ __forceinline__ void load_slim(const SlimJob &job, typename SlimElem<kFirst>::type (&x)[N], Row row, Col col) {
    auto there = [&](uint32_t k) { return row(k) < job.p && col(k) < job.q_cols; };
    if constexpr (kFirst) {
        load_elems<N>(job.src, job.type, x, [&](uint32_t k) { return row(k) * job.x_row + col(k) * job.x_col; }, there);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) x[k] = *(const FSTX_GLOBAL double *)(job.x + (there(k) ? row(k) * job.q_cols + col(k) : 0));
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) x[k] = there(k) ? x[k] : 0.0;
    }
}

// A workgroup's share of M, 64 columns at a time, the next ones on their way while these are multiplied; a wave takes 16 of
// them and the tiles on and below the diagonal.
template <bool kFirst> __global__ __launch_bounds__(256) void slim_gram_kernel(const SlimJobs t) {
    typedef typename SlimElem<kFirst>::type elem;
    constexpr uint32_t kWide = 64, kLoads = kSlim * kWide / 256;
    __shared__ union {
        elem x[kSlim][kWide + 4];
        double sums[4][256];
    } lds;
    const uint32_t ji = slim_job_of(t, blockIdx.x);
    const SlimJob &job = t.job[ji];
    const uint32_t me = blockIdx.x - t.first[ji], p = job.p, n = job.q_cols, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const bool across = kFirst && job.x_row < job.x_col; // columns of X lie along memory
    elem next[kLoads];
    auto row_of = [&](uint32_t k) { return across ? (threadIdx.x + 256 * k) % kSlim : (threadIdx.x + 256 * k) / kWide; };
    auto col_of = [&](uint32_t k) { return across ? (threadIdx.x + 256 * k) / kSlim : (threadIdx.x + 256 * k) % kWide; };
    auto load = [&](uint64_t c0) {
        load_slim<kFirst>(job, next, [&](uint32_t k) { return (uint64_t)row_of(k); }, [&](uint32_t k) { return c0 + col_of(k); });
    };
    f64x4 acc[3] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
    const uint64_t stride = (uint64_t)job.n_parts * kWide;
    load((uint64_t)me * kWide);
    for (uint64_t c0 = (uint64_t)me * kWide; c0 < n; c0 += stride) {
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kLoads; ++k) lds.x[row_of(k)][col_of(k)] = next[k];
        __syncthreads();
        if (c0 + stride < n) load(c0 + stride);
#pragma unroll
        for (uint32_t k = 0; k < 16; k += 4) {
            const double a = lds.x[lane % 16][wave * 16 + k + lane / 16];
            acc[0] = mfma64(a, a, acc[0]);
            if (p > 16) {
                const double b = lds.x[16 + lane % 16][wave * 16 + k + lane / 16];
                acc[1] = mfma64(b, a, acc[1]);
                acc[2] = mfma64(b, b, acc[2]);
            }
        }
    }
    double *out = job.grams + (uint64_t)me * kSlim * kSlim;
#pragma unroll
    for (uint32_t tile = 0; tile < 3; ++tile) { // the waves' sums, in order
        __syncthreads();
        for (uint32_t r = 0; r < 4; ++r) lds.sums[wave][(4 * r + lane / 16) * 16 + lane % 16] = acc[tile][r];
        __syncthreads();
        const uint32_t i = threadIdx.x / 16 + (tile > 0 ? 16 : 0), j = threadIdx.x % 16 + (tile > 1 ? 16 : 0);
        const double sum = lds.sums[0][threadIdx.x] + lds.sums[1][threadIdx.x] + lds.sums[2][threadIdx.x] + lds.sums[3][threadIdx.x];
        out[i * kSlim + j] = sum;
        if (tile == 1) out[j * kSlim + i] = sum;
    }
}

// One workgroup per matrix: Q.  Rows and columns from p on are zero throughout (those of P are not, but meet only zeros).
__global__ __launch_bounds__(512) void slim_steps_kernel(const SlimJobs t, const Steps steps) {
    using Matrix = double[kSlim][kSlim + 1];
    __shared__ Matrix a, q, m, w;
    const SlimJob &job = t.job[blockIdx.x];
    const uint32_t p = job.p, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t i0 = wave / 2 % 2 * 16, j0 = wave % 2 * 16, row = i0 + lane / 16, col = j0 + lane % 16;
    for (uint32_t e = threadIdx.x; e < kSlim * kSlim; e += 512) {
        double sum = 0;
#pragma unroll 8
        for (uint32_t k = 0; k < job.n_parts; ++k) sum += job.grams[(uint64_t)k * kSlim * kSlim + e];
        a[e / kSlim][e % kSlim] = sum;
    }
    __syncthreads();
    double trace = 0;
    for (uint32_t i = 0; i < p; ++i) trace += a[i][i];
    const double factor = steps.first ? 1.0 / (sqrt(trace) + (double)steps.eps) : 1.0;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < kSlim * kSlim; e += 512) {
        a[e / kSlim][e % kSlim] *= factor * factor;
        q[e / kSlim][e % kSlim] = e / kSlim == e % kSlim && e % kSlim < p ? factor : 0.0;
    }
    __syncthreads();
    // a wave's tile of x y; all of these are symmetric, so that y's rows serve as its columns
    auto product = [&](const Matrix &x, const Matrix &y) {
        f64x4 d = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t k = 0; k < kSlim; k += 4) d = mfma64(x[i0 + lane % 16][k + lane / 16], y[j0 + lane % 16][k + lane / 16], d);
        return d;
    };
    const bool first = wave < 4;
    const bool mine = i0 < p && j0 < p;
    for (uint32_t s = 0; s < steps.n; ++s) {
        const double ca = steps.c[3 * s], cb = steps.c[3 * s + 1], cc = steps.c[3 * s + 2];
        f64x4 d;
        if (first) {
            d = product(a, a);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
                m[row + 4 * r][col] = (row + 4 * r == col ? ca : 0.0) + cb * a[row + 4 * r][col] + cc * d[r];
        }
        __syncthreads();
        if (mine) d = first ? product(m, q) : product(m, a);
        __syncthreads();
        if (mine) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) (first ? q : w)[row + 4 * r][col] = d[r];
        }
        __syncthreads();
        if (first && mine) {
            d = product(w, m);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) a[row + 4 * r][col] = d[r];
        }
        __syncthreads();
    }
    for (uint32_t e = threadIdx.x; e < kSlim * kSlim; e += 512) job.q[e] = q[e / kSlim][e % kSlim];
}

// Q X, into the result or, between two runs, into X: 16 columns by wave, read whole before they are written
template <bool kFirst, bool kEnd> __global__ __launch_bounds__(256) void slim_apply_kernel(const SlimJobs t) {
    const uint32_t ji = slim_job_of(t, blockIdx.x);
    const SlimJob &job = t.job[ji];
    const uint32_t p = job.p, lane = threadIdx.x % 64, from = lane / 16;
    const uint64_t c = (uint64_t)(blockIdx.x - t.first[ji]) * 64 + threadIdx.x / 64 * 16 + lane % 16;
    typename SlimElem<kFirst>::type g[kSlim / 4];
    load_slim<kFirst>(job, g, [&](uint32_t k) { return (uint64_t)(4 * k + from); }, [&](uint32_t) { return c; });
#pragma unroll
    for (uint32_t i0 = 0; i0 < kSlim; i0 += 16) {
        if (i0 >= p) break;
        f64x4 d = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t k = 0; k < kSlim / 4; ++k) d = mfma64(job.q[(i0 + lane % 16) * kSlim + 4 * k + from], g[k], d);
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint64_t i = i0 + 4 * r + from;
            if (i >= p || c >= job.q_cols) continue;
            if constexpr (!kEnd) {
                *(FSTX_GLOBAL double *)(job.x + i * job.q_cols + c) = d[r];
                continue;
            }
            char *at = job.dst + (job.flipped ? c : i) * job.dst_pitch;
            const uint64_t along = job.flipped ? i : c;
            if (job.type == FSTX_F32) ((FSTX_GLOBAL float *)at)[along] = (float)d[r];
            else if (job.type == FSTX_BF16) ((FSTX_GLOBAL __bf16 *)at)[along] = (__bf16)(float)d[r];
            else ((FSTX_GLOBAL half_t *)at)[along] = (half_t)(float)d[r];
        }
    }
}

// --------------------------------------------------------------- host side

constexpr uint64_t kMaxSide = 1u << 20;
constexpr uint64_t kChunkBytes = 4ull << 30; // matrices of one set of launches share this much workspace, or one has its own
constexpr uint32_t kMaxSteps = 64;

inline bool type_ok(uint32_t t) { return t == FSTX_F32 || t == FSTX_F16 || t == FSTX_BF16; }
inline uint32_t size_of(uint32_t t) { return t == FSTX_F32 ? 4 : 2; }
inline bool empty(const fstx_orthogonalize_desc &d) { return d.rows == 0 || d.cols == 0; }
inline bool slim(const fstx_orthogonalize_desc &d) { return !empty(d) && (d.rows < d.cols ? d.rows : d.cols) <= kSlim; }

struct Sides {
    uint64_t p, q, pp, qp;
    explicit Sides(const fstx_orthogonalize_desc &d)
        : p(d.rows < d.cols ? d.rows : d.cols), q(d.rows < d.cols ? d.cols : d.rows), pp((p + kPadP - 1) / kPadP * kPadP), qp((q + kPadQ - 1) / kPadQ * kPadQ) {}
    uint64_t bytes() const { return (3 * pp * qp + 2 * pp * pp) * 2 * sizeof(half_t) + kPartials * sizeof(double); }
};

using fstx_overlap::Block;
using fstx_overlap::block_of;
Block dst_of(const fstx_orthogonalize_desc &d) { return block_of(d.dst, d.rows, d.cols, d.dst_pitch, size_of(d.type)); }
Block src_of(const fstx_orthogonalize_desc &d) { return block_of(d.src, d.rows, d.src_row_stride, d.cols, d.src_col_stride, size_of(d.type)); }

int check(const fstx_orthogonalize_desc *descs, uint32_t n) {
    if (n && !descs) return -FSTX_E_INVAL;
    for (uint32_t i = 0; i < n; ++i) {
        const fstx_orthogonalize_desc &d = descs[i];
        if (!type_ok(d.type)) return -FSTX_E_INVAL;
        if (empty(d)) continue;
        if (d.rows > kMaxSide || d.cols > kMaxSide || Sides(d).p > 65536) return -FSTX_E_RANGE;
        if ((d.src_row_stride | d.src_col_stride | d.dst_pitch) >> 40) return -FSTX_E_RANGE;
        if (!d.dst || !d.src || (uintptr_t)d.dst % size_of(d.type) || (uintptr_t)d.src % size_of(d.type)) return -FSTX_E_INVAL;
        if (d.rows > 1 && d.dst_pitch < d.cols) return -FSTX_E_INVAL;
        // exactly in place, or apart
        const bool in_place = d.dst == d.src && (d.rows == 1 || d.src_row_stride == d.dst_pitch) && (d.cols == 1 || d.src_col_stride == 1);
        if (!in_place && fstx_overlap::overlap(dst_of(d), src_of(d))) return -FSTX_E_INVAL;
    }
    fstx_overlap::List list(2ull * n);
    if (!list.at) return -ENOMEM;
    for (uint32_t i = 0; i < n; ++i) {
        if (empty(descs[i])) continue;
        list.add(dst_of(descs[i]), i, fstx_overlap::kWritten);
        list.add(src_of(descs[i]), i, fstx_overlap::kSource);
    }
    if (fstx_overlap::any_conflict(list.at, list.n)) return -FSTX_E_INVAL;
    return 0;
}

inline float power_of_two_below(double v) { return (float)ldexp(1.0, (int)floor(log2(v))); }

// What the tile sizes cost, measured (microseconds): a launch and the ends of a workgroup; 16 k of one workgroup when
// kResident share a compute unit, per workgroup, and when it is alone there.
template <uint32_t TR, uint32_t TC> struct Cost;
#define FSTX_COST(TR, TC, RESIDENT, FIXED, SHARED, ALONE)                                                     \
    template <> struct Cost<TR, TC> {                                                                         \
        static constexpr uint32_t kResident = RESIDENT;                                                              \
        static constexpr double kFixed = FIXED, kShared = SHARED, kAlone = ALONE;                                    \
    };
FSTX_COST(64, 64, 2, 2.5, 0.12, 0.15)
FSTX_COST(128, 128, 3, 3.5, 0.355, 0.36)
FSTX_COST(256, 128, 2, 5.0, 0.630, 0.70)
FSTX_COST(256, 256, 1, 8.0, 1.230, 1.230)
#undef FSTX_COST

struct Launcher {
    Jobs t;
    Deal d;
    uint32_t n = 0;
    uint32_t grid = 0;       // of the last deal
    uint64_t sum_tiles = 0;  // tiles of partial sums it takes
    hipStream_t stream = nullptr;
    bool run = false;        // false: only plan, and note how much room partial sums take
    uint64_t sum_bytes = 0;

    // Deals the tiles to workgroups.  Whole rounds take a tile each.  Tiles that are left over would keep a few compute
    // units busy for the time of a whole tile while the others idle: they can be cut along k into pieces instead, as many
    // as there is room for, at the price of a second launch that joins them.  Returns an estimate in microseconds.
    template <uint32_t kPhase, uint32_t TR, uint32_t TC> double deal() {
        typedef Cost<TR, TC> cost;
        uint64_t tiles = 0;
        uint32_t blocks = ~0u, longest = 0; // of 16 k
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t k = pad_to(kPhase == kGram ? t.job[i].q : t.job[i].p, kStepPad) / 16;
            tiles += tiles_of<kPhase, TR, TC>(t.job[i].p, t.job[i].q);
            if (k < blocks) blocks = k;
            if (k > longest) longest = k;
        }
        const uint32_t units = 32u << d.dies_log2;
        auto rounds = [&](uint64_t workgroups) { // time of 16 k for so many workgroups
            const uint64_t full = workgroups / (units * cost::kResident), rest = workgroups % (units * cost::kResident);
            const double last = cost::kShared * (double)((rest + units - 1) / units);
            return (double)full * cost::kResident * cost::kShared + (rest ? last > cost::kAlone ? last : cost::kAlone : 0.0);
        };
        double best = cost::kFixed + longest * rounds(tiles);
        uint32_t split = 1;
        uint64_t whole = tiles;
        for (uint32_t room = units; room <= 2 * units; room += units) {
            const uint64_t left = tiles % room;
            uint64_t cut = left ? room / left : 1;
            if (cut > blocks / 8) cut = blocks / 8; // eight blocks of 16 k at least
            if (cut < 2) continue;
            const double megabytes = (double)(left * cut) * TR * TC * sizeof(float) / 1e6;
            const double time = 2 * cost::kFixed + longest * (rounds(tiles - left) + rounds(left * cut) / (double)cut) + 2.0 + 0.35 * megabytes;
            if (time >= best) continue;
            best = time;
            split = (uint32_t)cut;
            whole = tiles - left;
        }
        d.split = split;
        uint64_t wgs = 0;
        sum_tiles = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const uint64_t mine = tiles_of<kPhase, TR, TC>(t.job[i].p, t.job[i].q), w = mine < whole ? mine : whole;
            whole -= w;
            t.first[i] = (uint32_t)wgs;
            d.whole[i] = (uint32_t)w;
            d.slot[i] = (uint32_t)sum_tiles;
            wgs += (w + (1u << d.dies_log2) - 1) >> d.dies_log2 << d.dies_log2;
            wgs += (mine - w) * split;
            sum_tiles += (mine - w) * split;
        }
        grid = wgs * 256 > 0xffffffffull ? 0 : (uint32_t)wgs;
        return best;
    }

    template <uint32_t kPhase, uint32_t TR, uint32_t TC> int launch(const At &step) {
        deal<kPhase, TR, TC>();
        if (!run) {
            const uint64_t bytes = sum_tiles * TR * TC * sizeof(float);
            if (bytes > sum_bytes) sum_bytes = bytes;
            return grid ? 0 : -FSTX_E_RANGE;
        }
        {
            fstx_internal::Range range("fstx newton_schulz_kernel: phase %u, %u matrices, %u workgroups, tiles of %u x %u", kPhase, n, grid, TR, TC);
            hipLaunchKernelGGL((newton_schulz_kernel<kPhase, TR, TC>), dim3(grid), dim3(256), 0, stream, t, d, step);
            const int rc = fstx_internal::check_launch("newton_schulz_kernel");
            if (rc < 0 || sum_tiles == 0) return rc;
        }
        uint32_t wgs = 0;
        for (uint32_t i = 0; i < n; ++i) {
            t.first[i] = wgs;
            wgs += (tiles_of<kPhase, TR, TC>(t.job[i].p, t.job[i].q) - d.whole[i]) * (TR / 32) * (TC / 32);
        }
        fstx_internal::Range range("fstx join_pieces_kernel: phase %u, %u workgroups", kPhase, wgs);
        hipLaunchKernelGGL((join_pieces_kernel<kPhase, TR, TC>), dim3(wgs), dim3(64), 0, stream, t, d, step);
        return fstx_internal::check_launch("join_pieces_kernel");
    }

    template <uint32_t kPhase> int phase(const At &step) {
        const double t256 = deal<kPhase, 256, 256>(), t128 = deal<kPhase, 256, 128>(), t = deal<kPhase, 128, 128>(), small = deal<kPhase, 64, 64>();
        if (small <= t && small <= t128 && small <= t256) return launch<kPhase, 64, 64>(step);
        if (t <= t128 && t <= t256) return launch<kPhase, 128, 128>(step);
        return t128 <= t256 ? launch<kPhase, 256, 128>(step) : launch<kPhase, 256, 256>(step);
    }

    int steps(uint32_t count) {
        for (uint32_t k = 0; k < count; ++k) {
            const At step{k};
            int rc;
            if ((rc = phase<kGram>(step)) < 0 || (rc = phase<kPoly>(step)) < 0) return rc;
            if ((rc = k + 1 == count ? phase<kLast>(step) : phase<kApply>(step)) < 0) return rc;
        }
        return 0;
    }

    void add(const fstx_orthogonalize_desc &desc, char *at) {
        const Sides s(desc);
        const bool flipped = desc.rows > desc.cols;
        Job &j = t.job[n++];
        j = Job{};
        j.src = static_cast<const char *>(desc.src);
        j.dst = static_cast<char *>(desc.dst);
        const uint64_t xb = s.pp * s.qp * 2 * sizeof(half_t), ab = s.pp * s.pp * 2 * sizeof(half_t);
        j.x = reinterpret_cast<half_t *>(at);
        j.xt0 = reinterpret_cast<half_t *>(at + xb);
        j.xt1 = reinterpret_cast<half_t *>(at + 2 * xb);
        j.a = reinterpret_cast<half_t *>(at + 3 * xb);
        j.b = reinterpret_cast<half_t *>(at + 3 * xb + ab);
        j.partials = reinterpret_cast<double *>(at + 3 * xb + 2 * ab);
        j.x_row = flipped ? desc.src_col_stride : desc.src_row_stride;
        j.x_col = flipped ? desc.src_row_stride : desc.src_col_stride;
        j.dst_pitch = desc.dst_pitch * size_of(desc.type);
        j.p = (uint32_t)s.p;
        j.q = (uint32_t)s.q;
        j.type = desc.type;
        j.flipped = flipped;
        // entries of X are at most about 1.2 (the spectral norm), their mean square is 1 / (p q) at first
        const double mid = sqrt((double)s.p * (double)s.q);
        j.scale = power_of_two_below(mid < 8192.0 ? mid : 8192.0);
        const uint64_t parts = (s.p * s.q + 2047) / 2048;
        j.n_partials = (uint32_t)(parts < kPartials ? parts : kPartials);
    }
};

// The matrices of one set of launches: as many from `first` on as fit.  Returns where the next set begins.
uint32_t next_set(const fstx_orthogonalize_desc *descs, uint32_t n, uint32_t first, char *at, Launcher *set, uint64_t *bytes) {
    *bytes = 0;
    set->n = 0;
    for (uint32_t k = 0; k < kMaxJobs; ++k) set->t.first[k] = 0xffffffffu;
    for (uint32_t i = first; i < n; ++i) {
        if (empty(descs[i]) || slim(descs[i])) continue;
        const uint64_t need = Sides(descs[i]).bytes();
        if (set->n == kMaxJobs || (set->n && *bytes + need > kChunkBytes)) return i;
        set->add(descs[i], at + *bytes);
        *bytes += need;
    }
    return n;
}

Steps steps_of(const float *coefficients, uint32_t n, bool first, float eps) {
    Steps steps = {};
    for (uint32_t i = 0; i < 3 * n; ++i) steps.c[i] = coefficients[i];
    steps.n = n;
    steps.first = first;
    steps.eps = eps;
    return steps;
}

// Where the run of steps that begins with `first` ends
uint32_t slim_run(const float *coefficients, uint32_t count, uint32_t first) {
    double growth = 1.0;
    uint32_t k = first;
    do growth *= fmax(1.0, fabs((double)coefficients[3 * k]));
    while (++k < count && growth * fmax(1.0, fabs((double)coefficients[3 * k])) <= kSlimGrowth);
    return k;
}

// Slim matrices from `first` on, as many as one set of launches takes; returns where the next set begins.
uint32_t slim_set(const fstx_orthogonalize_desc *descs, uint32_t n, bool one_run, uint32_t first, char *at, SlimJobs *t, uint64_t *bytes) {
    uint32_t k = 0;
    *bytes = 0;
    if (t)
        for (uint32_t i = 0; i < kSlimJobs; ++i) {
            t->first[i] = 0xffffffffu;
            t->job[i] = SlimJob{};
        }
    for (uint32_t i = first; i < n; ++i) {
        const fstx_orthogonalize_desc &d = descs[i];
        if (!slim(d)) continue;
        if (k == kSlimJobs) return i;
        const bool flipped = d.rows > d.cols;
        const uint64_t p = flipped ? d.cols : d.rows, q = flipped ? d.rows : d.cols, parts = (q + 255) / 256;
        const uint32_t n_parts = (uint32_t)(parts < kSlimParts ? parts : kSlimParts);
        const uint64_t squares = (uint64_t)(n_parts + 1) * kSlim * kSlim, need = (squares + (one_run ? 0 : (p * q + 31) / 32 * 32)) * sizeof(double);
        if (k && *bytes + need > kChunkBytes) return i;
        if (t) {
            double *space = reinterpret_cast<double *>(at + *bytes);
            t->job[k] = SlimJob{static_cast<const char *>(d.src), static_cast<char *>(d.dst), space + kSlim * kSlim, space, space + squares,
                                flipped ? d.src_col_stride : d.src_row_stride, flipped ? d.src_row_stride : d.src_col_stride,
                                d.dst_pitch * size_of(d.type), (uint32_t)p, (uint32_t)q, d.type, flipped, n_parts, 0};
        }
        *bytes += need;
        ++k;
    }
    return n;
}

template <bool kFirst> int slim_launch(SlimJobs &t, const Steps &steps, bool end, hipStream_t stream) {
    uint32_t n = 0, grid = 0;
    for (; n < kSlimJobs && t.job[n].p; ++n) {
        t.first[n] = grid;
        grid += t.job[n].n_parts;
    }
    fstx_internal::Range range("fstx slim kernels: %u matrices, %u steps", n, steps.n);
    hipLaunchKernelGGL((slim_gram_kernel<kFirst>), dim3(grid), dim3(256), 0, stream, t);
    int rc = fstx_internal::check_launch("slim_gram_kernel");
    if (rc < 0) return rc;
    hipLaunchKernelGGL(slim_steps_kernel, dim3(n), dim3(512), 0, stream, t, steps);
    if ((rc = fstx_internal::check_launch("slim_steps_kernel")) < 0) return rc;
    grid = 0;
    for (uint32_t i = 0; i < n; ++i) {
        t.first[i] = grid;
        grid += (t.job[i].q_cols + 63) / 64;
    }
    if (end) hipLaunchKernelGGL((slim_apply_kernel<kFirst, true>), dim3(grid), dim3(256), 0, stream, t);
    else hipLaunchKernelGGL((slim_apply_kernel<kFirst, false>), dim3(grid), dim3(256), 0, stream, t);
    return fstx_internal::check_launch("slim_apply_kernel");
}

int slim_runs(SlimJobs &t, const float *coefficients, uint32_t count, float eps, hipStream_t stream) {
    for (uint32_t from = 0, to; from < count; from = to) {
        to = slim_run(coefficients, count, from);
        const Steps steps = steps_of(coefficients + 3 * from, to - from, from == 0, eps);
        const int rc = from == 0 ? slim_launch<true>(t, steps, to == count, stream) : slim_launch<false>(t, steps, to == count, stream);
        if (rc < 0) return rc;
    }
    return 0;
}

} // namespace

extern "C" int64_t fstx_orthogonalize_workspace(const fstx_orthogonalize_desc *descs, uint32_t n, const float *coefficients, uint32_t steps) {
    const int rc = check(descs, n);
    if (rc < 0) return rc;
    if (steps < 1 || steps > kMaxSteps || !coefficients) return -FSTX_E_INVAL;
    for (uint32_t k = 0; k < 3 * steps; ++k)
        if (!isfinite(coefficients[k])) return -FSTX_E_INVAL;
    const bool one_run = slim_run(coefficients, steps, 0) == steps;
    uint64_t most = 0;
    for (uint32_t first = 0; first < n;) {
        uint64_t bytes;
        first = slim_set(descs, n, one_run, first, nullptr, nullptr, &bytes);
        if (bytes > most) most = bytes;
    }
    for (uint32_t first = 0; first < n;) {
        Launcher set;
        set.d.dies_log2 = fstx_internal::dies_log2();
        uint64_t bytes;
        first = next_set(descs, n, first, nullptr, &set, &bytes);
        if (set.n == 0) break;
        const int planned = set.steps(steps);
        if (planned < 0) return planned;
        if (bytes + set.sum_bytes > most) most = bytes + set.sum_bytes;
    }
    return (int64_t)most;
}

extern "C" int fstx_orthogonalize(const fstx_orthogonalize_desc *descs, uint32_t n, const float *coefficients, uint32_t steps, float eps,
                                  void *workspace, uint64_t workspace_bytes, void *stream) {
    const int64_t need = fstx_orthogonalize_workspace(descs, n, coefficients, steps);
    if (need < 0) return (int)need;
    if (!(eps >= 0) || !isfinite(eps)) return -FSTX_E_INVAL;
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (uint64_t)need)) return -FSTX_E_INVAL;
    const bool one_run = slim_run(coefficients, steps, 0) == steps;
    for (uint32_t first = 0; first < n;) {
        SlimJobs t;
        uint64_t bytes;
        first = slim_set(descs, n, one_run, first, static_cast<char *>(workspace), &t, &bytes);
        if (bytes == 0) continue;
        const int rc = slim_runs(t, coefficients, steps, eps, static_cast<hipStream_t>(stream));
        if (rc < 0) return rc;
    }
    const Steps all = steps_of(coefficients, steps, true, eps);
    for (uint32_t first = 0; first < n;) {
        Launcher set;
        set.d.dies_log2 = fstx_internal::dies_log2();
        set.stream = static_cast<hipStream_t>(stream);
        set.run = true;
        uint64_t bytes;
        first = next_set(descs, n, first, static_cast<char *>(workspace), &set, &bytes);
        if (set.n == 0) break;
        set.d.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + bytes);
        uint64_t grid = 0;
        for (uint32_t k = 0; k < set.n; ++k) {
            set.t.first[k] = (uint32_t)grid;
            grid += set.t.job[k].n_partials;
        }
        hipLaunchKernelGGL(sum_squares_kernel, dim3((uint32_t)grid), dim3(256), 0, set.stream, set.t);
        int rc = fstx_internal::check_launch("sum_squares_kernel");
        if (rc < 0) return rc;
        hipLaunchKernelGGL(plan_kernel, dim3(set.n), dim3(64), 0, set.stream, set.t, all);
        if ((rc = fstx_internal::check_launch("plan_kernel")) < 0) return rc;
        grid = 0;
        for (uint32_t k = 0; k < set.n; ++k) {
            set.t.first[k] = (uint32_t)grid;
            grid += (uint64_t)(pad_to(set.t.job[k].p, kPadP) / 32) * (pad_to(set.t.job[k].q, kPadQ) / 32) / 4;
        }
        hipLaunchKernelGGL(first_operands_kernel, dim3((uint32_t)grid), dim3(256), 0, set.stream, set.t);
        if ((rc = fstx_internal::check_launch("first_operands_kernel")) < 0) return rc;
        if ((rc = set.steps(steps)) < 0) return rc;
    }
    return 0;
}
