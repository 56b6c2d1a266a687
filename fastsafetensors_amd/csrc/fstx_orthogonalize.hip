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
// 20 %), measured on spectra with a ratio of 1000.  Errors of the LAST step are not amplified any more: where
// the result is rounded to bf16 (2^-9) it runs on one term, which costs 2^-11 or so.
// fp16 rather than bf16 terms because the iterates are bounded: entries of X are at most about
// 1.2, they are held times a power of two near sqrt(p q) so that their typical size stays in the
// middle of fp16's range; A and B are held times fixed powers of two likewise.
//
// Operand layout.  A matrix [R, K] that enters a product as rows x K is stored as blocks of 32
// rows x 16 k in the lane order of v_mfma_f32_32x32x16 (lane: row lane % 32, k = 8 (lane / 32) + 0..7), 1 KiB
// per block and term, terms adjacent, blocks of one row of blocks adjacent.  Tiles then go
// from memory to LDS with global_load_lds as they are, and from LDS to registers as
// conflict-free 16-byte reads.  Products run transposed (the second operand first), so that a
// lane holds four consecutive k of one row of the result seen as an operand: results go back to that
// layout in 8-byte stores.  The transposed copy that the next product needs (X^T; the tile mirrored
// at the diagonal) is made in registers by an MFMA with the identity, which is exact.
// Sides are padded with zeros to whole tiles; products of zeros stay zeros, nothing is masked.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fstx_gather_core.h"
#include "fstx_internal.h"
#include "fstx_update.h"

namespace {

#define FSTX_GLOBAL __attribute__((address_space(1)))
#define FSTX_LDS __attribute__((address_space(3)))
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 half_t;

constexpr uint32_t kBlk = 512;        // elements of one block (32 rows x 16 k) of one term
constexpr uint32_t kPad = 256;        // sides are stored padded to this
constexpr uint32_t kStepPad = 64;     // ... and computed padded to this
constexpr uint32_t kMaxJobs = 20;
constexpr uint32_t kPartials = 256;   // partial sums of squares per matrix
constexpr float kScaleA = 2048.0f;    // A is held times this

struct Job {
    const char *src;
    char *dst;
    half_t *x;        // [p, q]
    half_t *xt[2];    // [q, p], the current one and the next
    half_t *a, *b;    // [p, p]
    double *partials;
    uint64_t x_row, x_col;   // strides of G seen as X, elements
    uint64_t dst_pitch;      // bytes
    uint32_t p, q;
    uint32_t type, flipped;  // flipped: X is G transposed
    float scale;             // X is held times this
    uint32_t n_partials;
    uint64_t pad[2];
};
static_assert(sizeof(Job) == 128, "20 of them fit the kernel arguments");

struct Jobs {
    Job job[kMaxJobs];
    uint32_t first[kMaxJobs];
};

__device__ __forceinline__ uint32_t job_of(const Jobs &t, uint32_t b) {
    uint32_t ji = 0;
#pragma unroll
    for (uint32_t i = 1; i < kMaxJobs; ++i) ji += b >= t.first[i];
    return ji;
}

__host__ __device__ inline uint32_t pad_to(uint32_t n, uint32_t to) { return (n + to - 1) / to * to; }

__device__ __forceinline__ float load_elem(const char *src, uint64_t at, uint32_t type) {
    if (type == FSTX_F32) return *(const FSTX_GLOBAL float *)(src + at * 4);
    const uint16_t raw = *(const FSTX_GLOBAL uint16_t *)(src + at * 2);
    if (type == FSTX_BF16) return __builtin_bit_cast(float, (uint32_t)raw << 16);
    return (float)__builtin_bit_cast(half_t, raw);
}

// ------------------------------------------------------------ |G|_F and the first operands

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Partial sums of squares in 64 bits, each workgroup its own rows in a fixed order: the sum does
// not depend on which workgroup ends first, and squares of the largest floats do not overflow.
__global__ __launch_bounds__(256) void sum_squares_kernel(const Jobs t) {
    __shared__ double part[4];
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job &job = t.job[ji];
    const uint32_t me = blockIdx.x - t.first[ji];
    uint32_t across = 256; // threads along a row
    while (across > 1 && across / 2 >= job.q) across /= 2;
    const uint32_t down = 256 / across;
    double sum = 0;
    for (uint64_t i = (uint64_t)me * down + threadIdx.x / across; i < job.p; i += (uint64_t)job.n_partials * down)
        for (uint32_t j = threadIdx.x % across; j < job.q; j += across) {
            const double v = load_elem(job.src, i * job.x_row + (uint64_t)j * job.x_col, job.type);
            sum += v * v;
        }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) job.partials[me] = part[0] + part[1] + part[2] + part[3];
}

// Four wavefronts, one operand block of X or of X^T each.
__global__ __launch_bounds__(256) void first_operands_kernel(const Jobs t, const float eps) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job &job = t.job[ji];
    double sum = 0;
    for (uint32_t i = threadIdx.x & 63; i < job.n_partials; i += 64) sum += job.partials[i];
    const float norm = (float)sqrt(wave_sum(sum));
    const float factor = job.scale / (norm + eps);

    const uint32_t pp = pad_to(job.p, kPad), qp = pad_to(job.q, kPad);
    const uint32_t per_side = (pp / 32) * (qp / 16); // the same for both orders
    const uint32_t lane = threadIdx.x & 63;
    uint32_t blk = (blockIdx.x - t.first[ji]) * 4 + threadIdx.x / 64;
    const bool second = blk >= per_side;
    if (second) blk -= per_side;
    if (blk >= per_side) return;
    const uint32_t rows = second ? job.q : job.p, ks = second ? job.p : job.q;
    const uint64_t row_stride = second ? job.x_col : job.x_row, k_stride = second ? job.x_row : job.x_col;
    const uint32_t k_blocks = (second ? pp : qp) / 16;
    const uint32_t rb = blk / k_blocks, kb = blk - rb * k_blocks;
    const uint32_t row = rb * 32 + (lane & 31), k0 = kb * 16 + 8 * (lane >> 5);
    v8h h, l;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const float v = row < rows && k0 + e < ks
                            ? load_elem(job.src, (uint64_t)row * row_stride + (uint64_t)(k0 + e) * k_stride, job.type) * factor : 0.0f;
        h[e] = (half_t)v;
        l[e] = (half_t)(v - (float)h[e]);
    }
    half_t *out = (second ? job.xt[0] : job.x) + (uint64_t)blk * 2 * kBlk + lane * 8;
    *(FSTX_GLOBAL v8h *)out = h;
    *(FSTX_GLOBAL v8h *)(out + kBlk) = l;
}

// ------------------------------------------------------------ the products

// C = P Q^T over whole tiles: TR x TC per workgroup of four wavefronts (2 x 2), k in stages of which one is
// computed on while the next two are on their way to LDS.  Measured on a [14336, 4096] update, the product of
// 2 x 4096^2 x 14336 operations in two terms: 128 x 128 tiles 1.45 ms with stages of 32 k and one stage ahead, 1.2 to 1.3 with
// stages of 16 k and two ahead, 256 x 128 tiles 1.15 ms (1.25 PFLOP/s of fp16 products; fewer LDS reads per product).
template <uint32_t TR, uint32_t TC, uint32_t Terms> struct Product {
    static constexpr uint32_t kKb = Terms == 1 || TR == 64 ? 2 : 1;                // k blocks per stage
    static constexpr uint32_t kBufs = 3;                                      // stages in LDS: one computed on, two on their way
    static constexpr uint32_t kHalfP = TR / 32 * kKb * Terms;                 // blocks of either operand per stage
    static constexpr uint32_t kHalfQ = TC / 32 * kKb * Terms;
    static constexpr uint32_t kStage = (kHalfP + kHalfQ) * kBlk;              // elements per stage
    static constexpr uint32_t kLoads = (kHalfP + kHalfQ) / 4;                 // per wavefront and stage
    static constexpr uint32_t kNR = TR / 64, kNC = TC / 64;                   // 32-blocks per wavefront
    static_assert(kHalfP % 4 == 0 && kHalfQ % 4 == 0, "a load instruction of four wavefronts stays within one operand");

    // `Swap`: lanes hold rows of P (four consecutive rows of Q each); else rows of Q
    template <bool Swap>
    static __device__ __forceinline__ void run(const half_t *p, const half_t *q, uint32_t k_blocks_stored, uint32_t k_blocks,
                                               half_t *lds, v16f (&acc)[kNR][kNC]) {
        const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wr = wave >> 1, wc = wave & 1;
        const uint64_t row_step = (uint64_t)k_blocks_stored * 2 * kBlk;
        auto load_stage = [&](uint32_t kb0, uint32_t buf) {
#pragma unroll
            for (uint32_t n = 0; n < kLoads; ++n) {
                const uint32_t at = n * 4 + wave;
                const bool second = n * 4 >= kHalfP;
                const uint32_t in = second ? at - kHalfP : at;
                const uint32_t rb = in / (kKb * Terms), rest = in % (kKb * Terms);
                const half_t *from = (second ? q : p) + rb * row_step + (uint64_t)(kb0 + rest / Terms) * 2 * kBlk + (rest % Terms) * kBlk + lane * 8;
                __builtin_amdgcn_global_load_lds((const FSTX_GLOBAL void *)from, (FSTX_LDS void *)(lds + buf * kStage + at * kBlk), 16, 0, 0);
            }
        };
        v8h pf[kKb][kNR][Terms], qf[kKb][kNC][Terms];
        auto fetch = [&](uint32_t buf) {
            const half_t *base = lds + buf * kStage + lane * 8;
#pragma unroll
            for (uint32_t kb = 0; kb < kKb; ++kb)
#pragma unroll
                for (uint32_t m = 0; m < Terms; ++m) {
#pragma unroll
                    for (uint32_t i = 0; i < kNR; ++i) pf[kb][i][m] = *(const v8h *)(base + (((wr * kNR + i) * kKb + kb) * Terms + m) * kBlk);
#pragma unroll
                    for (uint32_t j = 0; j < kNC; ++j) qf[kb][j][m] = *(const v8h *)(base + (kHalfP + ((wc * kNC + j) * kKb + kb) * Terms + m) * kBlk);
                }
        };
        auto multiply = [&]() {
#pragma unroll
            for (uint32_t kb = 0; kb < kKb; ++kb)
#pragma unroll
                for (int sum = 0; sum < (int)Terms; ++sum)
#pragma unroll
                    for (int m = 0; m <= sum; ++m)
#pragma unroll
                        for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
                            for (uint32_t j = 0; j < kNC; ++j)
                                acc[i][j] = Swap ? __builtin_amdgcn_mfma_f32_32x32x16_f16(qf[kb][j][m], pf[kb][i][sum - m], acc[i][j], 0, 0, 0)
                                                 : __builtin_amdgcn_mfma_f32_32x32x16_f16(pf[kb][i][m], qf[kb][j][sum - m], acc[i][j], 0, 0, 0);
        };
        constexpr uint32_t kAhead = kBufs - 1;
        const uint32_t stages = k_blocks / kKb;
        for (uint32_t s = 0; s < kAhead && s < stages; ++s) load_stage(s * kKb, s);
        uint32_t s = 0, buf = 0;
        for (; s + kAhead < stages; ++s) {
            // This wavefront's loads of the stage have landed (those of the next one may be on their way) and its
            // reads of the stage before are done; behind the barrier that holds for all four.
            constexpr uint32_t kLeft = (kAhead - 1) * kLoads;
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
            fetch(buf);
            load_stage((s + kAhead) * kKb, buf == 0 ? kBufs - 1 : buf - 1); // where the stage before was
            multiply();
            buf = buf + 1 == kBufs ? 0 : buf + 1;
        }
        for (; s < stages; ++s) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            fetch(buf);
            multiply();
            buf = buf + 1 == kBufs ? 0 : buf + 1;
        }
    }
};

// Where a lane's four values 4g..4g+3 of a 32 x 32 block lie in an operand: row block `rb`, columns 32 cb + 8g + 4 (lane / 32)..+3
__device__ __forceinline__ uint64_t quad_at(uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t g, uint32_t lane) {
    return ((uint64_t)rb * k_blocks_stored + 2 * cb + (g >> 1)) * 2 * kBlk + ((g & 1) * 32 + (lane & 31)) * 8 + 4 * (lane >> 5);
}

__device__ __forceinline__ v16f load_block(const half_t *m, uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t lane, bool both) {
    v16f out;
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g) {
        const half_t *at = m + quad_at(rb, cb, k_blocks_stored, g, lane);
        const v4h h = *(const FSTX_GLOBAL v4h *)at;
        v4h l = {};
        if (both) l = *(const FSTX_GLOBAL v4h *)(at + kBlk);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) out[4 * g + e] = (float)h[e] + (float)l[e];
    }
    return out;
}

__device__ __forceinline__ void store_block(half_t *m, uint32_t rb, uint32_t cb, uint32_t k_blocks_stored, uint32_t lane, const half_t (&h)[16],
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
        *(FSTX_GLOBAL v4h *)(at + kBlk) = vl;
    }
}

__device__ __forceinline__ void split(const v16f &v, half_t (&h)[16], half_t (&l)[16]) {
#pragma unroll
    for (uint32_t r = 0; r < 16; ++r) {
        h[r] = (half_t)v[r];
        l[r] = (half_t)(v[r] - (float)h[r]);
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

enum Phase : uint32_t { kGram, kPoly, kApply, kLast };

struct Coefficients {
    float own, product; // result = own * (what is there) + product * (sum of the products)
    uint32_t current;   // which of xt[] is the current one
    uint32_t both;      // whether "what is there" is taken with both terms
};

// Tiles of a symmetric matrix that reach on or below the diagonal, row by row: row i has kAspect (i + 1) of
// them, a tile being kAspect times as high as wide.
template <uint32_t kAspect> __host__ __device__ inline uint32_t triangle_tiles(uint32_t rows) { return kAspect * (rows * (rows + 1) / 2); }
template <uint32_t kAspect> __device__ __forceinline__ void triangle(uint32_t t, uint32_t &i, uint32_t &j) {
    i = (uint32_t)((sqrtf(8.0f * (float)(t / kAspect) + 1.0f) - 1.0f) * 0.5f);
    while (triangle_tiles<kAspect>(i) > t) --i;
    while (triangle_tiles<kAspect>(i + 1) <= t) ++i;
    j = t - triangle_tiles<kAspect>(i);
}

template <uint32_t kPhase, uint32_t TR, uint32_t TC, uint32_t Terms>
__global__ __launch_bounds__(256, 2) void newton_schulz_kernel(const uint32_t dies_log2, const Jobs t, const Coefficients c) {
    typedef Product<TR, TC, Terms> Prod;
    constexpr uint32_t kNR = Prod::kNR, kNC = Prod::kNC;
    __shared__ __attribute__((aligned(1024))) half_t lds[Prod::kBufs * Prod::kStage];
    const uint32_t ji = job_of(t, blockIdx.x);
    const Job &job = t.job[ji];
    const uint32_t pt = (job.p + TR - 1) / TR, qt = (job.q + TC - 1) / TC;
    const uint32_t p_blocks = pad_to(job.p, kPad) / 16, q_blocks = pad_to(job.q, kPad) / 16; // as stored
    constexpr bool kSymmetric = kPhase == kGram || kPhase == kPoly;
    uint32_t tile, ti, tj;
    if (!fstx_gather::tile_for_die(blockIdx.x - t.first[ji], kSymmetric ? triangle_tiles<TR / TC>(pt) : pt * qt, dies_log2, tile)) return;
    if (kSymmetric) {
        triangle<TR / TC>(tile, ti, tj);
    } else { // columns of up to eight tiles, so that the tiles at work share both operands
        const uint32_t group = tile / (8 * qt), first = group * 8, height = pt - first < 8 ? pt - first : 8;
        const uint32_t in = tile - group * 8 * qt;
        ti = first + in % height;
        tj = in / height;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t rb0 = ti * (TR / 32) + (wave >> 1) * kNR, cb0 = tj * (TC / 32) + (wave & 1) * kNC;

    v16f acc[kNR][kNC] = {};
    if constexpr (kPhase == kGram) {
        const uint64_t row = (uint64_t)q_blocks * 2 * kBlk;
        Prod::template run<true>(job.x + ti * (TR / 32) * row, job.x + tj * (TC / 32) * row, q_blocks, pad_to(job.q, kStepPad) / 16, lds, acc);
    } else if constexpr (kPhase == kPoly) {
        const uint64_t row = (uint64_t)p_blocks * 2 * kBlk;
        Prod::template run<true>(job.a + ti * (TR / 32) * row, job.a + tj * (TC / 32) * row, p_blocks, pad_to(job.p, kStepPad) / 16, lds, acc);
    } else {
        const uint64_t row = (uint64_t)p_blocks * 2 * kBlk;
        const half_t *p = job.b + ti * (TR / 32) * row, *q = job.xt[c.current] + tj * (TC / 32) * row;
        if (kPhase == kLast && !job.flipped) Prod::template run<false>(p, q, p_blocks, pad_to(job.p, kStepPad) / 16, lds, acc);
        else Prod::template run<true>(p, q, p_blocks, pad_to(job.p, kStepPad) / 16, lds, acc);
    }

#pragma unroll
    for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
        for (uint32_t j = 0; j < kNC; ++j) {
            const uint32_t rb = rb0 + i, cb = cb0 + j;
            if (kSymmetric && cb > rb) continue; // written as the mirror of (cb, rb)
            v16f v = acc[i][j];
            if constexpr (kPhase == kLast) {
                // lanes run along the contiguous side of the destination: 64 or 128 contiguous bytes per row
                const v16f x = job.flipped ? load_block(job.x, rb, cb, q_blocks, lane, c.both) : load_block(job.xt[c.current], cb, rb, p_blocks, lane, c.both);
                const uint32_t along = (job.flipped ? rb : cb) * 32 + (lane & 31);
                const uint32_t rows = job.flipped ? job.q : job.p, cols = job.flipped ? job.p : job.q;
                const float back = 1.0f / job.scale;
                if (along < cols)
#pragma unroll
                    for (uint32_t r = 0; r < 16; ++r) {
                        const uint32_t row = (job.flipped ? cb : rb) * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
                        if (row >= rows) continue;
                        const float out = (c.own * x[r] + c.product * v[r]) * back;
                        char *at = job.dst + (uint64_t)row * job.dst_pitch;
                        if (job.type == FSTX_F32) ((FSTX_GLOBAL float *)at)[along] = out;
                        else if (job.type == FSTX_BF16) ((FSTX_GLOBAL __bf16 *)at)[along] = (__bf16)out;
                        else ((FSTX_GLOBAL half_t *)at)[along] = (half_t)out;
                    }
                continue;
            }
            if constexpr (kPhase == kGram) {
                v *= c.product / (job.scale * job.scale);
            } else {
                const v16f own = kPhase == kPoly ? load_block(job.a, rb, cb, p_blocks, lane, c.both) : load_block(job.x, rb, cb, q_blocks, lane, c.both);
#pragma unroll
                for (uint32_t r = 0; r < 16; ++r) v[r] = c.own * own[r] + c.product * v[r];
            }
            half_t h[16], l[16], ht[16], lt[16];
            split(v, h, l);
            half_t *to = kPhase == kGram ? job.a : kPhase == kPoly ? job.b : job.x;
            store_block(to, rb, cb, kPhase == kApply ? q_blocks : p_blocks, lane, h, l);
            if (kPhase == kApply || cb != rb) {
                exchange(h, ht, lane);
                exchange(l, lt, lane);
                store_block(kPhase == kApply ? job.xt[c.current ^ 1] : to, cb, rb, p_blocks, lane, ht, lt);
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

struct Sides {
    uint64_t p, q, pp, qp;
    explicit Sides(const fstx_orthogonalize_desc &d)
        : p(d.rows < d.cols ? d.rows : d.cols), q(d.rows < d.cols ? d.cols : d.rows), pp((p + kPad - 1) / kPad * kPad), qp((q + kPad - 1) / kPad * kPad) {}
    uint64_t bytes() const { return (3 * pp * qp + 2 * pp * pp) * 2 * sizeof(half_t) + kPartials * sizeof(double); }
};

// span of bytes a strided matrix lies in
struct Span {
    uint64_t at, end;
    Span(const void *p, uint64_t rows, uint64_t rs, uint64_t cols, uint64_t cs, uint64_t size)
        : at((uint64_t)(uintptr_t)p), end(at + ((rows - 1) * rs + (cols - 1) * cs + 1) * size) {}
    bool meets(const Span &o) const { return at < o.end && o.at < end; }
};
Span dst_of(const fstx_orthogonalize_desc &d) { return Span(d.dst, d.rows, d.dst_pitch, d.cols, 1, size_of(d.type)); }
Span src_of(const fstx_orthogonalize_desc &d) { return Span(d.src, d.rows, d.src_row_stride, d.cols, d.src_col_stride, size_of(d.type)); }

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
    }
    for (uint32_t i = 0; i < n; ++i)
        for (uint32_t j = 0; j < n; ++j)
            if (i != j && !empty(descs[i]) && !empty(descs[j]) &&
                (dst_of(descs[i]).meets(dst_of(descs[j])) || dst_of(descs[i]).meets(src_of(descs[j]))))
                return -FSTX_E_INVAL;
    return 0;
}

// bf16 matrices take one term in the last step, the others two: each kind has launches of its own, so
// that a matrix's result does not depend on what else is in the call.
inline bool skip(const fstx_orthogonalize_desc &d, bool bf16) { return empty(d) || (d.type == FSTX_BF16) != bf16; }

// the descriptors [first, end) of one kind in one set of launches, and the workspace they take
uint32_t next_chunk(const fstx_orthogonalize_desc *descs, uint32_t n, bool bf16, uint32_t first, uint64_t *bytes) {
    uint32_t k = 0;
    *bytes = 0;
    for (uint32_t i = first; i < n; ++i) {
        if (skip(descs[i], bf16)) continue;
        const uint64_t need = Sides(descs[i]).bytes();
        if (k == kMaxJobs || (k && *bytes + need > kChunkBytes)) return i;
        *bytes += need;
        ++k;
    }
    return n;
}

inline float power_of_two_below(double v) { return (float)ldexp(1.0, (int)floor(log2(v))); }

// Workgroups a launch needs before larger tiles are taken: below that most of the 256 compute units would idle.
constexpr uint64_t kLargeTiles = 200;

struct Launcher {
    Jobs t;
    uint32_t n = 0;
    hipStream_t stream;

    template <uint32_t kPhase, uint32_t TR, uint32_t TC> uint64_t tiles() const {
        uint64_t sum = 0;
        for (uint32_t i = 0; i < n; ++i) sum += tiles_of<kPhase, TR, TC>(t.job[i]);
        return sum;
    }
    template <uint32_t kPhase, uint32_t TR, uint32_t TC> static uint64_t tiles_of(const Job &j) {
        const uint32_t pt = (j.p + TR - 1) / TR, qt = (j.q + TC - 1) / TC;
        return kPhase == kGram || kPhase == kPoly ? triangle_tiles<TR / TC>(pt) : (uint64_t)pt * qt;
    }

    template <uint32_t kPhase, uint32_t TR, uint32_t TC, uint32_t Terms> int launch(const Coefficients &c) {
        const uint32_t dl = fstx_internal::dies_log2();
        uint64_t grid = 0;
        for (uint32_t i = 0; i < n; ++i) {
            t.first[i] = (uint32_t)grid;
            grid += (tiles_of<kPhase, TR, TC>(t.job[i]) + (1u << dl) - 1) >> dl << dl;
        }
        if (grid * 256 > 0xffffffffull) return -FSTX_E_RANGE;
        fstx_internal::Range range("fstx newton_schulz_kernel: phase %u, %u matrices, %llu tiles of %u x %u", kPhase, n, (unsigned long long)grid, TR, TC);
        hipLaunchKernelGGL((newton_schulz_kernel<kPhase, TR, TC, Terms>), dim3((uint32_t)grid), dim3(256), 0, stream, dl, t, c);
        return fstx_internal::check_launch("newton_schulz_kernel");
    }

    template <uint32_t kPhase, uint32_t Terms> int phase(const Coefficients &c) {
        if constexpr (kPhase == kApply || kPhase == kLast)
            if (tiles<kPhase, 256, 128>() >= kLargeTiles) return launch<kPhase, 256, 128, Terms>(c);
        return tiles<kPhase, 128, 128>() >= kLargeTiles ? launch<kPhase, 128, 128, Terms>(c) : launch<kPhase, 64, 64, Terms>(c);
    }
    template <uint32_t kPhase> int phase(uint32_t terms, const Coefficients &c) {
        if constexpr (kPhase == kApply) return phase<kPhase, 2>(c); // never the last step
        else return terms == 1 ? phase<kPhase, 1>(c) : phase<kPhase, 2>(c);
    }
};

} // namespace

extern "C" int64_t fstx_orthogonalize_workspace(const fstx_orthogonalize_desc *descs, uint32_t n) {
    const int rc = check(descs, n);
    if (rc < 0) return rc;
    uint64_t most = 0;
    for (int bf16 = 0; bf16 < 2; ++bf16)
        for (uint32_t i = 0; i < n;) {
            uint64_t bytes;
            i = next_chunk(descs, n, bf16, i, &bytes);
            if (bytes > most) most = bytes;
        }
    return (int64_t)most;
}

extern "C" int fstx_orthogonalize(const fstx_orthogonalize_desc *descs, uint32_t n, const float *coefficients, uint32_t steps, float eps,
                                  void *workspace, uint64_t workspace_bytes, void *stream) {
    const int64_t need = fstx_orthogonalize_workspace(descs, n);
    if (need < 0) return (int)need;
    if (steps < 1 || steps > kMaxSteps || !coefficients || !(eps >= 0)) return -FSTX_E_INVAL;
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (uint64_t)need)) return -FSTX_E_INVAL;
    for (int bf16 = 0; bf16 < 2; ++bf16)
        for (uint32_t i = 0; i < n;) {
            uint64_t bytes;
            const uint32_t end = next_chunk(descs, n, bf16, i, &bytes);
            Launcher run;
            run.stream = static_cast<hipStream_t>(stream);
            for (uint32_t k = 0; k < kMaxJobs; ++k) run.t.first[k] = 0xffffffffu;
            char *at = static_cast<char *>(workspace);
            for (; i < end; ++i) {
                const fstx_orthogonalize_desc &d = descs[i];
                if (skip(d, bf16)) continue;
                const Sides s(d);
                const bool flipped = d.rows > d.cols;
                Job &j = run.t.job[run.n++];
                j = Job{};
                j.src = static_cast<const char *>(d.src);
                j.dst = static_cast<char *>(d.dst);
                const uint64_t xb = s.pp * s.qp * 2 * sizeof(half_t), ab = s.pp * s.pp * 2 * sizeof(half_t);
                j.x = reinterpret_cast<half_t *>(at);
                j.xt[0] = reinterpret_cast<half_t *>(at + xb);
                j.xt[1] = reinterpret_cast<half_t *>(at + 2 * xb);
                j.a = reinterpret_cast<half_t *>(at + 3 * xb);
                j.b = reinterpret_cast<half_t *>(at + 3 * xb + ab);
                j.partials = reinterpret_cast<double *>(at + 3 * xb + 2 * ab);
                at += s.bytes();
                j.x_row = flipped ? d.src_col_stride : d.src_row_stride;
                j.x_col = flipped ? d.src_row_stride : d.src_col_stride;
                j.dst_pitch = d.dst_pitch * size_of(d.type);
                j.p = (uint32_t)s.p;
                j.q = (uint32_t)s.q;
                j.type = d.type;
                j.flipped = flipped;
                // entries of X are at most about 1.2 (the spectral norm), their mean square is 1 / (p q) at first
                const double mid = sqrt((double)s.p * (double)s.q);
                j.scale = power_of_two_below(mid < 8192.0 ? mid : 8192.0);
                const uint64_t parts = (s.p * s.q + 16383) / 16384;
                j.n_partials = (uint32_t)(parts < kPartials ? parts : kPartials);
            }
            if (run.n == 0) continue;
            uint64_t grid = 0;
            for (uint32_t k = 0; k < run.n; ++k) {
                run.t.first[k] = (uint32_t)grid;
                grid += run.t.job[k].n_partials;
            }
            hipLaunchKernelGGL(sum_squares_kernel, dim3((uint32_t)grid), dim3(256), 0, run.stream, run.t);
            int rc = fstx_internal::check_launch("sum_squares_kernel");
            if (rc < 0) return rc;
            grid = 0;
            for (uint32_t k = 0; k < run.n; ++k) {
                const uint64_t pp = pad_to(run.t.job[k].p, kPad), qp = pad_to(run.t.job[k].q, kPad);
                run.t.first[k] = (uint32_t)grid;
                grid += (pp / 32) * (qp / 16) * 2 / 4;
            }
            if (grid * 256 > 0xffffffffull) return -FSTX_E_RANGE;
            hipLaunchKernelGGL(first_operands_kernel, dim3((uint32_t)grid), dim3(256), 0, run.stream, run.t, eps);
            if ((rc = fstx_internal::check_launch("first_operands_kernel")) < 0) return rc;
            for (uint32_t step = 0; step < steps; ++step) {
                const float a = coefficients[3 * step], b = coefficients[3 * step + 1], c = coefficients[3 * step + 2];
                // B is held times this: its entries stay below fp16's largest while singular values are below sqrt(2)
                const float scale_b = power_of_two_below(30000.0 / (2.0 * fabs((double)b) + 4.0 * fabs((double)c) + 0.01));
                const bool last = step + 1 == steps;
                const uint32_t terms = last && bf16 ? 1 : 2, current = step & 1, both = terms == 2;
                if ((rc = run.phase<kGram>(terms, Coefficients{0, kScaleA, current, 1})) < 0) return rc;
                if ((rc = run.phase<kPoly>(terms, Coefficients{b * scale_b / kScaleA, c * scale_b / (kScaleA * kScaleA), current, both})) < 0) return rc;
                const Coefficients apply{a, 1.0f / scale_b, current, both};
                if ((rc = last ? run.phase<kLast>(terms, apply) : run.phase<kApply>(terms, apply)) < 0) return rc;
            }
        }
    return 0;
}
