// SPDX-License-Identifier: Apache-2.0
//
// Low-rank updates merged into weights:  W'[i,j] = round(W[i,j] + s * sum_k U[i,k] D[k,j]).
//
// With r = rank a few dozen the product costs 2r operations per element of W and the weight
// has to be read and written once, so HBM is the bound up to ranks of several hundreds and the
// kernel is built as a streaming pass over W with the product made on the side:
//
//   pack_factors_kernel  lays U and D out as MFMA operands (below).  They are r (M + N) elements
//                        against M N of the weight, and are re-read by every tile they feed, so that
//                        strides, element types, odd sizes and zero padding are dealt with once
//                        and the main kernel has none of them.
//   deep_low_rank_kernel for longer products, direct_low_rank_kernel for few tiles: see there.
//   low_rank_kernel      a wavefront walks along a panel of rows in tiles of one 128-byte line per row (64 rows;
//                        32 of fp8): the next tile's weights are on their way while it makes the product
//                        of this one from operands that L2 holds, adds, rounds and stores.
//                        No LDS and no barriers: nothing is shared but the factors.
//
// What bounds it, measured.  The seven matrices of a Llama-3-8B layer, bf16, rank 64 (883 MB read and written):
// 169 us + 14 us of packing, 5.2 TB/s; a plain copy of that size does 6.2.  A Llama-3-70B fp8 layer, rank 16
// (1.7 GB): 360 us, 4.8 TB/s.  Steps there (same layer): one 64 x 64 tile per wavefront with 64 contiguous bytes per row and
// instruction 241 us, 26 % more written to HBM than the weight holds, because half lines left L2 before their other
// halves came; whole lines per instruction 193 us; walks of four tiles 184 (of eight 189, of two 180 but 364 instead of
// 359 for the fp8 layer).  Streaming (non-temporal) accesses are worth 5 to 8 % where rows lie on whole lines and cost 25 %
// where tiles share them: see on_lines.
//
// Numerics.  MFMA products of bf16 / fp16 are exact in fp32 and are summed in fp32.  Factors of
// f32 are split into bf16 terms x = h + m (+ l), each the rounding of what is left: bf16 because it
// has f32's range.  Two terms (16 bits of each factor; h h + h m + m h, what is left out is at most
// 3 * 2^-16 of a product: the last bits of either factor, and m m) for weights of 8 or 16 bits, whose own rounding is 2^-11
// of the result or more: it hides what is left out unless the products cancel to less than 3 * 2^-5 of their sizes' sum on a weight
// near zero.  Three products instead of six; those of the [5120, 3456] cut with factors of rank 256 are what bounds that merge.
// Three terms (24 bits; six products, what is left out is at most 4 * 2^-24) for f32 weights.  One term where the
// factors are already bf16, or both fp16.
//
// Operand layout.  v_mfma_f32_16x16x32 takes 8 consecutive k of row lane % 16 from each lane
// (k = 8 (lane / 16) + 0..7): a block of 16 rows x 32 k is stored as the 64 lanes' 16 bytes in
// lane order, 1 KiB, so that an operand load is one fully coalesced global_load_dwordx4.  The
// product is computed transposed (D as the first operand): a lane then holds, for ONE row of W, the
// 4 columns that its quarter of the wavefront owns in each 16-column block; and the columns are
// dealt to the blocks so that the blocks of one 16-byte vector of W are consecutive (column_of).
// Two lanes of neighbouring rows trade their halves of the two lines (trade), and W moves
// between memory and the accumulator layout 16 bytes per lane and a whole line per row and instruction.

#include <errno.h>
#include <hip/hip_runtime.h>
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
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

constexpr uint32_t kTile = 256;  // rows and columns the packed factors are padded to: whole tiles of every type and kernel
constexpr uint32_t kBlk = 512;   // elements of one operand block (16 rows x 32 k)
constexpr uint32_t kK = 32;      // k per block
constexpr uint32_t kMaxJobs = 24;

// How the factors travel: the type and number of their terms.
enum : uint32_t { kTermsH1 = 0, kTermsB1 = 1, kTermsB2 = 2, kTermsB3 = 3, kTermClasses = 4 };
__host__ __device__ constexpr uint32_t terms_of(uint32_t cls) { return cls < 2 ? 1 : cls; }

struct alignas(32) MergeJob {
    char *dst;
    const char *src;
    const uint16_t *up, *down; // packed
    const float *weight_scale;
    uint64_t dst_pitch, src_pitch; // bytes
    uint32_t rows, cols, k_blocks, col_tiles;
    float scale;
    uint32_t scale_step;           // 0: one weight scale, 1: one per row
    uint32_t walk, walks, n_walks; // tiles per wavefront, wavefronts per panel of rows and in all
    uint32_t lines;                // see on_lines
    uint32_t pad[2];
};
static_assert(sizeof(MergeJob) == 128, "24 of them fit the kernel arguments");

struct PackJob {
    const char *src;
    uint16_t *dst;
    uint64_t row_stride, k_stride; // elements
    uint32_t rows, rank, k_blocks, tiles;
    uint32_t type, terms, half, per; // per: elements of W per 16 bytes (column operand), 0 for the row operand
};

template <typename Job> struct Jobs {
    Job job[kMaxJobs];
    uint32_t first[kMaxJobs]; // first workgroup of each job; unused entries ~0
};

template <typename Job> __device__ __forceinline__ uint32_t job_of(const Jobs<Job> &t, uint32_t b) {
    uint32_t ji = 0;
#pragma unroll
    for (uint32_t i = 1; i < kMaxJobs; ++i) ji += b >= t.first[i];
    return ji;
}

// Column of W that row `rho` of operand block `blk` stands for (within the whole operand): the
// 16-byte vectors of W hold `per` elements, four lane groups make 4 per columns, per / 4 blocks.
__device__ __forceinline__ uint32_t column_of(uint32_t blk, uint32_t rho, uint32_t per) {
    const uint32_t n_blk = per / 4, v = blk / n_blk, tt = blk % n_blk;
    return 4 * per * v + per * (rho >> 2) + 4 * tt + (rho & 3);
}

// Eight elements of a factor, those at(e) that are there(e), zeros else.  All eight loads go out together: the type is
// looked at once, and what is not there is read from the factor's first element and dropped, where a branch around each load
// would wait for one after the other (the merge of a Llama-3-8B layer 182.7 us instead of 185.1).
template <typename At, typename There>
__device__ __forceinline__ void load_factor(const char *src, uint32_t type, float (&x)[8], At at, There there) {
    if (type == FSTX_F32) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) x[e] = *(const FSTX_GLOBAL float *)(src + (there(e) ? at(e) : 0) * 4);
    } else {
        uint16_t raw[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) raw[e] = *(const FSTX_GLOBAL uint16_t *)(src + (there(e) ? at(e) : 0) * 2);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            x[e] = type == FSTX_BF16 ? __builtin_bit_cast(float, (uint32_t)raw[e] << 16) : (float)__builtin_bit_cast(_Float16, raw[e]);
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) x[e] = there(e) ? x[e] : 0.0f;
}

// the bf16 nearest to x; where that would overflow a finite x, the one below it
__device__ __forceinline__ float bf16_term(float x) {
    const float h = (float)(__bf16)x;
    if (__builtin_isinf(h) && !__builtin_isinf(x)) return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
    return h;
}

__device__ __forceinline__ v8h half_terms(const float (&x)[8]) {
    v8h h;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) h[e] = (_Float16)x[e];
    return h;
}
// the next bf16 term of eight values, which become what is left of them
__device__ __forceinline__ v8b next_term(float (&x)[8]) {
    v8b h;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const float f = bf16_term(x[e]);
        h[e] = (__bf16)f;
        x[e] = __builtin_isfinite(f) ? x[e] - f : 0.0f; // nothing behind an infinity or a NaN
    }
    return h;
}

// One wavefront per operand block, four per workgroup (a side has a multiple of eight blocks).
__global__ __launch_bounds__(256) void pack_factors_kernel(const Jobs<PackJob> t) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const PackJob &job = t.job[ji];
    const uint32_t lb = (blockIdx.x - t.first[ji]) * 4 + (threadIdx.x >> 6);
    const uint32_t blk = lb / job.k_blocks, kb = lb - blk * job.k_blocks;
    const uint32_t lane = threadIdx.x & 63, rho = lane & 15;
    const uint32_t row = job.per ? column_of(blk, rho, job.per) : blk * 16 + rho;
    const uint32_t k0 = kb * kK + 8 * (lane >> 4);
    float x[8];
    load_factor(job.src, job.type, x, [&](uint32_t e) { return (uint64_t)row * job.row_stride + (uint64_t)(k0 + e) * job.k_stride; },
                [&](uint32_t e) { return row < job.rows && k0 + e < job.rank; });
    uint16_t *out = job.dst + ((uint64_t)lb * job.terms) * kBlk + lane * 8;
    if (job.half) {
        *(FSTX_GLOBAL v8h *)out = half_terms(x);
        return;
    }
    for (uint32_t term = 0; term < job.terms; ++term) *(FSTX_GLOBAL v8b *)(out + term * kBlk) = next_term(x);
}

template <uint32_t Cls> struct Operand { typedef v8b type; };
template <> struct Operand<kTermsH1> { typedef v8h type; };

__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Element types of W.  Vectors are as aligned as one element: global accesses of any width take
// element-aligned addresses on this hardware.
template <uint32_t T> struct Weight;
template <> struct Weight<FSTX_F32> { static constexpr uint32_t size = 4; typedef v4u loose __attribute__((aligned(4))); };
template <> struct Weight<FSTX_BF16> { static constexpr uint32_t size = 2; typedef v4u loose __attribute__((aligned(2))); };
template <> struct Weight<FSTX_F16> { static constexpr uint32_t size = 2; typedef v4u loose __attribute__((aligned(2))); };
template <> struct Weight<FSTX_F8_E4M3> { static constexpr uint32_t size = 1; typedef v4u loose __attribute__((aligned(1))); };

// clamp to e4m3's largest finite values; a NaN stays one
__device__ __forceinline__ float saturate_e4m3(float v) { return v != v ? v : __builtin_amdgcn_fmed3f(v, -448.0f, 448.0f); }

// the vector of W's elements + s * acc, acc[e] being the sum for element e
template <uint32_t T>
__device__ __forceinline__ v4u merged(v4u w, const float *acc, float s) {
    v4u out;
    if constexpr (T == FSTX_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t bits = w[e]; // (a bit cast of a vector's element itself takes element 0)
            out[e] = __builtin_bit_cast(uint32_t, __builtin_fmaf(s, acc[e], __builtin_bit_cast(float, bits)));
        }
    } else if constexpr (T == FSTX_BF16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lo = __builtin_bit_cast(float, w[e] << 16), hi = __builtin_bit_cast(float, w[e] & 0xffff0000u);
            typedef __bf16 v2b __attribute__((ext_vector_type(2)));
            const v2b r = {(__bf16)__builtin_fmaf(s, acc[2 * e], lo), (__bf16)__builtin_fmaf(s, acc[2 * e + 1], hi)};
            out[e] = __builtin_bit_cast(uint32_t, r);
        }
    } else if constexpr (T == FSTX_F16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            typedef _Float16 v2h __attribute__((ext_vector_type(2)));
            const uint32_t bits = w[e];
            const v2h in = __builtin_bit_cast(v2h, bits);
            const v2h r = {(_Float16)__builtin_fmaf(s, acc[2 * e], (float)in[0]), (_Float16)__builtin_fmaf(s, acc[2 * e + 1], (float)in[1])};
            out[e] = __builtin_bit_cast(uint32_t, r);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = saturate_e4m3(__builtin_fmaf(s, acc[4 * e], __builtin_amdgcn_cvt_f32_fp8((int)w[e], 0)));
            const float b = saturate_e4m3(__builtin_fmaf(s, acc[4 * e + 1], __builtin_amdgcn_cvt_f32_fp8((int)w[e], 1)));
            const float c = saturate_e4m3(__builtin_fmaf(s, acc[4 * e + 2], __builtin_amdgcn_cvt_f32_fp8((int)w[e], 2)));
            const float d = saturate_e4m3(__builtin_fmaf(s, acc[4 * e + 3], __builtin_amdgcn_cvt_f32_fp8((int)w[e], 3)));
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
            out[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
        }
    }
    return out;
}

// Lanes 2n and 2n + 1 (two rows of a tile): what the even one holds in b against what the odd one holds in a.
// Each row's two halves of a line, held by one lane each way, become two whole lines held by both: its own inverse.
__device__ __forceinline__ void trade(v4u &a, v4u &b, bool odd) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t give = odd ? a[k] : b[k];
        const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0xb1 /* quad_perm:[1,0,3,2] */, 0xf, 0xf, true);
        const uint32_t x = odd ? got : a[k], y = odd ? b[k] : got;
        a[k] = x;
        b[k] = y;
    }
}

// Shape of a wavefront's tile: kRows rows of one 128-byte line.
template <uint32_t T> struct Tile {
    static constexpr uint32_t kSize = Weight<T>::size, kPer = 16 / kSize;
    static constexpr uint32_t kCols = 128 / kSize;                // 32, 64 or 128
    static constexpr uint32_t kRows = kSize == 1 ? 32 : 64;
    static constexpr uint32_t kNR = kRows / 16, kNC = kCols / 16; // operand blocks
};

// The 1..15 bytes that end a row, in pieces of 8, 4, 2 and 1: all loads of a wavefront at once, where a loop over
// elements would wait for each.
__device__ __forceinline__ v4u load_tail(const char *at, uint32_t bytes) {
    typedef uint64_t by1_8 __attribute__((aligned(1)));
    typedef uint32_t by1_4 __attribute__((aligned(1)));
    typedef uint16_t by1_2 __attribute__((aligned(1)));
    unsigned __int128 v = 0;
    if (bytes & 8) v = *(const FSTX_GLOBAL by1_8 *)at;
    if (bytes & 4) v |= (unsigned __int128) * (const FSTX_GLOBAL by1_4 *)(at + (bytes & 8)) << 8 * (bytes & 8);
    if (bytes & 2) v |= (unsigned __int128) * (const FSTX_GLOBAL by1_2 *)(at + (bytes & 12)) << 8 * (bytes & 12);
    if (bytes & 1) v |= (unsigned __int128) * (const FSTX_GLOBAL uint8_t *)(at + (bytes & 14)) << 8 * (bytes & 14);
    return __builtin_bit_cast(v4u, v);
}
__device__ __forceinline__ void store_tail(char *at, uint32_t bytes, v4u value) {
    typedef uint64_t by1_8 __attribute__((aligned(1)));
    typedef uint32_t by1_4 __attribute__((aligned(1)));
    typedef uint16_t by1_2 __attribute__((aligned(1)));
    const unsigned __int128 v = __builtin_bit_cast(unsigned __int128, value);
    if (bytes & 8) *(FSTX_GLOBAL by1_8 *)at = (uint64_t)v;
    if (bytes & 4) *(FSTX_GLOBAL by1_4 *)(at + (bytes & 8)) = (uint32_t)(v >> 8 * (bytes & 8));
    if (bytes & 2) *(FSTX_GLOBAL by1_2 *)(at + (bytes & 12)) = (uint16_t)(v >> 8 * (bytes & 12));
    if (bytes & 1) *(FSTX_GLOBAL uint8_t *)(at + (bytes & 14)) = (uint8_t)(v >> 8 * (bytes & 14));
}

template <uint32_t T, uint32_t Cls, uint32_t NR = Tile<T>::kNR> struct Merge {
    typedef Tile<T> S;
    typedef typename Operand<Cls>::type op_t;
    typedef typename Weight<T>::loose loose_t;
    static constexpr uint32_t kTerms = terms_of(Cls), kNR = NR, kNC = S::kNC, kPer = S::kPer;

    // the tile's vectors: [i][0] and [i][1] are the two halves of the line of row 16 i + lane % 16
    // Whole lines, which only this wavefront touches, are streamed past L2 (Stream); where tiles share lines they meet there.
    template <bool Edge, bool Stream> static __device__ __forceinline__ void load(const MergeJob &job, uint32_t r0, uint32_t c0, uint32_t lane, v4u (&w)[kNR][2]) {
        const uint32_t col = c0 + (lane & 1) * 4 * kPer + (lane >> 4) * kPer;
#pragma unroll
        for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
            for (uint32_t v = 0; v < 2; ++v) { // as loaded: even rows, then odd rows, a line by eight lanes
                const uint32_t row = r0 + 16 * i + (lane & 14) + v;
                const char *at = job.src + (uint64_t)row * job.src_pitch + (uint64_t)col * S::kSize;
                if (!Edge || (row < job.rows && col + kPer <= job.cols)) {
                    if constexpr (Stream) w[i][v] = __builtin_nontemporal_load((const FSTX_GLOBAL loose_t *)at);
                    else w[i][v] = *(const FSTX_GLOBAL loose_t *)at;
                } else {
                    w[i][v] = v4u{0, 0, 0, 0};
                    if (row < job.rows && col < job.cols) w[i][v] = load_tail(at, (job.cols - col) * S::kSize);
                }
            }
    }

    template <bool Edge, bool Stream>
    static __device__ __forceinline__ void finish(const MergeJob &job, uint32_t r0, uint32_t c0, uint32_t lane, v4u (&w)[kNR][2], const v4f (&acc)[kNR][kNC],
                                                  const float (&scale)[kNR]) {
        const uint32_t col = c0 + (lane & 1) * 4 * kPer + (lane >> 4) * kPer;
#pragma unroll
        for (uint32_t i = 0; i < kNR; ++i) {
            trade(w[i][0], w[i][1], lane & 1);
#pragma unroll
            for (uint32_t v = 0; v < 2; ++v) {
                float sums[kPer];
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) sums[e] = acc[i][v * (kPer / 4) + e / 4][e % 4];
                w[i][v] = merged<T>(w[i][v], sums, scale[i]);
            }
            trade(w[i][0], w[i][1], lane & 1);
#pragma unroll
            for (uint32_t v = 0; v < 2; ++v) {
                const uint32_t row = r0 + 16 * i + (lane & 14) + v;
                char *at = job.dst + (uint64_t)row * job.dst_pitch + (uint64_t)col * S::kSize;
                if (!Edge || (row < job.rows && col + kPer <= job.cols)) {
                    if constexpr (Stream) __builtin_nontemporal_store(w[i][v], (FSTX_GLOBAL loose_t *)at);
                    else *(FSTX_GLOBAL loose_t *)at = w[i][v];
                } else if (row < job.rows && col < job.cols) {
                    store_tail(at, (job.cols - col) * S::kSize, w[i][v]);
                }
            }
        }
    }

    // what a lane's sums are multiplied with, per row
    static __device__ __forceinline__ void scales(const MergeJob &job, uint32_t r0, uint32_t lane, float (&scale)[kNR]) {
#pragma unroll
        for (uint32_t i = 0; i < kNR; ++i) {
            scale[i] = job.scale;
            if constexpr (T == FSTX_F8_E4M3) {
                const uint32_t row = r0 + 16 * i + (lane & 15), at = row < job.rows ? row : 0;
                scale[i] = job.scale / *(const FSTX_GLOBAL float *)(job.weight_scale + (uint64_t)at * job.scale_step);
            }
        }
    }

    static __device__ __forceinline__ void fetch(const uint16_t *at, uint64_t step, op_t (&f)[kTerms], uint32_t i) {
#pragma unroll
        for (uint32_t p = 0; p < kTerms; ++p) f[p] = *(const FSTX_GLOBAL op_t *)(at + i * step + p * kBlk);
    }

    // term a of one factor with term b of the other as long as a + b < terms, small ones first
    static __device__ __forceinline__ void multiply(const op_t (&u)[kNR][kTerms], const op_t (&d)[kNC][kTerms], v4f (&acc)[kNR][kNC]) {
#pragma unroll
        for (int sum = (int)kTerms - 1; sum >= 0; --sum)
#pragma unroll
            for (int a = 0; a <= sum; ++a)
#pragma unroll
                for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < kNC; ++j) acc[i][j] = mfma(d[j][a], u[i][sum - a], acc[i][j]);
    }

    // one tile whose weights are in w (or on their way)
    template <uint32_t kHeld, bool Edge, bool Stream>
    static __device__ __forceinline__ void tile(const MergeJob &job, uint32_t r0, uint32_t c0, uint32_t lane, v4u (&w)[kNR][2],
                                                const op_t (&held)[kHeld ? kHeld : 1][kNR][kTerms], const op_t (&d)[kHeld ? kHeld : 1][kNC][kTerms],
                                                const float (&scale)[kNR]) {
        v4f acc[kNR][kNC] = {};
        if constexpr (kHeld > 0) {
#pragma unroll
            for (uint32_t kb = 0; kb < kHeld; ++kb) multiply(held[kb], d[kb], acc);
        } else {
            const uint64_t step = (uint64_t)job.k_blocks * kTerms * kBlk;
            const uint16_t *up = job.up + r0 / 16 * step + lane * 8, *down = job.down + c0 / 16 * step + lane * 8;
            for (uint32_t kb = 0; kb < job.k_blocks; ++kb, up += kTerms * kBlk, down += kTerms * kBlk) {
                op_t u[kNR][kTerms], dd[kNC][kTerms];
#pragma unroll
                for (uint32_t i = 0; i < kNR; ++i) fetch(up, step, u[i], i);
#pragma unroll
                for (uint32_t j = 0; j < kNC; ++j) fetch(down, step, dd[j], j);
                multiply(u, dd, acc);
            }
        }
        finish<Edge, Stream>(job, r0, c0, lane, w, acc, scale);
    }

    // A wavefront walks along a panel of kRows rows: the rows' factor stays in registers (kHeld blocks of 32 k; 0: too
    // many, both factors are read per tile), the columns' factor comes from L2, and the weights of the next tile are on
    // their way while one is worked on.
    // (Stream and the tiles at the edges are told apart outside the loop: with a branch around the loads the compiler
    // would have to wait for all of them.)
    template <uint32_t kHeld, bool Stream> static __device__ __forceinline__ void walk(const MergeJob &job, uint32_t r0, uint32_t first, uint32_t last, uint32_t lane) {
        constexpr uint32_t kH = kHeld ? kHeld : 1;
        float scale[kNR];
        scales(job, r0, lane, scale);
        const uint64_t step = (uint64_t)job.k_blocks * kTerms * kBlk;
        op_t held[kH][kNR][kTerms], d[kH][kNC][kTerms];
        if constexpr (kHeld > 0)
#pragma unroll
            for (uint32_t kb = 0; kb < kHeld; ++kb)
#pragma unroll
                for (uint32_t i = 0; i < kNR; ++i) fetch(job.up + r0 / 16 * step + kb * kTerms * kBlk + lane * 8, step, held[kb][i], i);
        auto columns = [&](uint32_t t) {
            if constexpr (kHeld > 0)
#pragma unroll
                for (uint32_t kb = 0; kb < kHeld; ++kb)
#pragma unroll
                    for (uint32_t j = 0; j < kNC; ++j) fetch(job.down + (uint64_t)t * kNC * step + kb * kTerms * kBlk + lane * 8, step, d[kb][j], j);
        };
        const uint32_t whole = r0 + 16 * kNR <= job.rows ? job.cols / S::kCols : 0; // tiles of the panel without an edge
        const uint32_t full = last < whole ? last : whole;
        v4u w[kNR][2], next[kNR][2];
        auto advance = [&]() {
#pragma unroll
            for (uint32_t i = 0; i < kNR; ++i)
#pragma unroll
                for (uint32_t v = 0; v < 2; ++v) w[i][v] = next[i][v];
        };
        uint32_t t = first;
        if (t < full) {
            load<false, Stream>(job, r0, t * S::kCols, lane, w);
            for (; t + 1 < full; ++t) {
                columns(t);
                load<false, Stream>(job, r0, (t + 1) * S::kCols, lane, next);
                tile<kHeld, false, Stream>(job, r0, t * S::kCols, lane, w, held, d, scale);
                advance();
            }
            columns(t);
            if (t + 1 < last) load<true, false>(job, r0, (t + 1) * S::kCols, lane, next);
            tile<kHeld, false, Stream>(job, r0, t * S::kCols, lane, w, held, d, scale);
            advance();
            ++t;
        } else {
            load<true, false>(job, r0, t * S::kCols, lane, w);
        }
        for (; t < last; ++t) {
            columns(t);
            if (t + 1 < last) load<true, false>(job, r0, (t + 1) * S::kCols, lane, next);
            tile<kHeld, true, false>(job, r0, t * S::kCols, lane, w, held, d, scale);
            advance();
        }
    }
};

template <uint32_t T, uint32_t Cls, uint32_t kHeld>
__global__ __launch_bounds__(64, 2) void low_rank_kernel(const uint32_t dies_log2, const Jobs<MergeJob> t) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const MergeJob &job = t.job[ji];
    uint32_t at;
    if (!fstx_gather::tile_for_die(blockIdx.x - t.first[ji], job.n_walks, dies_log2, at)) return;
    const uint32_t panel = at / job.walks, nth = at - panel * job.walks; // neighbours walk along the same panel
    const uint32_t first = nth * job.walk, last = first + job.walk < job.col_tiles ? first + job.walk : job.col_tiles;
    if (job.lines == 3) Merge<T, Cls>::template walk<kHeld, true>(job, panel * Tile<T>::kRows, first, last, threadIdx.x);
    else Merge<T, Cls>::template walk<kHeld, false>(job, panel * Tile<T>::kRows, first, last, threadIdx.x);
}

// Longer products: four wavefronts (2 x 2 tiles) share the operands through LDS, 32 k at a time, the next ones on
// their way while these are multiplied; a wavefront of its own would read both factors from L2 for each of its tiles. The
// weights come last: another workgroup on the compute unit fills that time.
template <uint32_t T, uint32_t Cls>
__global__ __launch_bounds__(256, 2) void deep_low_rank_kernel(const uint32_t dies_log2, const Jobs<MergeJob> t) {
    typedef Merge<T, Cls> M;
    typedef typename M::op_t op_t;
    constexpr uint32_t kTerms = M::kTerms, kNR = M::kNR, kNC = M::kNC;
    constexpr uint32_t kUp = 2 * kNR * kTerms, kStage = kUp + 2 * kNC * kTerms; // operand blocks of a stage: rows', then columns'
    __shared__ __attribute__((aligned(1024))) uint16_t lds[2 * kStage * kBlk];
    const uint32_t ji = job_of(t, blockIdx.x);
    const MergeJob &job = t.job[ji];
    uint32_t at;
    if (!fstx_gather::tile_for_die(blockIdx.x - t.first[ji], job.n_walks, dies_log2, at)) return;
    const uint32_t panel = at / job.walks, nth = at - panel * job.walks;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t step = (uint64_t)job.k_blocks * kTerms * kBlk;
    const uint16_t *up = job.up + (uint64_t)panel * 2 * kNR * step + lane * 8, *down = job.down + (uint64_t)nth * 2 * kNC * step + lane * 8;
    auto load_stage = [&](uint32_t kb, uint32_t buf) {
#pragma unroll
        for (uint32_t n = 0; n < kStage / 4; ++n) {
            const uint32_t b = n * 4 + wave, in = b < kUp ? b : b - kUp;
            const uint16_t *from = (b < kUp ? up : down) + in / kTerms * step + ((uint64_t)kb * kTerms + in % kTerms) * kBlk;
            __builtin_amdgcn_global_load_lds((const FSTX_GLOBAL void *)from, (FSTX_LDS void *)(lds + (buf * kStage + b) * kBlk), 16, 0, 0);
        }
    };
    v4f acc[kNR][kNC] = {};
    load_stage(0, 0);
    for (uint32_t kb = 0; kb < job.k_blocks; ++kb) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070); // this wavefront's loads have landed and its reads are done,
        __builtin_amdgcn_s_barrier();       // and everybody's
        asm volatile("" ::: "memory");
        const uint16_t *base = lds + (kb & 1) * kStage * kBlk + lane * 8;
        op_t u[kNR][kTerms], d[kNC][kTerms];
#pragma unroll
        for (uint32_t p = 0; p < kTerms; ++p) {
#pragma unroll
            for (uint32_t i = 0; i < kNR; ++i) u[i][p] = *(const op_t *)(base + (((wave >> 1) * kNR + i) * kTerms + p) * kBlk);
#pragma unroll
            for (uint32_t j = 0; j < kNC; ++j) d[j][p] = *(const op_t *)(base + (kUp + ((wave & 1) * kNC + j) * kTerms + p) * kBlk);
        }
        if (kb + 1 < job.k_blocks) load_stage(kb + 1, (kb + 1) & 1);
        M::multiply(u, d, acc);
    }
    const uint32_t r0 = (panel * 2 + (wave >> 1)) * Tile<T>::kRows, c0 = (nth * 2 + (wave & 1)) * Tile<T>::kCols;
    if (r0 >= job.rows || c0 >= job.cols) return; // (no barrier follows)
    float scale[kNR];
    M::scales(job, r0, lane, scale);
    v4u w[kNR][2];
    if (r0 + Tile<T>::kRows <= job.rows && c0 + Tile<T>::kCols <= job.cols) {
        if (job.lines == 3) {
            M::template load<false, true>(job, r0, c0, lane, w);
            M::template finish<false, true>(job, r0, c0, lane, w, acc, scale);
        } else {
            M::template load<false, false>(job, r0, c0, lane, w);
            M::template finish<false, false>(job, r0, c0, lane, w, acc, scale);
        }
    } else {
        M::template load<true, false>(job, r0, c0, lane, w);
        M::template finish<true, false>(job, r0, c0, lane, w, acc, scale);
    }
}

// Few tiles and a rank of at most 32: a launch of its own for the factors would take as long as the merge.  Four wavefronts lay
// out the operands of their common tile (64 rows of one line) in LDS and take 16 rows of it each.
struct alignas(64) DirectJob {
    MergeJob merge;
    const char *up, *down;
    uint64_t up_row, up_k, down_col, down_k; // strides, elements
    uint32_t rank, up_type, down_type, pad;
};
static_assert(sizeof(DirectJob) == 192, "12 of them fit the kernel arguments");
constexpr uint32_t kDirectJobs = 12;
struct DirectJobs {
    DirectJob job[kDirectJobs];
    uint32_t first[kDirectJobs];
};

template <uint32_t T, uint32_t Cls> __global__ __launch_bounds__(256) void direct_low_rank_kernel(const DirectJobs t) {
    typedef Merge<T, Cls, 1> M;
    typedef typename M::op_t op_t;
    constexpr uint32_t kTerms = M::kTerms, kNC = M::kNC, kBlocks = 4 + kNC;
    __shared__ __attribute__((aligned(16))) uint16_t lds[kBlocks * kTerms * kBlk];
    uint32_t ji = 0;
#pragma unroll
    for (uint32_t i = 1; i < kDirectJobs; ++i) ji += blockIdx.x >= t.first[i];
    const DirectJob &job = t.job[ji];
    const MergeJob &m = job.merge;
    const uint32_t at = blockIdx.x - t.first[ji], panel = at / m.col_tiles, tile = at - panel * m.col_tiles;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rho = lane & 15, k0 = 8 * (lane >> 4);
    const uint32_t r0 = panel * 64 + wave * 16, c0 = tile * Tile<T>::kCols;
    const bool inside = r0 + 16 <= m.rows && c0 + Tile<T>::kCols <= m.cols;
    v4u w[1][2];
    if (inside) M::template load<false, false>(m, r0, c0, lane, w);
    else M::template load<true, false>(m, r0, c0, lane, w);
#pragma unroll
    for (uint32_t n = 0; n < (kBlocks + 3) / 4; ++n) { // blocks of the rows' factor, then of the columns'
        const uint32_t b = n * 4 + wave;
        if (b >= kBlocks) break;
        const bool cols = b >= 4;
        const uint32_t row = cols ? c0 + column_of(b - 4, rho, M::kPer) : panel * 64 + b * 16 + rho;
        const char *src = cols ? job.down : job.up;
        const uint64_t row_stride = cols ? job.down_col : job.up_row, k_stride = cols ? job.down_k : job.up_k;
        const uint32_t type = cols ? job.down_type : job.up_type;
        const bool live = row < (cols ? m.cols : m.rows);
        float x[8] = {};
        if (job.rank)
            load_factor(src, type, x, [&](uint32_t e) { return (uint64_t)row * row_stride + (uint64_t)(k0 + e) * k_stride; },
                        [&](uint32_t e) { return live && k0 + e < job.rank; });
        uint16_t *out = lds + b * kTerms * kBlk + lane * 8;
        if constexpr (Cls == kTermsH1) *(v8h *)out = half_terms(x);
        else
#pragma unroll
            for (uint32_t p = 0; p < kTerms; ++p) *(v8b *)(out + p * kBlk) = next_term(x);
    }
    __syncthreads();
    op_t u[1][kTerms], d[kNC][kTerms];
#pragma unroll
    for (uint32_t p = 0; p < kTerms; ++p) {
        u[0][p] = *(const op_t *)(lds + (wave * kTerms + p) * kBlk + lane * 8);
#pragma unroll
        for (uint32_t j = 0; j < kNC; ++j) d[j][p] = *(const op_t *)(lds + ((4 + j) * kTerms + p) * kBlk + lane * 8);
    }
    v4f acc[1][kNC] = {};
    M::multiply(u, d, acc);
    float scale[1];
    M::scales(m, r0, lane, scale);
    if (inside) M::template finish<false, false>(m, r0, c0, lane, w, acc, scale);
    else M::template finish<true, false>(m, r0, c0, lane, w, acc, scale);
}

// --------------------------------------------------------------- host side

constexpr uint64_t kMaxSide = 0x7fffff00ull;    // rows, columns: positions stay in 32 bits
// One launch without packing up to here: a [768, 2304] fp32 weight (864 tiles) 12 us instead of 16 with what the host does, three
// fp16 ones of 2304 tiles 18.6 instead of 21.9; beyond it the tiles' own reads of the factors take more than that.
constexpr uint64_t kDirectTiles = 4096;
constexpr uint64_t kWaves = 4096;          // wavefronts that fill the device (eight per compute unit) twice
constexpr uint64_t kLongestWalk = 4;
constexpr uint64_t kLaunchBlocks = 12ull << 20; // workgroups of up to 256 lanes per launch: 32 bits of lanes

inline uint32_t size_of(uint32_t type) { return type == FSTX_F32 ? 4 : type == FSTX_F8_E4M3 ? 1 : 2; }
inline bool factor_type_ok(uint32_t t) { return t == FSTX_F32 || t == FSTX_F16 || t == FSTX_BF16; }
inline uint64_t blocks16(uint64_t n) { return (n + kTile - 1) / kTile * (kTile / 16); }
inline uint64_t k_blocks_of(const fstx_low_rank_desc &d) { return (d.rank + kK - 1) / kK; }

inline uint32_t class_of(const fstx_low_rank_desc &d) {
    if (d.up_type == FSTX_BF16 && d.down_type == FSTX_BF16) return kTermsB1;
    if (d.up_type == FSTX_F16 && d.down_type == FSTX_F16) return kTermsH1;
    return d.type == FSTX_F32 ? kTermsB3 : kTermsB2;
}

inline bool empty(const fstx_low_rank_desc &d) { return d.rows == 0 || d.cols == 0; }

using fstx_overlap::Block;
using fstx_overlap::block_of;
Block dst_of(const fstx_low_rank_desc &d) { return block_of(d.dst, d.rows, d.cols, d.dst_pitch, size_of(d.type)); }
Block src_of(const fstx_low_rank_desc &d) { return block_of(d.src, d.rows, d.cols, d.src_pitch, size_of(d.type)); }
constexpr uint64_t kMaxSpan = 1ull << 48; // elements from a matrix's first to its last

int check(const fstx_low_rank_desc *descs, uint32_t n) {
    if (n && !descs) return -FSTX_E_INVAL;
    for (uint32_t i = 0; i < n; ++i) {
        const fstx_low_rank_desc &d = descs[i];
        if (d.type != FSTX_F32 && d.type != FSTX_F16 && d.type != FSTX_BF16 && d.type != FSTX_F8_E4M3) return -FSTX_E_INVAL;
        if (!factor_type_ok(d.up_type) || !factor_type_ok(d.down_type)) return -FSTX_E_INVAL;
        if (empty(d)) continue;
        const uint64_t size = size_of(d.type);
        if (d.rows > kMaxSide || d.cols > kMaxSide || d.rank > kMaxSide) return -FSTX_E_RANGE;
        if (!d.dst || !d.src || (uintptr_t)d.dst % size || (uintptr_t)d.src % size) return -FSTX_E_INVAL;
        if (d.rows > 1 && (d.dst_pitch < d.cols || d.src_pitch < d.cols || d.dst_pitch >> 40 || d.src_pitch >> 40)) return -FSTX_E_INVAL;
        if (d.rank) {
            if (!d.up || !d.down || (uintptr_t)d.up % size_of(d.up_type) || (uintptr_t)d.down % size_of(d.down_type)) return -FSTX_E_INVAL;
            if ((d.up_row_stride | d.up_col_stride | d.down_row_stride | d.down_col_stride) >> 31) return -FSTX_E_RANGE;
        }
        if (d.rows > 1 && ((d.dst_pitch > d.src_pitch ? d.dst_pitch : d.src_pitch) > kMaxSpan / d.rows)) return -FSTX_E_RANGE;
        const bool eight = d.type == FSTX_F8_E4M3;
        if (eight ? !d.weight_scale || (uintptr_t)d.weight_scale % 4 || (d.n_weight_scales != 1 && d.n_weight_scales != d.rows)
                  : d.weight_scale != nullptr || d.n_weight_scales != 0)
            return -FSTX_E_INVAL;
        const uint64_t tiles = (d.rows + 31) / 32 * ((d.cols + 31) / 32); // more than there are of any type
        if (tiles > kLaunchBlocks / 2 || (blocks16(d.rows) + blocks16(d.cols)) * k_blocks_of(d) > kLaunchBlocks / 2) return -FSTX_E_RANGE;
        // in place, or a source that the destination does not touch
        const bool in_place = d.dst == d.src && (d.rows == 1 || d.dst_pitch == d.src_pitch);
        if (!in_place && fstx_overlap::overlap(dst_of(d), src_of(d))) return -FSTX_E_INVAL;
    }
    fstx_overlap::List list(5ull * n);
    if (!list.at) return -ENOMEM;
    for (uint32_t i = 0; i < n; ++i) {
        const fstx_low_rank_desc &d = descs[i];
        if (empty(d)) continue;
        list.add(dst_of(d), i, fstx_overlap::kWritten);
        list.add(src_of(d), i, fstx_overlap::kSource);
        if (d.rank) {
            list.add(block_of(d.up, d.rows, d.up_row_stride, d.rank, d.up_col_stride, size_of(d.up_type)), i, fstx_overlap::kRead);
            list.add(block_of(d.down, d.rank, d.down_row_stride, d.cols, d.down_col_stride, size_of(d.down_type)), i, fstx_overlap::kRead);
        }
        if (d.weight_scale) list.add(block_of(d.weight_scale, 1, d.n_weight_scales, 0, sizeof(float)), i, fstx_overlap::kRead);
    }
    if (fstx_overlap::any_conflict(list.at, list.n)) return -FSTX_E_INVAL;
    return 0;
}

uint64_t packed_elems(uint64_t side, const fstx_low_rank_desc &d) {
    return blocks16(side) * k_blocks_of(d) * terms_of(class_of(d)) * kBlk;
}

template <typename Job> void clear(Jobs<Job> &t) {
    for (uint32_t i = 0; i < kMaxJobs; ++i) t.first[i] = 0xffffffffu;
}

constexpr uint32_t kDeep = 3;
// Blocks of 32 k of the rows' factor that stay in registers
template <uint32_t T, uint32_t Cls> constexpr uint32_t held_most() { return Cls == kTermsB3 ? 1 : Cls == kTermsB2 ? 1 : 2; }

template <uint32_t T, uint32_t Cls> void launch(uint32_t grid, uint32_t held, const Jobs<MergeJob> &t, hipStream_t s) {
    const uint32_t dies = fstx_internal::dies_log2();
    if (held == 1) hipLaunchKernelGGL((low_rank_kernel<T, Cls, 1>), dim3(grid), dim3(64), 0, s, dies, t);
    else if (held == 2 && held_most<T, Cls>() >= 2) hipLaunchKernelGGL((low_rank_kernel<T, Cls, held_most<T, Cls>() >= 2 ? 2 : 1>), dim3(grid), dim3(64), 0, s, dies, t);
    else if (held == kDeep) hipLaunchKernelGGL((deep_low_rank_kernel<T, Cls>), dim3(grid), dim3(256), 0, s, dies, t);
    else hipLaunchKernelGGL((low_rank_kernel<T, Cls, 0>), dim3(grid), dim3(64), 0, s, dies, t);
}

void launch_class(uint32_t type, uint32_t cls, uint32_t held, uint32_t grid, const Jobs<MergeJob> &t, hipStream_t s) {
#define FSTX_CASE(T, C) case (T) * kTermClasses + (C): launch<T, C>(grid, held, t, s); break;
    switch (type * kTermClasses + cls) {
        FSTX_CASE(FSTX_F32, kTermsH1) FSTX_CASE(FSTX_F32, kTermsB1) FSTX_CASE(FSTX_F32, kTermsB3)
        FSTX_CASE(FSTX_BF16, kTermsH1) FSTX_CASE(FSTX_BF16, kTermsB1) FSTX_CASE(FSTX_BF16, kTermsB2)
        FSTX_CASE(FSTX_F16, kTermsH1) FSTX_CASE(FSTX_F16, kTermsB1) FSTX_CASE(FSTX_F16, kTermsB2)
        FSTX_CASE(FSTX_F8_E4M3, kTermsH1) FSTX_CASE(FSTX_F8_E4M3, kTermsB1) FSTX_CASE(FSTX_F8_E4M3, kTermsB2)
    default: break; // class_of gives no others
    }
#undef FSTX_CASE
}

// whether rows lie on whole 128-byte lines: bit 0 the destination's, bit 1 the source's
inline uint32_t on_lines(const fstx_low_rank_desc &d) {
    const uint64_t size = size_of(d.type), dp = d.rows == 1 ? 0 : d.dst_pitch * size, sp = d.rows == 1 ? 0 : d.src_pitch * size;
    return ((((uint64_t)(uintptr_t)d.dst | dp) & 127) == 0 ? 1u : 0u) | ((((uint64_t)(uintptr_t)d.src | sp) & 127) == 0 ? 2u : 0u);
}

// Which kernel variant serves a descriptor: the number of blocks of the rows' factor that stay in registers, or 0 (walks
// without), or kDeep.  [4096, 4096], walks against the deep kernel: bf16 weights, rank 96 24.0 / 22.7 us, 256 35.5 / 29.2, 512 52.6 /
// 39.3; fp8, rank 256 34.2 / 22.7; f32 weights, which have half the products per byte and twice the bytes to bring,
// rank 64 in three terms 41.0 / 48.4 and 128 53.5 / 56.1, rank 256 in one 47.8 / 50.0: from about 14 blocks times terms on.
inline uint32_t held_of(const fstx_low_rank_desc &d) {
    const uint64_t kb = k_blocks_of(d), most = terms_of(class_of(d)) > 1 ? 1 : 2;
    return kb <= most ? (uint32_t)kb : size_of(d.type) == 4 && kb * terms_of(class_of(d)) < 14 ? 0 : kDeep;
}

// Whether the whole call goes through direct_low_rank_kernel
bool direct(const fstx_low_rank_desc *descs, uint32_t n) {
    uint64_t tiles = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const fstx_low_rank_desc &d = descs[i];
        if (empty(d)) continue;
        if (d.rank > kK) return false;
        tiles += (d.rows + 63) / 64 * ((d.cols * size_of(d.type) + 127) / 128);
    }
    return tiles <= kDirectTiles;
}

} // namespace

extern "C" int64_t fstx_merge_low_rank_workspace(const fstx_low_rank_desc *descs, uint32_t n) {
    const int rc = check(descs, n);
    if (rc < 0) return rc;
    if (direct(descs, n)) return 0;
    uint64_t elems = 0;
    for (uint32_t i = 0; i < n; ++i)
        if (!empty(descs[i])) elems += packed_elems(descs[i].rows, descs[i]) + packed_elems(descs[i].cols, descs[i]);
    return (int64_t)(elems * 2);
}

namespace {

template <uint32_t T, uint32_t Cls> void launch_direct(uint32_t grid, const DirectJobs &t, hipStream_t s) {
    hipLaunchKernelGGL((direct_low_rank_kernel<T, Cls>), dim3(grid), dim3(256), 0, s, t);
}

int merge_direct(const fstx_low_rank_desc *descs, uint32_t n, hipStream_t s) {
    uint64_t done = 0; // variants met so far
    for (uint32_t first = 0; first < n; ++first) {
        if (empty(descs[first])) continue;
        const uint32_t type = descs[first].type, cls = class_of(descs[first]), variant = type * kTermClasses + cls;
        if (done >> variant & 1) continue;
        done |= 1ull << variant;
        DirectJobs t;
        for (uint32_t i = 0; i < kDirectJobs; ++i) t.first[i] = 0xffffffffu;
        uint32_t k = 0;
        uint64_t grid = 0;
        auto flush = [&]() -> int {
            if (k == 0) return 0;
            fstx_internal::Range range("fstx direct_low_rank_kernel: %u jobs, %llu workgroups", k, (unsigned long long)grid);
#define FSTX_CASE(T, C) case (T) * kTermClasses + (C): launch_direct<T, C>((uint32_t)grid, t, s); break;
            switch (variant) {
                FSTX_CASE(FSTX_F32, kTermsH1) FSTX_CASE(FSTX_F32, kTermsB1) FSTX_CASE(FSTX_F32, kTermsB3)
                FSTX_CASE(FSTX_BF16, kTermsH1) FSTX_CASE(FSTX_BF16, kTermsB1) FSTX_CASE(FSTX_BF16, kTermsB2)
                FSTX_CASE(FSTX_F16, kTermsH1) FSTX_CASE(FSTX_F16, kTermsB1) FSTX_CASE(FSTX_F16, kTermsB2)
                FSTX_CASE(FSTX_F8_E4M3, kTermsH1) FSTX_CASE(FSTX_F8_E4M3, kTermsB1) FSTX_CASE(FSTX_F8_E4M3, kTermsB2)
            default: break; // class_of gives no others
            }
#undef FSTX_CASE
            k = 0;
            grid = 0;
            for (uint32_t i = 0; i < kDirectJobs; ++i) t.first[i] = 0xffffffffu;
            return fstx_internal::check_launch("direct_low_rank_kernel");
        };
        for (uint32_t i = first; i < n; ++i) {
            const fstx_low_rank_desc &d = descs[i];
            if (empty(d) || d.type != type || class_of(d) != cls) continue;
            if (k == kDirectJobs) {
                const int rc = flush();
                if (rc < 0) return rc;
            }
            const uint64_t size = size_of(type), col_tiles = (d.cols * size + 127) / 128;
            DirectJob &j = t.job[k];
            j = DirectJob{};
            j.merge.dst = static_cast<char *>(d.dst);
            j.merge.src = static_cast<const char *>(d.src);
            j.merge.weight_scale = d.weight_scale;
            j.merge.dst_pitch = d.dst_pitch * size;
            j.merge.src_pitch = d.src_pitch * size;
            j.merge.rows = (uint32_t)d.rows;
            j.merge.cols = (uint32_t)d.cols;
            j.merge.col_tiles = (uint32_t)col_tiles;
            j.merge.scale = d.scale;
            j.merge.scale_step = d.n_weight_scales > 1;
            j.up = static_cast<const char *>(d.up);
            j.down = static_cast<const char *>(d.down);
            j.up_row = d.up_row_stride;
            j.up_k = d.up_col_stride;
            j.down_col = d.down_col_stride;
            j.down_k = d.down_row_stride;
            j.rank = (uint32_t)d.rank;
            j.up_type = d.up_type;
            j.down_type = d.down_type;
            t.first[k++] = (uint32_t)grid;
            grid += (d.rows + 63) / 64 * col_tiles;
        }
        const int rc = flush();
        if (rc < 0) return rc;
    }
    return 0;
}

} // namespace

extern "C" int fstx_merge_low_rank(const fstx_low_rank_desc *descs, uint32_t n, void *workspace, uint64_t workspace_bytes, void *stream) {
    const int64_t need = fstx_merge_low_rank_workspace(descs, n);
    if (need < 0) return (int)need;
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (uint64_t)need)) return -FSTX_E_INVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (direct(descs, n)) return merge_direct(descs, n, s);
    uint16_t *const space = static_cast<uint16_t *>(workspace);
    { // factors -> operands
        Jobs<PackJob> t;
        clear(t);
        uint32_t k = 0;
        uint64_t grid = 0, at = 0;
        auto flush = [&]() -> int {
            if (k == 0) return 0;
            fstx_internal::Range range("fstx pack_factors_kernel: %u jobs, %llu workgroups", k, (unsigned long long)grid);
            hipLaunchKernelGGL(pack_factors_kernel, dim3((uint32_t)grid), dim3(256), 0, s, t);
            k = 0;
            grid = 0;
            clear(t);
            return fstx_internal::check_launch("pack_factors_kernel");
        };
        for (uint32_t i = 0; i < n; ++i) {
            const fstx_low_rank_desc &d = descs[i];
            if (empty(d) || d.rank == 0) continue;
            const uint64_t kb = k_blocks_of(d), need_blocks = (blocks16(d.rows) + blocks16(d.cols)) * kb / 4;
            if (k + 2 > kMaxJobs || grid + need_blocks > kLaunchBlocks) {
                const int rc = flush();
                if (rc < 0) return rc;
            }
            const uint32_t cls = class_of(d), per = 16 / size_of(d.type);
            for (uint32_t side = 0; side < 2; ++side) {
                const uint64_t len = side ? d.cols : d.rows;
                t.job[k] = side ? PackJob{static_cast<const char *>(d.down), space + at, d.down_col_stride, d.down_row_stride, (uint32_t)len,
                                          (uint32_t)d.rank, (uint32_t)kb, (uint32_t)blocks16(len), d.down_type, terms_of(cls), cls == kTermsH1, per}
                                : PackJob{static_cast<const char *>(d.up), space + at, d.up_row_stride, d.up_col_stride, (uint32_t)len,
                                          (uint32_t)d.rank, (uint32_t)kb, (uint32_t)blocks16(len), d.up_type, terms_of(cls), cls == kTermsH1, 0};
                t.first[k++] = (uint32_t)grid;
                grid += blocks16(len) * kb / 4;
                at += packed_elems(len, d);
            }
        }
        const int rc = flush();
        if (rc < 0) return rc;
    }
    // one launch (or a few) per kernel variant that occurs
    static const uint32_t types[4] = {FSTX_F32, FSTX_BF16, FSTX_F16, FSTX_F8_E4M3};
    const uint64_t dies = 1ull << fstx_internal::dies_log2();
    for (uint32_t variant = 0; variant < 4 * kTermClasses * 4; ++variant) {
        const uint32_t type = types[variant / (kTermClasses * 4)], cls = variant / 4 % kTermClasses, held = variant % 4;
        Jobs<MergeJob> t;
        clear(t);
        uint32_t k = 0;
        uint64_t grid = 0, at = 0;
        auto flush = [&]() -> int {
            if (k == 0) return 0;
            fstx_internal::Range range("fstx low_rank_kernel: %u jobs, %llu workgroups", k, (unsigned long long)grid);
            launch_class(type, cls, held, (uint32_t)grid, t, s);
            k = 0;
            grid = 0;
            clear(t);
            return fstx_internal::check_launch("low_rank_kernel");
        };
        const uint64_t size = size_of(type), across = held == kDeep ? 2 : 1; // a deep workgroup's tile is two by two
        const uint64_t tile_cols = across * 128 / size, tile_rows = across * (size == 1 ? 32 : 64);
        uint64_t tiles = 0; // of the whole call, for the length of the walks
        for (uint32_t i = 0; i < n; ++i)
            if (!empty(descs[i])) tiles += (descs[i].cols + tile_cols - 1) / tile_cols * ((descs[i].rows + tile_rows - 1) / tile_rows);
        for (uint32_t i = 0; i < n; ++i) {
            const fstx_low_rank_desc &d = descs[i];
            if (empty(d)) continue;
            const uint64_t up_at = at, down_at = at + packed_elems(d.rows, d);
            at = down_at + packed_elems(d.cols, d);
            if (d.type != type || class_of(d) != cls || held_of(d) != held) continue;
            const uint64_t col_tiles = (d.cols + tile_cols - 1) / tile_cols, panels = (d.rows + tile_rows - 1) / tile_rows;
            uint64_t walk = tiles / kWaves;
            walk = held == kDeep || walk < 1 ? 1 : walk > kLongestWalk ? kLongestWalk : walk;
            const uint64_t walks = (col_tiles + walk - 1) / walk;
            const uint64_t blocks = (panels * walks + dies - 1) / dies * dies;
            if (k == kMaxJobs || grid + blocks > kLaunchBlocks) {
                const int rc = flush();
                if (rc < 0) return rc;
            }
            t.job[k] = MergeJob{static_cast<char *>(d.dst), static_cast<const char *>(d.src), space + up_at, space + down_at, d.weight_scale,
                                d.dst_pitch * size, d.src_pitch * size, (uint32_t)d.rows, (uint32_t)d.cols, (uint32_t)k_blocks_of(d),
                                (uint32_t)col_tiles, d.scale, d.n_weight_scales > 1 ? 1u : 0u, (uint32_t)walk, (uint32_t)walks, (uint32_t)(panels * walks), on_lines(d), {}};
            t.first[k++] = (uint32_t)grid;
            grid += blocks;
        }
        const int rc = flush();
        if (rc < 0) return rc;
    }
    return 0;
}
