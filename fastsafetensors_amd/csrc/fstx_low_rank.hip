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
//   low_rank_kernel      one wavefront per 64 x 64 tile of W: loads its tile of W first (all of it
//                        in flight), accumulates the product from operands that L2 holds, adds,
//                        rounds, stores.  No LDS and no barriers: nothing is shared but the factors.
//
// Numerics.  MFMA products of bf16 / fp16 are exact in fp32 and are summed in fp32.  Factors of
// f32 are split into bf16 terms x = h + m (+ l), each the rounding of what is left: bf16 because it
// has f32's range.  Two terms (16 bits of each factor; h h + h m + m h, what is left out is below
// 2^-17 of a product) for weights of 8 or 16 bits, whose own rounding is 2^-12 at best; three terms
// (24 bits; six products, 2^-25 left out) for f32 weights.  One term where the factors are already
// bf16, or both fp16.
//
// Operand layout.  v_mfma_f32_16x16x32 takes 8 consecutive k of row lane % 16 from each lane
// (k = 8 (lane / 16) + 0..7): a block of 16 rows x 32 k is stored as the 64 lanes' 16 bytes in
// lane order, 1 KiB, so that an operand load is one fully coalesced global_load_dwordx4.  The
// product is computed transposed (D as the first operand): a lane then holds, for ONE row of W, the
// 4 columns that its quarter of the wavefront owns in each 16-column block; and the columns are
// dealt to the blocks so that the blocks of one 16-byte vector of W are consecutive (column_of):
// W goes straight between memory and the accumulator layout, 16 bytes per lane, 64 contiguous
// bytes per row and instruction.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fstx_gather_core.h"
#include "fstx_internal.h"
#include "fstx_update.h"

namespace {

#define FSTX_GLOBAL __attribute__((address_space(1)))
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

constexpr uint32_t kTile = 64;   // rows and columns of W per wavefront
constexpr uint32_t kBlk = 512;   // elements of one operand block (16 rows x 32 k)
constexpr uint32_t kK = 32;      // k per block
constexpr uint32_t kMaxJobs = 32;

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
    uint32_t scale_step; // 0: one weight scale, 1: one per row
    uint32_t n_tiles, pad;
};
static_assert(sizeof(MergeJob) == 96, "32 of them fit the kernel arguments");

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

__device__ __forceinline__ float load_factor(const char *src, uint64_t at, uint32_t type) {
    if (type == FSTX_F32) return *(const FSTX_GLOBAL float *)(src + at * 4);
    const uint16_t raw = *(const FSTX_GLOBAL uint16_t *)(src + at * 2);
    if (type == FSTX_BF16) return __builtin_bit_cast(float, (uint32_t)raw << 16);
    return (float)__builtin_bit_cast(_Float16, raw);
}

// the bf16 nearest to x; where that would overflow a finite x, the one below it
__device__ __forceinline__ float bf16_term(float x) {
    const float h = (float)(__bf16)x;
    if (__builtin_isinf(h) && !__builtin_isinf(x)) return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
    return h;
}

// One wavefront per operand block.
__global__ __launch_bounds__(64) void pack_factors_kernel(const Jobs<PackJob> t) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const PackJob &job = t.job[ji];
    const uint32_t lb = blockIdx.x - t.first[ji];
    const uint32_t blk = lb / job.k_blocks, kb = lb - blk * job.k_blocks;
    const uint32_t lane = threadIdx.x, rho = lane & 15;
    const uint32_t row = job.per ? column_of(blk, rho, job.per) : blk * 16 + rho;
    const uint32_t k0 = kb * kK + 8 * (lane >> 4);
    float x[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
        x[e] = row < job.rows && k0 + e < job.rank
                   ? load_factor(job.src, (uint64_t)row * job.row_stride + (uint64_t)(k0 + e) * job.k_stride, job.type) : 0.0f;
    uint16_t *out = job.dst + ((uint64_t)lb * job.terms) * kBlk + lane * 8;
    if (job.half) {
        v8h h;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) h[e] = (_Float16)x[e];
        *(FSTX_GLOBAL v8h *)out = h;
        return;
    }
    for (uint32_t term = 0; term < job.terms; ++term) {
        v8b h;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const float f = bf16_term(x[e]);
            h[e] = (__bf16)f;
            // what is left for the next term; nothing behind an infinity or a NaN
            x[e] = __builtin_isfinite(f) ? x[e] - f : 0.0f;
        }
        *(FSTX_GLOBAL v8b *)(out + term * kBlk) = h;
    }
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

template <uint32_t T, uint32_t Cls, bool Edge>
__device__ __forceinline__ void merge_tile(const MergeJob &job, uint32_t r0, uint32_t c0) {
    typedef typename Operand<Cls>::type op_t;
    typedef typename Weight<T>::loose loose_t;
    constexpr uint32_t kTerms = terms_of(Cls), kSize = Weight<T>::size, kPer = 16 / kSize;
    constexpr uint32_t kVecs = kTile / (4 * kPer); // 16-byte vectors per lane and row
    constexpr uint32_t kNB = kTile / 16;           // operand blocks along either side
    const uint32_t lane = threadIdx.x, g = lane >> 4;

    // the tile of W, all of it in flight before the product begins
    v4u w[kNB][kVecs];
#pragma unroll
    for (uint32_t i = 0; i < kNB; ++i) {
        const uint32_t row = r0 + 16 * i + (lane & 15);
        const char *at = job.src + (uint64_t)row * job.src_pitch;
#pragma unroll
        for (uint32_t v = 0; v < kVecs; ++v) {
            const uint32_t col = c0 + v * 4 * kPer + g * kPer;
            if (!Edge || (row < job.rows && col + kPer <= job.cols)) {
                w[i][v] = __builtin_nontemporal_load((const FSTX_GLOBAL loose_t *)(at + (uint64_t)col * kSize));
            } else {
                w[i][v] = v4u{0, 0, 0, 0};
                if (row < job.rows && col < job.cols) { // the vector that ends the row: element by element
                    uint8_t part[16] = {};
                    for (uint32_t e = 0; e < (job.cols - col) * kSize; ++e) part[e] = *(const FSTX_GLOBAL uint8_t *)(at + (uint64_t)col * kSize + e);
                    __builtin_memcpy(&w[i][v], part, 16);
                }
            }
        }
    }
    float row_scale[kNB];
#pragma unroll
    for (uint32_t i = 0; i < kNB; ++i) {
        row_scale[i] = job.scale;
        if constexpr (T == FSTX_F8_E4M3) {
            const uint32_t row = r0 + 16 * i + (lane & 15);
            const uint32_t at = Edge && row >= job.rows ? 0 : row;
            row_scale[i] = job.scale / *(const FSTX_GLOBAL float *)(job.weight_scale + (uint64_t)at * job.scale_step);
        }
    }

    v4f acc[kNB][kNB] = {};
    const uint16_t *up = job.up + (uint64_t)(r0 / 16) * job.k_blocks * kTerms * kBlk + lane * 8;
    const uint16_t *down = job.down + (uint64_t)(c0 / 16) * job.k_blocks * kTerms * kBlk + lane * 8;
    const uint64_t step = (uint64_t)job.k_blocks * kTerms * kBlk;
    for (uint32_t kb = 0; kb < job.k_blocks; ++kb) {
        op_t u[kNB][kTerms], d[kNB][kTerms];
#pragma unroll
        for (uint32_t i = 0; i < kNB; ++i)
#pragma unroll
            for (uint32_t p = 0; p < kTerms; ++p) {
                u[i][p] = *(const FSTX_GLOBAL op_t *)(up + i * step + p * kBlk);
                d[i][p] = *(const FSTX_GLOBAL op_t *)(down + i * step + p * kBlk);
            }
#pragma unroll
        for (uint32_t i = 0; i < kNB; ++i)
#pragma unroll
            for (uint32_t j = 0; j < kNB; ++j)
                // term a of one factor with term b of the other as long as a + b < terms, small ones first
#pragma unroll
                for (int sum = (int)kTerms - 1; sum >= 0; --sum)
#pragma unroll
                    for (int a = 0; a <= sum; ++a) acc[i][j] = mfma(d[j][a], u[i][sum - a], acc[i][j]);
        up += kTerms * kBlk;
        down += kTerms * kBlk;
    }

#pragma unroll
    for (uint32_t i = 0; i < kNB; ++i) {
        const uint32_t row = r0 + 16 * i + (lane & 15);
        char *at = job.dst + (uint64_t)row * job.dst_pitch;
#pragma unroll
        for (uint32_t v = 0; v < kVecs; ++v) {
            const uint32_t col = c0 + v * 4 * kPer + g * kPer;
            float sums[kPer];
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) sums[e] = acc[i][v * (kPer / 4) + e / 4][e % 4];
            const v4u out = merged<T>(w[i][v], sums, row_scale[i]);
            if (!Edge || (row < job.rows && col + kPer <= job.cols)) {
                __builtin_nontemporal_store(out, (FSTX_GLOBAL loose_t *)(at + (uint64_t)col * kSize));
            } else if (row < job.rows && col < job.cols) {
                uint8_t part[16];
                __builtin_memcpy(part, &out, 16);
                for (uint32_t e = 0; e < (job.cols - col) * kSize; ++e) *(FSTX_GLOBAL uint8_t *)(at + (uint64_t)col * kSize + e) = part[e];
            }
        }
    }
}

template <uint32_t T, uint32_t Cls>
__global__ __launch_bounds__(64) void low_rank_kernel(const uint32_t dies_log2, const Jobs<MergeJob> t) {
    const uint32_t ji = job_of(t, blockIdx.x);
    const MergeJob &job = t.job[ji];
    uint32_t tile;
    if (!fstx_gather::tile_for_die(blockIdx.x - t.first[ji], job.n_tiles, dies_log2, tile)) return;
    const uint32_t rt = tile / job.col_tiles, ct = tile - rt * job.col_tiles;
    const uint32_t r0 = rt * kTile, c0 = ct * kTile;
    if (r0 + kTile <= job.rows && c0 + kTile <= job.cols) merge_tile<T, Cls, false>(job, r0, c0);
    else merge_tile<T, Cls, true>(job, r0, c0);
}

// --------------------------------------------------------------- host side

constexpr uint64_t kMaxSide = 0x7fffff00ull;    // rows, columns: positions stay in 32 bits
constexpr uint64_t kLaunchBlocks = 48ull << 20; // workgroups of 64 lanes per launch: 32 bits of lanes

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

// a block of bytes: `rows` segments of `width` bytes, `pitch` apart
struct Block {
    uint64_t at, width, pitch, rows;
    uint64_t end() const { return at + (rows - 1) * pitch + width; }
};

bool overlap(const Block &a, const Block &b) {
    if (a.at >= b.end() || b.at >= a.end()) return false;
    if (a.pitch != b.pitch || a.rows == 1 || b.rows == 1) return true; // spans that touch: not told apart further
    if (b.at < a.at) return overlap(b, a);
    // rows of one tensor: b starts `shift` rows and `col` bytes behind a
    const uint64_t shift = (b.at - a.at) / a.pitch, col = (b.at - a.at) % a.pitch;
    if (shift < a.rows && col < a.width) return true;
    return shift + 1 < a.rows && col + b.width > a.pitch; // b's rows run on into a's next rows
}

Block block_of(const void *p, uint64_t rows, uint64_t cols, uint64_t pitch, uint64_t size) {
    return Block{(uint64_t)(uintptr_t)p, cols * size, (rows == 1 ? cols : pitch) * size, rows};
}
Block dst_of(const fstx_low_rank_desc &d) { return block_of(d.dst, d.rows, d.cols, d.dst_pitch, size_of(d.type)); }
Block src_of(const fstx_low_rank_desc &d) { return block_of(d.src, d.rows, d.cols, d.src_pitch, size_of(d.type)); }
Block factor_of(const void *p, uint64_t n0, uint64_t s0, uint64_t n1, uint64_t s1, uint32_t type) {
    const uint64_t last = (n0 - 1) * s0 + (n1 - 1) * s1 + 1;
    return Block{(uint64_t)(uintptr_t)p, last * size_of(type), last * size_of(type), 1};
}

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
        const bool eight = d.type == FSTX_F8_E4M3;
        if (eight ? !d.weight_scale || (uintptr_t)d.weight_scale % 4 || (d.n_weight_scales != 1 && d.n_weight_scales != d.rows)
                  : d.weight_scale != nullptr || d.n_weight_scales != 0)
            return -FSTX_E_INVAL;
        const uint64_t tiles = (d.rows + kTile - 1) / kTile * ((d.cols + kTile - 1) / kTile);
        if (tiles > kLaunchBlocks / 2 || (blocks16(d.rows) + blocks16(d.cols)) * k_blocks_of(d) > kLaunchBlocks / 2) return -FSTX_E_RANGE;
        // in place, or a source that the destination does not touch
        const bool in_place = d.dst == d.src && (d.rows == 1 || d.dst_pitch == d.src_pitch);
        if (!in_place && overlap(dst_of(d), src_of(d))) return -FSTX_E_INVAL;
    }
    for (uint32_t i = 0; i < n; ++i) {
        if (empty(descs[i])) continue;
        const Block out = dst_of(descs[i]);
        for (uint32_t j = 0; j < n; ++j) {
            const fstx_low_rank_desc &d = descs[j];
            if (empty(d)) continue;
            if (j != i && ((j > i && overlap(out, dst_of(d))) || overlap(out, src_of(d)))) return -FSTX_E_INVAL;
            if (d.rank && (overlap(out, factor_of(d.up, d.rows, d.up_row_stride, d.rank, d.up_col_stride, d.up_type)) ||
                           overlap(out, factor_of(d.down, d.rank, d.down_row_stride, d.cols, d.down_col_stride, d.down_type))))
                return -FSTX_E_INVAL;
        }
    }
    return 0;
}

uint64_t packed_elems(uint64_t side, const fstx_low_rank_desc &d) {
    return blocks16(side) * k_blocks_of(d) * terms_of(class_of(d)) * kBlk;
}

template <typename Job> void clear(Jobs<Job> &t) {
    for (uint32_t i = 0; i < kMaxJobs; ++i) t.first[i] = 0xffffffffu;
}

template <uint32_t T, uint32_t Cls> void launch(uint32_t grid, const Jobs<MergeJob> &t, hipStream_t s) {
    hipLaunchKernelGGL((low_rank_kernel<T, Cls>), dim3(grid), dim3(64), 0, s, fstx_internal::dies_log2(), t);
}

void launch_class(uint32_t type, uint32_t cls, uint32_t grid, const Jobs<MergeJob> &t, hipStream_t s) {
#define FSTX_CASE(T, C) case (T) * kTermClasses + (C): launch<T, C>(grid, t, s); break;
    switch (type * kTermClasses + cls) {
        FSTX_CASE(FSTX_F32, kTermsH1) FSTX_CASE(FSTX_F32, kTermsB1) FSTX_CASE(FSTX_F32, kTermsB3)
        FSTX_CASE(FSTX_BF16, kTermsH1) FSTX_CASE(FSTX_BF16, kTermsB1) FSTX_CASE(FSTX_BF16, kTermsB2)
        FSTX_CASE(FSTX_F16, kTermsH1) FSTX_CASE(FSTX_F16, kTermsB1) FSTX_CASE(FSTX_F16, kTermsB2)
        FSTX_CASE(FSTX_F8_E4M3, kTermsH1) FSTX_CASE(FSTX_F8_E4M3, kTermsB1) FSTX_CASE(FSTX_F8_E4M3, kTermsB2)
    default: break; // class_of gives no others
    }
#undef FSTX_CASE
}

} // namespace

extern "C" int64_t fstx_merge_low_rank_workspace(const fstx_low_rank_desc *descs, uint32_t n) {
    const int rc = check(descs, n);
    if (rc < 0) return rc;
    uint64_t elems = 0;
    for (uint32_t i = 0; i < n; ++i)
        if (!empty(descs[i])) elems += packed_elems(descs[i].rows, descs[i]) + packed_elems(descs[i].cols, descs[i]);
    return (int64_t)(elems * 2);
}

extern "C" int fstx_merge_low_rank(const fstx_low_rank_desc *descs, uint32_t n, void *workspace, uint64_t workspace_bytes, void *stream) {
    const int64_t need = fstx_merge_low_rank_workspace(descs, n);
    if (need < 0) return (int)need;
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (uint64_t)need)) return -FSTX_E_INVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint16_t *const space = static_cast<uint16_t *>(workspace);
    { // factors -> operands
        Jobs<PackJob> t;
        clear(t);
        uint32_t k = 0;
        uint64_t grid = 0, at = 0;
        auto flush = [&]() -> int {
            if (k == 0) return 0;
            fstx_internal::Range range("fstx pack_factors_kernel: %u jobs, %llu workgroups", k, (unsigned long long)grid);
            hipLaunchKernelGGL(pack_factors_kernel, dim3((uint32_t)grid), dim3(64), 0, s, t);
            k = 0;
            grid = 0;
            clear(t);
            return fstx_internal::check_launch("pack_factors_kernel");
        };
        for (uint32_t i = 0; i < n; ++i) {
            const fstx_low_rank_desc &d = descs[i];
            if (empty(d) || d.rank == 0) continue;
            const uint64_t kb = k_blocks_of(d), need_blocks = (blocks16(d.rows) + blocks16(d.cols)) * kb;
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
                grid += blocks16(len) * kb;
                at += packed_elems(len, d);
            }
        }
        const int rc = flush();
        if (rc < 0) return rc;
    }
    // one launch (or a few) per kernel variant that occurs
    static const uint32_t types[4] = {FSTX_F32, FSTX_BF16, FSTX_F16, FSTX_F8_E4M3};
    const uint64_t dies = 1ull << fstx_internal::dies_log2();
    for (uint32_t type : types)
        for (uint32_t cls = 0; cls < kTermClasses; ++cls) {
            Jobs<MergeJob> t;
            clear(t);
            uint32_t k = 0;
            uint64_t grid = 0, at = 0;
            auto flush = [&]() -> int {
                if (k == 0) return 0;
                fstx_internal::Range range("fstx low_rank_kernel: %u jobs, %llu workgroups", k, (unsigned long long)grid);
                launch_class(type, cls, (uint32_t)grid, t, s);
                k = 0;
                grid = 0;
                clear(t);
                return fstx_internal::check_launch("low_rank_kernel");
            };
            for (uint32_t i = 0; i < n; ++i) {
                const fstx_low_rank_desc &d = descs[i];
                if (empty(d)) continue;
                const uint64_t up_at = at, down_at = at + packed_elems(d.rows, d);
                at = down_at + packed_elems(d.cols, d);
                if (d.type != type || class_of(d) != cls) continue;
                const uint64_t col_tiles = (d.cols + kTile - 1) / kTile, tiles = (d.rows + kTile - 1) / kTile * col_tiles;
                const uint64_t blocks = (tiles + dies - 1) / dies * dies;
                if (k == kMaxJobs || grid + blocks > kLaunchBlocks) {
                    const int rc = flush();
                    if (rc < 0) return rc;
                }
                const uint64_t size = size_of(type);
                t.job[k] = MergeJob{static_cast<char *>(d.dst), static_cast<const char *>(d.src), space + up_at, space + down_at, d.weight_scale,
                                    d.dst_pitch * size, d.src_pitch * size, (uint32_t)d.rows, (uint32_t)d.cols, (uint32_t)k_blocks_of(d),
                                    (uint32_t)col_tiles, d.scale, d.n_weight_scales > 1 ? 1u : 0u, (uint32_t)tiles, 0};
                t.first[k++] = (uint32_t)grid;
                grid += blocks;
            }
            const int rc = flush();
            if (rc < 0) return rc;
        }
    return 0;
}
