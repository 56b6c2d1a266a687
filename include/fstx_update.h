/* SPDX-License-Identifier: Apache-2.0
 *
 * fstx: kernels that change weights which are in HBM already (same library, libfstx.so).
 *
 *   fstx_merge_low_rank   W' = W + scale * (up @ down): an adapter's factors merged into weights
 *   fstx_orthogonalize    the nearest orthogonal matrix of an update, by Newton-Schulz products
 *
 * No counterpart in the reference, which only moves weights.  Conventions are those of fstx.h:
 * 0 or a negative status, plain pointers and sizes, work is only enqueued on `stream`, nothing is
 * allocated or synchronized, so that calls can be recorded into a HIP graph.  Scratch memory is the
 * caller's: a call uses the first bytes of `workspace`, which must be 256-byte aligned, hold what the
 * matching *_workspace function says, and stay untouched by others until the work on `stream` is done.
 * All arguments are checked before anything is enqueued.
 */
#ifndef FSTX_UPDATE_H
#define FSTX_UPDATE_H

#include "fstx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* dst = round(src + scale * (up @ down)); dst == src (same pitch) merges in place.
 * Products and sums are held in 32 bits; factors of f32 are split into bf16 terms, three for f32 weights
 * (off by 4 * 2^-24 of each product at most) and two for others (3 * 2^-16, which their own rounding hides unless
 * the products cancel).  With FSTX_F8_E4M3 weights W stands for W * weight_scale[row] and the
 * result is (W * weight_scale + scale * up @ down) / weight_scale, saturated to +-448 (a NaN stays one).
 * An infinity in a factor makes its row or column infinite or NaN.  Up to about
 * 6 * 10^9 elements, and 10^8 rows and columns together per 32 of the rank (-FSTX_E_RANGE). */
typedef struct fstx_low_rank_desc {
    void *dst;                  /* [rows, cols] elements of `type`, rows dst_pitch elements apart       */
    const void *src;            /* [rows, cols] elements of `type`, rows src_pitch elements apart       */
    const void *up;             /* [rows, rank] of `up_type`, any strides (elements, below 2^31)         */
    const void *down;           /* [rank, cols] of `down_type`                                          */
    const float *weight_scale;  /* device memory, FSTX_F8_E4M3 only: 1 or `rows` floats                 */
    uint64_t rows, cols, rank;
    uint64_t dst_pitch, src_pitch;
    uint64_t up_row_stride, up_col_stride;
    uint64_t down_row_stride, down_col_stride;
    float scale;
    uint32_t type;              /* FSTX_F32, FSTX_F16, FSTX_BF16 or FSTX_F8_E4M3                        */
    uint32_t up_type;           /* FSTX_F32, FSTX_F16 or FSTX_BF16                                      */
    uint32_t down_type;
    uint32_t n_weight_scales;   /* 0 (other types), 1 or rows                                           */
    uint32_t reserved;
} fstx_low_rank_desc;

/* Bytes of workspace for these descriptors, or a negative status. */
int64_t fstx_merge_low_rank_workspace(const fstx_low_rank_desc *descs, uint32_t n);

/* Any number of merges in a few launches.  No destination may overlap another destination, another
 * descriptor's source, any factor or weight scale (column blocks of one tensor do not overlap). */
int fstx_merge_low_rank(const fstx_low_rank_desc *descs, uint32_t n, void *workspace,
                        uint64_t workspace_bytes, void *stream);

/* dst = the nearest orthogonal matrix of src, approximated by `steps` Newton-Schulz steps:
 *   X = src / (|src|_F + eps);   per step (a, b, c):  A = X X^T,  X <- a X + (b A + c A A) X
 * with the shorter side as rows (orthogonal rows if rows <= cols, else orthogonal columns).  Iterates and
 * operands are held in 22 bits whatever the type, scaled by a bound of the singular values (|src| / (|src| + eps),
 * then |a| s + |b| s^3 + |c| s^5 per step; a step that leaves X far below that, as a = 0 does to many small
 * singular values, costs the bits between the two); sums are held in 32 bits, the norm's in 64.  While the steps run the
 * iterates' singular values must not exceed 2 (those of X start at 1 or less).  With up to 32 rows
 * or columns everything is done in 64 bits.  Infinities and NaN spread through the result
 * as they do in the formula. */
typedef struct fstx_orthogonalize_desc {
    void *dst;                              /* [rows, cols] of `type`, rows dst_pitch elements apart     */
    const void *src;                        /* [rows, cols] of `type`, any strides (elements); dst or apart */
    uint64_t rows, cols;                    /* up to 2^20, the smaller one up to 2^16                    */
    uint64_t dst_pitch;
    uint64_t src_row_stride, src_col_stride;
    uint32_t type;                          /* FSTX_F32, FSTX_F16 or FSTX_BF16                           */
    uint32_t reserved;
} fstx_orthogonalize_desc;

/* Bytes of workspace for these descriptors and steps on the current device, or a negative status. */
int64_t fstx_orthogonalize_workspace(const fstx_orthogonalize_desc *descs, uint32_t n, const float *coefficients,
                                     uint32_t steps);

/* Any number of matrices; those that fit one set of launches together run together.  `coefficients`
 * (host memory) are a, b, c of each of the 1..64 steps, all finite.  No destination may overlap another
 * descriptor's source or destination, or its own source partly. */
int fstx_orthogonalize(const fstx_orthogonalize_desc *descs, uint32_t n, const float *coefficients, uint32_t steps,
                       float eps, void *workspace, uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* FSTX_UPDATE_H */
