/*
 * mft/rms_norm.h — C ABI of the root-mean-square norm of a residual stream on gfx950.
 *
 * Forward, per row n of D elements:
 *
 *   s = x + residual (rounded to `dtype`, as it is stored), or x without residual
 *   rstd = 1 / sqrt(sum s^2 / D + eps)
 *   y = s * rstd * f,  f = 1 + weight (MFT_NORM_GEMMA) or weight (MFT_NORM_AFFINE); 1 without weight
 *
 * In 8 bits y is held as e4m3 numbers (OCP: largest 448, no infinity) with one
 * fp32 scale a row:
 *
 *   scale = max(max |y| / 448, 2^-126),  q = e4m3(y / scale) to nearest even
 *
 * the division by 448 being a product by the fp32 number next to 1 / 448 (as torch's
 * kernels have it), and y / scale rounded to fp32 first.  A row with an infinity
 * or a NaN has no numbers (its q are NaN, or 0 where y is finite in a row with an
 * infinity).
 * MFT_NORM_NONE holds s itself so: the form in which mft/gated_linear.h takes
 * activations and weights in 8 bits.
 *
 * Backward, with h = s * rstd and g = dy * f:
 *
 *   dx = rstd * (g - h * sum(g h) / D) + dtotal   (also the residual's gradient)
 *   dweight = sum over rows of dy * h
 *
 * dtotal is the gradient that reaches s from elsewhere (the stream behind it).
 *
 * x, residual, total, y, dy, dtotal and dx have element type `dtype`; weight,
 * its gradient, rstd and the scales are fp32, as are all sums.  Each value is
 * rounded to its type once, where it is stored.  Results do not depend on the
 * order in which workgroups run.
 *
 * Conventions are those of mft/layer_norm.h: caller-owned device memory, rows
 * that may start at any element, N from 0 (a zero dweight) to below 2^31, D at
 * most 2^30.
 */
#ifndef MFT_RMS_NORM_H
#define MFT_RMS_NORM_H

#include "mft/attention.h"
#include "mft/prologue.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int64_t N;           /* rows                                              */
    int64_t D;           /* elements of a row                                 */
    int32_t dtype;       /* mft_dtype of the rows                             */
    int32_t norm;        /* mft_norm: how the weight enters                   */
    float eps;
    /* Elements from one row to the next (>= D); 0 = D.  `y` is the 8-bit
     * output's, too. */
    int64_t x_stride, residual_stride, total_stride, y_stride, dy_stride, dtotal_stride, dx_stride;
} mft_rms_norm_desc;

/* y, and the rows' rstd ([N], may be NULL).  weight ([D]) may be NULL.  With a
 * residual, total gets s; without, both are NULL.  y and total may be x or
 * residual where the strides agree; they may not be each other.  MFT_NORM_NONE is refused. */
mft_status mft_rms_norm_fwd(const mft_rms_norm_desc* desc, const void* x, const void* residual, const float* weight,
                            void* total, void* y, float* rstd, hipStream_t stream);

/* The same with y as e4m3 numbers q ([N, D] bytes) and the rows' scales ([N]).
 * MFT_NORM_NONE: y = s, with no weight. */
mft_status mft_rms_norm_e4m3_fwd(const mft_rms_norm_desc* desc, const void* x, const void* residual,
                                 const float* weight, void* total, void* q, float* scale, hipStream_t stream);

/* Bytes of device workspace mft_rms_norm_bwd needs. */
mft_status mft_rms_norm_workspace_size(const mft_rms_norm_desc* desc, size_t* bytes);

/* dx and dweight ([D]) from s (as x: the forward's total, or its x without a
 * residual), the forward's rstd, dy, and dtotal (may be NULL).  dx or dweight may
 * be NULL and is then left out; they are written, not accumulated.  dx may be
 * dy or dtotal where the strides agree; it may not be x. */
mft_status mft_rms_norm_bwd(const mft_rms_norm_desc* desc, const void* x, const float* weight, const float* rstd,
                            const void* dy, const void* dtotal, void* dx, float* dweight, void* workspace,
                            hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MFT_RMS_NORM_H */
