/*
 * mft/layer_norm.h — C ABI of layer norm over the last dimension on gfx950.
 *
 * Forward, per row n of D elements:
 *
 *   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
 *   y = (x - mean) * rstd * weight + bias
 *
 * Backward, with h = (x - mean) * rstd and g = dy * weight:
 *
 *   dx = rstd * (g - sum(g) / D - h * sum(g h) / D)
 *   dweight = sum over rows of dy * h,  dbias = sum over rows of dy
 *
 * x, y, dy and dx have element type `dtype`; weight, bias, their gradients and
 * the row statistics are fp32, as are all sums.  Each value is rounded to
 * `dtype` once, where it is stored.  Results do not depend on the order in
 * which workgroups run.
 *
 * Conventions are those of mft/attention.h (status codes, mft_last_error,
 * caller-owned device memory, stream ordering, no allocation), but rows may
 * start at any element: the base addresses need no more than the alignment of
 * their type, and row strides may be odd.  N may be 0 (the parameters'
 * gradients are then zero); it is below 2^31, and D at most 2^30.
 */
#ifndef MFT_LAYER_NORM_H
#define MFT_LAYER_NORM_H

#include "mft/attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int64_t N;           /* rows                                              */
    int64_t D;           /* elements of a row                                 */
    int32_t dtype;       /* mft_dtype of x, y, dy and dx                      */
    float eps;
    /* Elements from one row to the next (>= D); 0 = D. */
    int64_t x_stride, y_stride, dy_stride, dx_stride;
} mft_layer_norm_desc;

/* y, and the rows' mean and rstd ([N] fp32, each may be NULL).  weight and bias
 * ([D] fp32) may be NULL (1 and 0).  y may be x where the strides agree. */
mft_status mft_layer_norm_fwd(const mft_layer_norm_desc* desc, const void* x, const float* weight, const float* bias,
                              void* y, float* mean, float* rstd, hipStream_t stream);

/* Bytes of device workspace mft_layer_norm_bwd needs. */
mft_status mft_layer_norm_workspace_size(const mft_layer_norm_desc* desc, size_t* bytes);

/* dx, dweight and dbias ([D] fp32) from dy and the forward's mean and rstd.  Any
 * of the three may be NULL and is then left out; the others are written, not
 * accumulated.  dx may be dy where the strides agree; it may not be x. */
mft_status mft_layer_norm_bwd(const mft_layer_norm_desc* desc, const void* x, const float* weight, const float* mean,
                              const float* rstd, const void* dy, void* dx, float* dweight, float* dbias,
                              void* workspace, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MFT_LAYER_NORM_H */
