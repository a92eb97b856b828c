/*
 * mft/adamw.h — C ABI of one AdamW step over many tensors on gfx950.
 *
 * With t the step's number (1 for the first), every value of every tensor:
 *
 *   g  = c * grad,  c = min(1, max_norm / (norm + 1e-6)) with norm = |all grads|, or 1
 *   m  = beta1 m + (1 - beta1) g
 *   v  = beta2 v + (1 - beta2) g^2
 *   p  = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
 *
 * p is fp32: the parameter itself, or the fp32 master of a bf16 parameter, which
 * gets p rounded to nearest (stepped in bf16 alone it would drop every change
 * under 2^-9 of its value).  grad is fp32, or bf16 beside a bf16 parameter.
 *
 * States in 32 bits are m and v in fp32.  In 8 bits each 256 consecutive values of
 * a tensor (fewer at its end) share one fp32 scale for m and one for sqrt(v):
 *
 *   scale = max(max |x| / 448, 2^-126),  q = e4m3(x / scale) to nearest even
 *
 * (as mft/rms_norm.h rounds them) for x = m and x = sqrt(v), a positive sqrt(v)
 * being at least the smallest number 2^-9 (as zero it would leave m / eps of the
 * next step).  p is stepped with m and v as they are before that.
 *
 * All arithmetic is in fp32, the norm and the powers of beta in 64 bits.  A
 * gradient that is no number makes its p, m and v (in 8 bits: its 256 states)
 * NaN, and with max_norm every value whose c g is.  Results do not depend on
 * the order in which workgroups run.
 *
 * Conventions are those of mft/attention.h (status codes, mft_last_error,
 * caller-owned device memory, stream ordering, no allocation).  The step's number
 * lies in device memory and a launch counts it, so that a captured step counts
 * its replays.  `tensors` is host memory, read before the call returns.
 */
#ifndef MFT_ADAMW_H
#define MFT_ADAMW_H

#include "mft/attention.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MFT_ADAMW_GROUP 256 /* values of an 8-bit state with one scale */

typedef struct {
    int64_t n;               /* values (0: nothing is read or written)           */
    float* param;            /* fp32 parameter, or the master of param_bf16      */
    void* param_bf16;        /* bf16 parameter, or NULL                          */
    const void* grad;        /* fp32, or bf16 with param_bf16; NULL: no step     */
    void* exp_avg;           /* m: n fp32, or n e4m3 numbers                     */
    void* exp_avg_sq;        /* v: n fp32, or n e4m3 numbers of sqrt(v)          */
    float* exp_avg_scale;    /* 8 bits: ceil(n / 256) scales; else NULL          */
    float* exp_avg_sq_scale;
    double weight_decay;
} mft_adamw_tensor;

typedef struct {
    double lr;
    const float* lr_device;  /* NULL, or one fp32 in device memory instead of lr */
    double beta1, beta2;     /* in [0, 1)                                        */
    double eps;
    double max_norm;         /* gradients are clipped to it; 0: they are not     */
    int32_t state_bits;      /* 32 or 8                                          */
} mft_adamw_desc;

/* Bytes of device workspace of a step over n tensors. */
mft_status mft_adamw_workspace_size(const mft_adamw_desc* desc, int32_t n, const mft_adamw_tensor* tensors,
                                    size_t* bytes);

/* One step.  *step (device) is the number of steps before it and is counted up.
 * norm (device, one fp32) gets the gradients' norm where it is not NULL; it needs
 * max_norm.  Where no tensor has a gradient nothing is done.  No tensor's memory
 * may be another's or step's. */
mft_status mft_adamw_step(const mft_adamw_desc* desc, int32_t n, const mft_adamw_tensor* tensors, int64_t* step,
                          float* norm, void* workspace, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MFT_ADAMW_H */
