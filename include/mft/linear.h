/*
 * mft/linear.h — C ABI of a linear layer with a fused epilogue on gfx950.
 *
 *   z = x W + bias,  y = act(z) + residual
 *
 * x [N, in], W [in, out] or, with w_transposed, [out, in]; y, z and residual
 * [N, out].  act is none, relu, the tanh form of GELU (z / 2 (1 + tanh(sqrt(2 /
 * pi) (z + 0.044715 z^3)))) or SiLU (z / (1 + exp(-z))).  Backward, with
 * dz = dy act'(z):
 *
 *   dx = dz W^T,  dW = x^T dz (in W's layout),  dbias = sum over rows of dz
 *
 * and the residual's gradient is dy itself.
 *
 * x, W, y, z, residual, dy, dx and dW have element type `dtype`, bias and
 * dbias are fp32.  Products accumulate in fp32, and bias, activation and
 * residual are applied to the accumulators: y and z are rounded once.  With
 * bf16, dz is rounded to bf16 for the matrix units where there is an activation
 * (half a step of each product's operand, as x and W have; dbias is summed
 * before that), dx and dW once more where they are stored.  With fp32 the
 * products are those of the LoRA layer's (csrc/gemm_f32.hip), and with one or two
 * rows fp32 sums.  Results do not depend on the order in which workgroups run.
 *
 * Conventions are those of mft/attention.h (status codes, mft_last_error,
 * caller-owned device memory, stream ordering, no allocation).  All operands
 * are contiguous.  N may be 0 (the gradients of W and bias are then zero).
 * Refused: N of 2^31 or more, in and out above 2^24, and products of more than
 * 2^23 tiles of 64 x 64.
 */
#ifndef MFT_LINEAR_H
#define MFT_LINEAR_H

#include "mft/attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { MFT_ACT_NONE = 0, MFT_ACT_RELU = 1, MFT_ACT_GELU_TANH = 2, MFT_ACT_SILU = 3 } mft_activation;

typedef struct {
    int64_t N;             /* rows of x and y                                 */
    int64_t in_dim;        /* columns of x                                    */
    int64_t out_dim;       /* columns of y                                    */
    int32_t dtype;         /* MFT_F32 or MFT_BF16                             */
    int32_t w_transposed;  /* W stored [out, in]                              */
    int32_t activation;    /* mft_activation                                  */
} mft_linear_desc;

/* Workspace bytes of the forward and backward (either may be 0). */
mft_status mft_linear_workspace_size(const mft_linear_desc* desc, size_t* fwd_bytes, size_t* bwd_bytes);

/* y, and z where it is not NULL (the backward's input with an activation; not
 * with MFT_ACT_NONE, where z would be y without the residual).  bias [out] and
 * residual may be NULL; residual may be y. */
mft_status mft_linear_fwd(const mft_linear_desc* desc, const void* x, const void* W, const float* bias,
                          const void* residual, void* y, void* z, void* workspace, hipStream_t stream);

/* dx, dW and dbias, each left out where NULL, written and not accumulated.  z
 * (the forward's) is read with an activation only.  x may be NULL without dW,
 * W without dx. */
mft_status mft_linear_bwd(const mft_linear_desc* desc, const void* x, const void* W, const void* z, const void* dy,
                          void* dx, void* dW, float* dbias, void* workspace, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MFT_LINEAR_H */
