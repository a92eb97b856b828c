/*
 * mft/logprobs.h — C ABI of the log probabilities of given tokens on gfx950.
 *
 * Row n of the logits [N, V] gives the distribution p = softmax(z) that scores
 * tokens[n] (no shift: the caller pairs rows and tokens):
 *
 *   logprob[n] = log p(tokens[n]),  entropy[n] = - sum_j p_j log p_j
 *   top_logprobs[n, i], top_ids[n, i]: the `top` largest log probabilities and
 *       their indices, in falling order, equal ones in the order of their indices
 *
 * and, backward,
 *
 *   dz_j = grad_logprob[n] (1[j = tokens[n]] - p_j) - grad_entropy[n] p_j (log p_j + entropy[n])
 *
 * The logits and their gradient have element type `dtype`; all else is fp32,
 * as are the sums.  A probability of zero (a logit of -inf, or one so far below
 * the row's largest that exp is 0, as a mask of the type's lowest value is) adds
 * nothing to the entropy or its gradient.  A row that holds a NaN or +inf, or
 * nothing but -inf, has NaN log probabilities and entropy; NaN logits are never
 * alternatives (top_ids is -1 where a row has fewer numbers than `top`).
 *
 * Rows whose token is ignore_index are not read: logprob, entropy and stats are
 * 0, top_logprobs -inf, top_ids -1, and the gradient is 0.  A token outside
 * [0, V) that is not ignore_index sets *status to 1 and has logprob NaN and a
 * gradient of 0; its row's entropy and alternatives are computed.
 *
 * The alternatives are those of the given logits, so there is no form that
 * computes logits of its own: its roundings would decide between near ones.
 *
 * Conventions are those of mft/attention.h (status codes, mft_last_error,
 * caller-owned device memory, stream ordering, no allocation), but rows may
 * start at any element.  N may be 0; it is below 2^24, and V at most 2^30.
 */
#ifndef MFT_LOGPROBS_H
#define MFT_LOGPROBS_H

#include "mft/attention.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MFT_LOGPROBS_MAX_TOP 64

typedef struct {
    int64_t N;             /* rows                                            */
    int64_t V;             /* vocabulary                                      */
    int64_t ld;            /* elements between rows of the logits; 0 = V      */
    int64_t grad_ld;       /* the same of grad_logits                         */
    int32_t dtype;         /* mft_dtype of logits and grad_logits             */
    int32_t ignore_index;
    int32_t top;           /* 0 .. min(V, MFT_LOGPROBS_MAX_TOP)               */
} mft_logprobs_desc;

/* Bytes of device workspace of mft_logprobs_fwd (may be 0). */
mft_status mft_logprobs_workspace_size(const mft_logprobs_desc* desc, size_t* bytes);

/* tokens [N] int32; logprob [N], entropy [N]; stats [N, 2] (the row's largest
 * logit, and the log of the sum of exp(z - it)) for the backward; top_logprobs
 * [N, top] and top_ids [N, top] int32, not NULL with top > 0.  entropy, stats and
 * status ([1], written only by a token out of range) may be NULL. */
mft_status mft_logprobs_fwd(const mft_logprobs_desc* desc, const void* logits, const int32_t* tokens, float* logprob,
                            float* entropy, float* stats, float* top_logprobs, int32_t* top_ids, int32_t* status,
                            void* workspace, hipStream_t stream);

/* grad_logits [N, V] from the forward's stats and entropy.  grad_logprob and
 * grad_entropy ([N]) may be NULL (0); entropy may be NULL without grad_entropy.
 * grad_logits may be the logits where the strides agree. */
mft_status mft_logprobs_bwd(const mft_logprobs_desc* desc, const void* logits, const int32_t* tokens,
                            const float* stats, const float* entropy, const float* grad_logprob,
                            const float* grad_entropy, void* grad_logits, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MFT_LOGPROBS_H */
