// C ABI of the token log probabilities (declared in include/mft/logprobs.h).
#include "mft/logprobs.h"

#include <algorithm>
#include <string>

#include "capi_util.h"
#include "logprobs_kernels.h"

namespace {

using namespace mft::capi;

static_assert(MFT_LOGPROBS_MAX_TOP == mft::kLogprobsMaxTop, "the header's limit is the kernels'");

mft_status check(const mft_logprobs_desc* d, const char* who, mft::LogprobsArgs* a) {
    if (!d) return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": desc is NULL");
    if (d->N < 0 || d->V <= 0)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": logits must be [N, V] with N >= 0 and V > 0");
    if (d->N >= (int64_t(1) << 24) || d->V > (int64_t(1) << 30))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N must be below 2^24 and V at most 2^30");
    if (d->dtype != MFT_F32 && d->dtype != MFT_BF16)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": dtype must be MFT_F32 or MFT_BF16");
    if (d->top < 0 || d->top > std::min<int64_t>(d->V, MFT_LOGPROBS_MAX_TOP))
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": top must be 0 .. min(V, " +
                                             std::to_string(MFT_LOGPROBS_MAX_TOP) + ")");
    if ((d->ld != 0 && d->ld < d->V) || (d->grad_ld != 0 && d->grad_ld < d->V))
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": a row stride must be 0 or at least V");
    a->N = d->N;
    a->V = d->V;
    a->ld = d->ld ? d->ld : d->V;
    a->ldg = d->grad_ld ? d->grad_ld : d->V;
    a->ignore = d->ignore_index;
    a->top = d->top;
    return MFT_OK;
}

}  // namespace

extern "C" {

mft_status mft_logprobs_workspace_size(const mft_logprobs_desc* desc, size_t* bytes) {
    mft::LogprobsArgs a{};
    const mft_status r = check(desc, "mft_logprobs_workspace_size", &a);
    if (r != MFT_OK) return r;
    if (bytes) *bytes = mft::logprobs_workspace(a.N, a.V, a.top);
    return MFT_OK;
}

mft_status mft_logprobs_fwd(const mft_logprobs_desc* desc, const void* logits, const int32_t* tokens, float* logprob,
                            float* entropy, float* stats, float* top_logprobs, int32_t* top_ids, int32_t* status,
                            void* workspace, hipStream_t stream) {
    mft::LogprobsArgs a{};
    const mft_status r = check(desc, "mft_logprobs_fwd", &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && (!logits || !tokens || !logprob))
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_fwd: logits, tokens and logprob must be non-NULL");
    if (desc->N > 0 && desc->top > 0 && (!top_logprobs || !top_ids))
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_fwd: top_logprobs and top_ids must be non-NULL with top > 0");
    if (desc->N > 0 && !workspace && mft::logprobs_workspace(a.N, a.V, a.top) > 0)
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_fwd: workspace must be non-NULL");
    a.z = logits;
    a.tokens = tokens;
    a.logprob = logprob;
    a.entropy = entropy;
    a.stats = reinterpret_cast<float2*>(stats);
    a.top_logprobs = top_logprobs;
    a.top_ids = top_ids;
    a.status = status;
    return hip_status(mft::launch_logprobs_fwd(a, desc->dtype == MFT_BF16, workspace, stream),
                      "mft_logprobs_fwd launch");
}

mft_status mft_logprobs_bwd(const mft_logprobs_desc* desc, const void* logits, const int32_t* tokens,
                            const float* stats, const float* entropy, const float* grad_logprob,
                            const float* grad_entropy, void* grad_logits, hipStream_t stream) {
    mft::LogprobsArgs a{};
    const mft_status r = check(desc, "mft_logprobs_bwd", &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && (!logits || !tokens || !stats || !grad_logits))
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_bwd: logits, tokens, stats and grad_logits must be non-NULL");
    if (desc->N > 0 && grad_entropy && !entropy)
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_bwd: grad_entropy needs the forward's entropy");
    if (grad_logits == logits && a.ld != a.ldg)
        return fail(MFT_ERR_INVALID_ARG, "mft_logprobs_bwd: grad_logits in place needs the logits' row stride");
    a.z = logits;
    a.tokens = tokens;
    a.stats_in = reinterpret_cast<const float2*>(stats);
    a.entropy_in = entropy;
    a.grad_logprob = grad_logprob;
    a.grad_entropy = grad_entropy;
    a.grad = grad_logits;
    return hip_status(mft::launch_logprobs_bwd(a, desc->dtype == MFT_BF16, stream), "mft_logprobs_bwd launch");
}

}  // extern "C"
