// C ABI of the AdamW step (declared in include/mft/adamw.h).
#include "mft/adamw.h"

#include <cmath>
#include <string>

#include "adamw_kernels.h"
#include "capi_util.h"

namespace {

using namespace mft::capi;

bool at_least_zero(double x) { return std::isfinite(x) && x >= 0.0; }

mft_status check(const mft_adamw_desc* d, int32_t n, const mft_adamw_tensor* tensors, const char* who) {
    const std::string w(who);
    if (!d) return fail(MFT_ERR_INVALID_ARG, w + ": desc is NULL");
    if (n < 0 || (n > 0 && !tensors))
        return fail(MFT_ERR_INVALID_ARG, w + ": n must be >= 0 and tensors non-NULL");
    if (d->state_bits != 32 && d->state_bits != 8)
        return fail(MFT_ERR_INVALID_ARG, w + ": state_bits must be 32 or 8");
    if (!(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0))
        return fail(MFT_ERR_INVALID_ARG, w + ": beta1 and beta2 must be in [0, 1)");
    if (!at_least_zero(d->lr) || !at_least_zero(d->eps) || !at_least_zero(d->max_norm))
        return fail(MFT_ERR_INVALID_ARG, w + ": lr, eps and max_norm must be finite and >= 0");
    int64_t total = 0;
    for (int32_t i = 0; i < n; ++i) {
        const mft_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > int64_t(1) << 40 || (total += t.n) > int64_t(1) << 40)
            return fail(MFT_ERR_INVALID_ARG, w + ": a tensor's n must be >= 0, and all together at most 2^40");
        if (!at_least_zero(t.weight_decay))
            return fail(MFT_ERR_INVALID_ARG, w + ": weight_decay must be finite and >= 0");
    }
    return MFT_OK;
}

}  // namespace

extern "C" {

mft_status mft_adamw_workspace_size(const mft_adamw_desc* desc, int32_t n, const mft_adamw_tensor* tensors,
                                    size_t* bytes) {
    const mft_status r = check(desc, n, tensors, "mft_adamw_workspace_size");
    if (r != MFT_OK) return r;
    if (bytes) *bytes = mft::adamw_workspace(n);
    return MFT_OK;
}

mft_status mft_adamw_step(const mft_adamw_desc* desc, int32_t n, const mft_adamw_tensor* tensors, int64_t* step,
                          float* norm, void* workspace, hipStream_t stream) {
    const char* who = "mft_adamw_step";
    const mft_status r = check(desc, n, tensors, who);
    if (r != MFT_OK) return r;
    if (norm && desc->max_norm == 0.0)
        return fail(MFT_ERR_INVALID_ARG, "mft_adamw_step: the norm is computed with max_norm only");
    for (int32_t i = 0; i < n; ++i) {
        const mft_adamw_tensor& t = tensors[i];
        if (t.n == 0 || !t.grad) continue;
        if (!step || !workspace) return fail(MFT_ERR_INVALID_ARG, "mft_adamw_step: step and workspace must be non-NULL");
        if (!t.param || !t.exp_avg || !t.exp_avg_sq || (desc->state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
            return fail(MFT_ERR_INVALID_ARG, "mft_adamw_step: a tensor's param and states must be non-NULL");
        const void* own[6] = {t.param, t.param_bf16, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale};
        for (int j = 0; j < 6; ++j) {
            if (own[j] && (own[j] == t.grad || own[j] == step || own[j] == workspace))
                return fail(MFT_ERR_INVALID_ARG, "mft_adamw_step: a tensor's memory may not be its gradient, step or workspace");
            for (int k = 0; k < j; ++k)
                if (own[j] && own[j] == own[k])
                    return fail(MFT_ERR_INVALID_ARG, "mft_adamw_step: a tensor's param and states may not be one another");
        }
    }
    return hip_status(mft::launch_adamw(*desc, n, tensors, step, norm, workspace, stream), "mft_adamw_step launch");
}

}  // extern "C"
