// C ABI of layer norm (declared in include/mft/layer_norm.h).
#include "mft/layer_norm.h"

#include <cmath>
#include <string>

#include "capi_util.h"
#include "layer_norm_kernels.h"

namespace {

using namespace mft::capi;

mft_status check(const mft_layer_norm_desc* d, const char* who, mft::LayerNormArgs* a) {
    if (!d) return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": desc is NULL");
    if (d->N < 0 || d->D <= 0)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": x must be [N, D] with N >= 0 and D > 0");
    if (d->N > (int64_t(1) << 31) - 1 || d->D > (int64_t(1) << 30))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N must be below 2^31 and D at most 2^30");
    if (d->dtype != MFT_F32 && d->dtype != MFT_BF16)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": dtype must be MFT_F32 or MFT_BF16");
    if (!std::isfinite(d->eps) || d->eps < 0.f)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": eps must be finite and >= 0");
    a->N = d->N;
    a->D = d->D;
    a->eps = d->eps;
    const int64_t in[4] = {d->x_stride, d->y_stride, d->dy_stride, d->dx_stride};
    int64_t* out[4] = {&a->sx, &a->sy, &a->sdy, &a->sdx};
    for (int i = 0; i < 4; ++i) {
        if (in[i] != 0 && in[i] < d->D)
            return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": a row stride must be 0 or at least D");
        *out[i] = in[i] ? in[i] : d->D;
    }
    return MFT_OK;
}

}  // namespace

extern "C" {

mft_status mft_layer_norm_fwd(const mft_layer_norm_desc* desc, const void* x, const float* weight, const float* bias,
                              void* y, float* mean, float* rstd, hipStream_t stream) {
    mft::LayerNormArgs a{};
    const mft_status r = check(desc, "mft_layer_norm_fwd", &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && (!x || !y)) return fail(MFT_ERR_INVALID_ARG, "mft_layer_norm_fwd: x and y must be non-NULL");
    if (desc->N > 1 && y == x && a.sy != a.sx)
        return fail(MFT_ERR_INVALID_ARG, "mft_layer_norm_fwd: y in place needs x's row stride");
    a.x = x;
    a.w = weight;
    a.b = bias;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    return hip_status(mft::launch_layer_norm_fwd(a, desc->dtype == MFT_BF16, stream), "mft_layer_norm_fwd launch");
}

mft_status mft_layer_norm_workspace_size(const mft_layer_norm_desc* desc, size_t* bytes) {
    mft::LayerNormArgs a{};
    const mft_status r = check(desc, "mft_layer_norm_workspace_size", &a);
    if (r != MFT_OK) return r;
    if (bytes) *bytes = mft::layer_norm_workspace(a.N, a.D, desc->dtype == MFT_BF16);
    return MFT_OK;
}

mft_status mft_layer_norm_bwd(const mft_layer_norm_desc* desc, const void* x, const float* weight, const float* mean,
                              const float* rstd, const void* dy, void* dx, float* dweight, float* dbias,
                              void* workspace, hipStream_t stream) {
    mft::LayerNormArgs a{};
    const mft_status r = check(desc, "mft_layer_norm_bwd", &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && (!x || !mean || !rstd || !dy || !workspace))
        return fail(MFT_ERR_INVALID_ARG, "mft_layer_norm_bwd: x, mean, rstd, dy and workspace must be non-NULL");
    if (desc->N > 0 && dx == x) return fail(MFT_ERR_INVALID_ARG, "mft_layer_norm_bwd: dx may not be x");
    if (desc->N > 1 && dx == dy && a.sdx != a.sdy)
        return fail(MFT_ERR_INVALID_ARG, "mft_layer_norm_bwd: dx in place needs dy's row stride");
    a.x = x;
    a.w = weight;
    a.mean_in = mean;
    a.rstd_in = rstd;
    a.dy = dy;
    a.dx = dx;
    a.dw = dweight;
    a.db = dbias;
    return hip_status(mft::launch_layer_norm_bwd(a, desc->dtype == MFT_BF16, workspace, stream),
                      "mft_layer_norm_bwd launch");
}

}  // extern "C"
