// C ABI of the root-mean-square norm (declared in include/mft/rms_norm.h).
#include "mft/rms_norm.h"

#include <cmath>
#include <string>

#include "capi_util.h"
#include "rms_norm_kernels.h"

namespace {

using namespace mft::capi;

mft_status check(const mft_rms_norm_desc* d, const char* who, bool none, mft::RmsNormArgs* a) {
    if (!d) return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": desc is NULL");
    if (d->N < 0 || d->D <= 0)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": x must be [N, D] with N >= 0 and D > 0");
    if (d->N > (int64_t(1) << 31) - 1 || d->D > (int64_t(1) << 30))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N must be below 2^31 and D at most 2^30");
    if (d->dtype != MFT_F32 && d->dtype != MFT_BF16)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": dtype must be MFT_F32 or MFT_BF16");
    if (d->norm != MFT_NORM_GEMMA && d->norm != MFT_NORM_AFFINE && !(none && d->norm == MFT_NORM_NONE))
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": norm must be MFT_NORM_GEMMA or MFT_NORM_AFFINE" +
                                             (none ? ", or MFT_NORM_NONE" : ""));
    if (!std::isfinite(d->eps) || d->eps < 0.f)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": eps must be finite and >= 0");
    a->N = d->N;
    a->D = d->D;
    a->eps = d->eps;
    a->norm = d->norm != MFT_NORM_NONE;
    a->one = d->norm == MFT_NORM_GEMMA ? 1.f : 0.f;
    const int64_t in[7] = {d->x_stride,  d->residual_stride, d->total_stride, d->y_stride,
                           d->dy_stride, d->dtotal_stride,   d->dx_stride};
    int64_t* out[7] = {&a->sx, &a->sr, &a->st, &a->sy, &a->sdy, &a->sdt, &a->sdx};
    for (int i = 0; i < 7; ++i) {
        if (in[i] != 0 && in[i] < d->D)
            return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": a row stride must be 0 or at least D");
        *out[i] = in[i] ? in[i] : d->D;
    }
    return MFT_OK;
}

// An output `o` that lies where the input `i` does: row by row, with one stride.
bool clash(const mft::RmsNormArgs& a, const void* o, int64_t so, const void* i, int64_t si) {
    return a.N > 1 && o && o == i && so != si;
}

mft_status forward(mft::RmsNormArgs a, const char* who, const mft_rms_norm_desc* d, const void* x, const void* residual,
                   const float* weight, void* total, void* y, hipStream_t stream) {
    const std::string w(who);
    if (d->N > 0 && (!x || !y)) return fail(MFT_ERR_INVALID_ARG, w + ": x and the output must be non-NULL");
    if (d->N > 0 && (!residual) != (!total))
        return fail(MFT_ERR_INVALID_ARG, w + ": residual and total come together");
    if (d->N > 0 && y == total) return fail(MFT_ERR_INVALID_ARG, w + ": the output may not be total");
    if (clash(a, y, a.sy, x, a.sx) || clash(a, y, a.sy, residual, a.sr) || clash(a, total, a.st, x, a.sx) ||
        clash(a, total, a.st, residual, a.sr))
        return fail(MFT_ERR_INVALID_ARG, w + ": an output in place needs its input's row stride");
    a.x = x;
    a.r = residual;
    a.w = weight;
    a.total = total;
    a.y = y;
    return hip_status(mft::launch_rms_norm_fwd(a, d->dtype == MFT_BF16, stream), who);
}

}  // namespace

extern "C" {

mft_status mft_rms_norm_fwd(const mft_rms_norm_desc* desc, const void* x, const void* residual, const float* weight,
                            void* total, void* y, float* rstd, hipStream_t stream) {
    mft::RmsNormArgs a{};
    const mft_status r = check(desc, "mft_rms_norm_fwd", false, &a);
    if (r != MFT_OK) return r;
    a.rstd = rstd;
    return forward(a, "mft_rms_norm_fwd", desc, x, residual, weight, total, y, stream);
}

mft_status mft_rms_norm_e4m3_fwd(const mft_rms_norm_desc* desc, const void* x, const void* residual,
                                 const float* weight, void* total, void* q, float* scale, hipStream_t stream) {
    const char* who = "mft_rms_norm_e4m3_fwd";
    mft::RmsNormArgs a{};
    const mft_status r = check(desc, who, true, &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && !scale) return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_e4m3_fwd: scale must be non-NULL");
    if (!a.norm && weight) return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_e4m3_fwd: no weight without a norm");
    if (desc->N > 0 && q && (q == x || q == residual))
        return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_e4m3_fwd: q may not be x or residual");
    a.scale = scale;
    return desc->N == 0 ? MFT_OK : forward(a, who, desc, x, residual, weight, total, q, stream);
}

mft_status mft_rms_norm_workspace_size(const mft_rms_norm_desc* desc, size_t* bytes) {
    mft::RmsNormArgs a{};
    const mft_status r = check(desc, "mft_rms_norm_workspace_size", false, &a);
    if (r != MFT_OK) return r;
    if (bytes) *bytes = mft::rms_norm_workspace(a.N, a.D, desc->dtype == MFT_BF16);
    return MFT_OK;
}

mft_status mft_rms_norm_bwd(const mft_rms_norm_desc* desc, const void* x, const float* weight, const float* rstd,
                            const void* dy, const void* dtotal, void* dx, float* dweight, void* workspace,
                            hipStream_t stream) {
    mft::RmsNormArgs a{};
    const mft_status r = check(desc, "mft_rms_norm_bwd", false, &a);
    if (r != MFT_OK) return r;
    if (desc->N > 0 && (!x || !rstd || !dy || !workspace))
        return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_bwd: x, rstd, dy and workspace must be non-NULL");
    if (desc->N > 0 && dx && dx == x) return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_bwd: dx may not be x");
    if (clash(a, dx, a.sdx, dy, a.sdy) || clash(a, dx, a.sdx, dtotal, a.sdt))
        return fail(MFT_ERR_INVALID_ARG, "mft_rms_norm_bwd: dx in place needs its input's row stride");
    a.x = x;
    a.w = weight;
    a.rstd_in = rstd;
    a.dy = dy;
    a.dt = dtotal;
    a.dx = dx;
    a.dw = dweight;
    return hip_status(mft::launch_rms_norm_bwd(a, desc->dtype == MFT_BF16, workspace, stream), "mft_rms_norm_bwd launch");
}

}  // extern "C"
