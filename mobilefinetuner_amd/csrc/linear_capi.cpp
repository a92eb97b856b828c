// C ABI of the linear layer with a fused epilogue (declared in include/mft/linear.h).
#include "mft/linear.h"

#include <algorithm>
#include <string>

#include "capi_util.h"
#include "gemm_f32.h"
#include "linear_kernels.h"

namespace {

using namespace mft::capi;

static_assert((int)MFT_ACT_NONE == (int)mft::ACT_NONE && (int)MFT_ACT_RELU == (int)mft::ACT_RELU &&
                  (int)MFT_ACT_GELU_TANH == (int)mft::ACT_GELU_TANH && (int)MFT_ACT_SILU == (int)mft::ACT_SILU,
              "the header's activations are the kernels'");

size_t up(size_t x) { return (x + 255) & ~size_t(255); }

mft_status check(const mft_linear_desc* d, const char* who) {
    if (!d) return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": desc is NULL");
    if (d->N < 0 || d->in_dim <= 0 || d->out_dim <= 0)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": x must be [N, in] and W [in, out] with N >= 0 and "
                                                            "positive dimensions");
    if (d->N > (int64_t(1) << 31) - 1 || d->in_dim > (int64_t(1) << 24) || d->out_dim > (int64_t(1) << 24))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N must be below 2^31, in and out at most 2^24");
    if (d->dtype != MFT_F32 && d->dtype != MFT_BF16)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": dtype must be MFT_F32 or MFT_BF16");
    if (d->activation < MFT_ACT_NONE || d->activation > MFT_ACT_SILU)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": activation must be NONE, RELU, GELU_TANH or SILU");
    // a launch takes fewer than 2^32 threads: 2^23 tiles of at most 256
    const int64_t n = (d->N + 63) / 64, i = (d->in_dim + 63) / 64, o = (d->out_dim + 63) / 64;
    if (std::max(n * o, std::max(n * i, i * o)) > (int64_t(1) << 23))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N, in and out are too large together");
    return MFT_OK;
}

// The three products.  fp32: terms[0] = (A, B) with the strides of the storage.
mft::LinearProduct product_fwd(const mft_linear_desc* d) {
    mft::LinearProduct g{};
    g.M = d->N, g.N = d->out_dim, g.K = d->in_dim;
    g.p_kc = 1, g.q_kc = d->w_transposed != 0;
    g.act = d->activation;
    return g;
}
mft::LinearProduct product_dx(const mft_linear_desc* d) {
    mft::LinearProduct g{};
    g.M = d->N, g.N = d->in_dim, g.K = d->out_dim;
    g.p_kc = 1, g.q_kc = d->w_transposed == 0;
    return g;
}
mft::LinearProduct product_dw(const mft_linear_desc* d) {  // rows: W's first dimension
    mft::LinearProduct g{};
    g.M = d->w_transposed ? d->out_dim : d->in_dim;
    g.N = d->w_transposed ? d->in_dim : d->out_dim;
    g.K = d->N;
    return g;
}
mft::GemmF32 f_fwd(const mft_linear_desc* d) {
    mft::GemmF32 g{};
    g.M = d->N, g.N = g.ldc = d->out_dim;
    g.terms[0] = {nullptr, nullptr, d->in_dim, d->w_transposed ? d->in_dim : d->out_dim, d->in_dim, 0,
                  d->w_transposed != 0, 1.f};
    return g;
}
mft::GemmF32 f_dx(const mft_linear_desc* d) {
    mft::GemmF32 g{};
    g.M = d->N, g.N = g.ldc = d->in_dim;
    g.terms[0] = {nullptr, nullptr, d->out_dim, d->w_transposed ? d->in_dim : d->out_dim, d->out_dim, 0,
                  d->w_transposed == 0, 1.f};
    return g;
}
mft::GemmF32 f_dw(const mft_linear_desc* d) {
    mft::GemmF32 g{};
    g.M = d->w_transposed ? d->out_dim : d->in_dim;
    g.N = g.ldc = d->w_transposed ? d->in_dim : d->out_dim;
    g.terms[0] = {nullptr, nullptr, g.M, g.N, d->N, 1, 0, 1.f};
    return g;
}

size_t product_workspace(const mft::LinearProduct& g, const mft::GemmF32& f, bool bf) {
    return mft::few_rows(g) ? 0 : bf ? mft::bf_gemm_workspace(g) : mft::gemm_f32_workspace(f);
}

struct BwdLayout {
    size_t dz, db, gemm, total;
};
BwdLayout bwd_layout(const mft_linear_desc* d) {
    BwdLayout l{};
    const bool bf = d->dtype == MFT_BF16;
    size_t o = 0;
    l.dz = o, o += d->activation == MFT_ACT_NONE ? 0 : up((size_t)d->N * d->out_dim * (bf ? 2 : 4));
    l.db = o, o += up(mft::dz_workspace(d->N, d->out_dim));
    l.gemm = o;
    o += std::max(product_workspace(product_dx(d), f_dx(d), bf), product_workspace(product_dw(d), f_dw(d), bf));
    l.total = o;
    return l;
}

hipError_t run_f32(mft::GemmF32 g, const void* A, const void* B, void* C, char* ws, hipStream_t st) {
    g.terms[0].A = static_cast<const float*>(A);
    g.terms[0].B = static_cast<const float*>(B);
    g.C = static_cast<float*>(C);
    g.partial = reinterpret_cast<float*>(ws);
    return mft::launch_gemm_f32(g, st);
}
// A bf16 product, or one of few rows of either type.
hipError_t run(mft::LinearProduct g, bool bf, const void* P, const void* Q, void* C, char* ws, hipStream_t st) {
    g.P = P;
    g.Q = Q;
    g.C = C;
    g.partial = reinterpret_cast<float*>(ws);
    return mft::few_rows(g) ? mft::launch_few_rows(g, bf, st) : mft::launch_bf_gemm(g, st);
}
}  // namespace

extern "C" {

mft_status mft_linear_workspace_size(const mft_linear_desc* desc, size_t* fwd_bytes, size_t* bwd_bytes) {
    const mft_status r = check(desc, "mft_linear_workspace_size");
    if (r != MFT_OK) return r;
    const bool empty = desc->N == 0;
    if (fwd_bytes)
        *fwd_bytes = empty ? 0 : product_workspace(product_fwd(desc), f_fwd(desc), desc->dtype == MFT_BF16);
    if (bwd_bytes) *bwd_bytes = empty ? 0 : bwd_layout(desc).total;
    return MFT_OK;
}

mft_status mft_linear_fwd(const mft_linear_desc* desc, const void* x, const void* W, const float* bias,
                          const void* residual, void* y, void* z, void* workspace, hipStream_t stream) {
    const char* who = "mft_linear_fwd";
    const mft_status r = check(desc, who);
    if (r != MFT_OK) return r;
    if (desc->N == 0) return MFT_OK;
    if (!x || !W || !y) return fail(MFT_ERR_INVALID_ARG, "mft_linear_fwd: x, W and y must be non-NULL");
    if (z && desc->activation == MFT_ACT_NONE)
        return fail(MFT_ERR_INVALID_ARG, "mft_linear_fwd: z is kept with an activation only");
    if (y == x || y == W || (z && (z == y || z == x || z == W || z == residual)))
        return fail(MFT_ERR_INVALID_ARG, "mft_linear_fwd: y may not be x or W, nor z another operand");
    char* ws = static_cast<char*>(workspace);
    const bool bf = desc->dtype == MFT_BF16;
    mft::LinearProduct q = product_fwd(desc);
    if (!ws && product_workspace(q, f_fwd(desc), bf) > 0)
        return fail(MFT_ERR_INVALID_ARG, "mft_linear_fwd: workspace must be non-NULL");
    if (bf || mft::few_rows(q)) {
        q.bias = bias;
        q.residual = residual;
        q.z = z;
        return hip_status(run(q, bf, x, W, y, ws, stream), "mft_linear_fwd launch");
    }
    mft::GemmF32 g = f_fwd(desc);
    g.bias = bias;
    g.act = desc->activation;
    g.residual = static_cast<const float*>(residual);
    g.z = static_cast<float*>(z);
    return hip_status(run_f32(g, x, W, y, ws, stream), "mft_linear_fwd launch");
}

mft_status mft_linear_bwd(const mft_linear_desc* desc, const void* x, const void* W, const void* z, const void* dy,
                          void* dx, void* dW, float* dbias, void* workspace, hipStream_t stream) {
    const char* who = "mft_linear_bwd";
    const mft_status r = check(desc, who);
    if (r != MFT_OK) return r;
    const bool bf = desc->dtype == MFT_BF16, act = desc->activation != MFT_ACT_NONE;
    if (desc->N == 0) {
        hipError_t e = hipSuccess;
        if (dW) e = mft::launch_fill_zero(dW, (size_t)desc->in_dim * desc->out_dim * (bf ? 2 : 4), stream);
        if (e == hipSuccess && dbias) e = mft::launch_fill_zero(dbias, (size_t)desc->out_dim * 4, stream);
        return hip_status(e, "mft_linear_bwd launch");
    }
    if (!dx && !dW && !dbias) return MFT_OK;
    if (!dy || !workspace || (dW && !x) || (dx && !W) || (act && !z))
        return fail(MFT_ERR_INVALID_ARG, "mft_linear_bwd: dy, workspace, x (for dW), W (for dx) and z (with an "
                                         "activation) must be non-NULL");
    if ((dx && (dx == dy || dx == x || dx == W || dx == z)) || (dW && (dW == W || dW == x || dW == dy || dW == z)))
        return fail(MFT_ERR_INVALID_ARG, "mft_linear_bwd: dx and dW may not be operands");
    if (dx && dx == dW) return fail(MFT_ERR_INVALID_ARG, "mft_linear_bwd: dx and dW may not be one tensor");
    const BwdLayout l = bwd_layout(desc);
    char* ws = static_cast<char*>(workspace);
    const void* dz = act ? ws + l.dz : dy;
    hipError_t e = mft::launch_dz(dy, z, dx || dW ? ws + l.dz : nullptr, dbias, desc->N, desc->out_dim,
                                  desc->activation, bf, reinterpret_cast<float*>(ws + l.db), stream);
    if (e == hipSuccess && dx)
        e = bf || mft::few_rows(product_dx(desc)) ? run(product_dx(desc), bf, dz, W, dx, ws + l.gemm, stream)
                                                  : run_f32(f_dx(desc), dz, W, dx, ws + l.gemm, stream);
    if (e == hipSuccess && dW) {
        const void* rows = desc->w_transposed ? dz : x;
        const void* cols = desc->w_transposed ? x : dz;
        e = bf ? run(product_dw(desc), bf, rows, cols, dW, ws + l.gemm, stream)
               : run_f32(f_dw(desc), rows, cols, dW, ws + l.gemm, stream);
    }
    return hip_status(e, "mft_linear_bwd launch");
}

}  // extern "C"
