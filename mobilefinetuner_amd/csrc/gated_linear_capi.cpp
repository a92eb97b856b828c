// C ABI of the gated linear layer (declared in include/mft/gated_linear.h).
#include "mft/gated_linear.h"

#include <algorithm>
#include <initializer_list>
#include <string>

#include "capi_util.h"
#include "gemm_f32.h"
#include "linear_kernels.h"

namespace {

using namespace mft::capi;

size_t up(size_t x) { return (x + 255) & ~size_t(255); }

mft_status check(const mft_gated_linear_desc* d, const char* who, bool e4m3 = false) {
    if (!d) return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": desc is NULL");
    if (d->N < 0 || d->in_dim <= 0 || d->ff_dim <= 0)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": x must be [N, in] and the weights [in, ff] with N >= 0 "
                                                            "and positive dimensions");
    if (d->N > (int64_t(1) << 31) - 1 || d->in_dim > (int64_t(1) << 24) || d->ff_dim > (int64_t(1) << 24))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N must be below 2^31, in and ff at most 2^24");
    if (e4m3 ? d->dtype != MFT_BF16 : d->dtype != MFT_F32 && d->dtype != MFT_BF16)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + (e4m3 ? ": dtype (of h) must be MFT_BF16"
                                                                  : ": dtype must be MFT_F32 or MFT_BF16"));
    if (e4m3 && !d->w_transposed)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": weights in 8 bits are stored [ff, in]");
    if (d->activation <= MFT_ACT_NONE || d->activation > MFT_ACT_SILU)
        return fail(MFT_ERR_INVALID_ARG, std::string(who) + ": activation must be RELU, GELU_TANH or SILU");
    // a launch takes fewer than 2^32 threads: 2^23 tiles of at most 256
    const int64_t n = (d->N + 63) / 64, i = (d->in_dim + 63) / 64, f = (d->ff_dim + 63) / 64;
    if (std::max(n * f, std::max(n * i, i * f)) > (int64_t(1) << 23))
        return fail(MFT_ERR_UNSUPPORTED, std::string(who) + ": N, in and ff are too large together");
    return MFT_OK;
}

bool is_bf(const mft_gated_linear_desc* d) { return d->dtype == MFT_BF16; }
// Columns of either half of dz: whole vectors in bf16.
int64_t half_ld(const mft_gated_linear_desc* d) { return is_bf(d) ? (d->ff_dim + 7) / 8 * 8 : d->ff_dim; }

mft::LinearProduct product_fwd(const mft_gated_linear_desc* d) {
    mft::LinearProduct g{};
    g.M = d->N, g.N = d->ff_dim, g.K = d->in_dim;
    g.p_kc = 1, g.q_kc = d->w_transposed != 0;
    g.act = d->activation;
    return g;
}
mft::LinearProduct product_dx(const mft_gated_linear_desc* d) {  // along both halves of dz
    mft::LinearProduct g{};
    g.M = d->N, g.N = d->in_dim, g.K = g.ldp = 2 * half_ld(d);
    g.joint = d->ff_dim;
    g.p_kc = 1, g.q_kc = d->w_transposed == 0;
    return g;
}
mft::LinearProduct product_dw(const mft_gated_linear_desc* d) {  // rows: the weight's first dimension
    mft::LinearProduct g{};
    g.M = d->w_transposed ? d->ff_dim : d->in_dim;
    g.N = d->w_transposed ? d->in_dim : d->ff_dim;
    g.K = d->N;
    (d->w_transposed ? g.ldp : g.ldq) = 2 * half_ld(d);
    return g;
}
mft::GemmF32 f_fwd(const mft_gated_linear_desc* d) {
    mft::GemmF32 g{};
    g.M = d->N, g.N = g.ldc = d->ff_dim;
    g.terms[0] = {nullptr, nullptr, d->in_dim, d->w_transposed ? d->in_dim : d->ff_dim, d->in_dim, 0,
                  d->w_transposed != 0, 1.f};
    return g;
}
// fp32: dx along both halves of dz as one product, with the weights laid beside one
// another, or as two, the second added to the first: the copy costs less than the second
// launch's start and end up to about 4 M weights, and more beyond (the limit stays clear of that).  dx alone, copied and
// added, us, weights [ff, in]: 509 x 640 -> 2048 45 and 51, 2048 rows 95 and 109; 509 x 1024 ->
// 2048 50 and 62; 509 x 896 -> 4864 86 and 90; 128 x 1152 -> 6912 66 and 55, 2048 rows 602 and 587.
constexpr int64_t kJoinedWeight = int64_t(1) << 21;
bool f_joins(const mft_gated_linear_desc* d) { return d->in_dim * d->ff_dim <= kJoinedWeight; }
mft::GemmF32 f_dx(const mft_gated_linear_desc* d) {
    mft::GemmF32 g{};
    const int64_t k = d->ff_dim * (f_joins(d) ? 2 : 1);
    g.M = d->N, g.N = g.ldc = d->in_dim;
    g.terms[0] = {nullptr, nullptr, 2 * d->ff_dim, d->w_transposed ? d->in_dim : k, k, 0, d->w_transposed == 0, 1.f};
    return g;
}
mft::GemmF32 f_dw(const mft_gated_linear_desc* d, bool both) {
    mft::GemmF32 g{};
    g.M = d->w_transposed ? d->ff_dim * (both ? 2 : 1) : d->in_dim;
    g.N = g.ldc = d->w_transposed ? d->in_dim : d->ff_dim;
    g.terms[0] = {nullptr, nullptr, d->w_transposed ? 2 * d->ff_dim : d->in_dim,
                  d->w_transposed ? d->in_dim : 2 * d->ff_dim, d->N, 1, 0, 1.f};
    return g;
}

struct FwdLayout {
    size_t gate, gemm, total;  // fp32: gate where the caller keeps none
};
FwdLayout fwd_layout(const mft_gated_linear_desc* d) {
    FwdLayout l{};
    const mft::LinearProduct g = product_fwd(d);
    if (mft::few_rows(g)) return l;
    if (is_bf(d)) {
        l.total = mft::gated_gemm_workspace(g);
        return l;
    }
    l.gemm = up((size_t)d->N * d->ff_dim * 4);
    l.total = l.gemm + mft::gemm_f32_workspace(f_fwd(d));
    return l;
}
// fp32: one product for both weights' gradients stored [ff, in], each to memory of its own.  Twice the tiles at
// once: 509 x 640 -> 2048 31 us against 45 (bf16 at 4096 x 1152 -> 6912, whose single products fill the GPU: 341 us
// of a backward against 338).
bool may_be_both(const mft_gated_linear_desc* d) { return !is_bf(d) && d->w_transposed; }

struct BwdLayout {
    size_t dz, join, gemm, total;
};
BwdLayout bwd_layout(const mft_gated_linear_desc* d) {
    BwdLayout l{};
    size_t o = up((size_t)d->N * 2 * half_ld(d) * (is_bf(d) ? 2 : 4));
    l.join = o, o += !is_bf(d) && f_joins(d) ? up((size_t)2 * d->in_dim * d->ff_dim * 4) : 0;
    l.gemm = o;
    l.total = o + (is_bf(d) ? std::max(mft::joined_gemm_workspace(product_dx(d)), mft::bf_gemm_workspace(product_dw(d)))
                            : std::max({mft::gemm_f32_workspace(f_dx(d)), mft::gemm_f32_workspace(f_dw(d, false)),
                                        may_be_both(d) ? mft::gemm_f32_workspace(f_dw(d, true)) : 0}));
    return l;
}

bool any_is(const void* p, std::initializer_list<const void*> of) {
    return p && std::find(of.begin(), of.end(), p) != of.end();
}

}  // namespace

extern "C" {

mft_status mft_gated_linear_workspace_size(const mft_gated_linear_desc* desc, size_t* fwd_bytes, size_t* bwd_bytes) {
    const mft_status r = check(desc, "mft_gated_linear_workspace_size");
    if (r != MFT_OK) return r;
    const bool empty = desc->N == 0;
    if (fwd_bytes) *fwd_bytes = empty ? 0 : fwd_layout(desc).total;
    if (bwd_bytes) *bwd_bytes = empty ? 0 : bwd_layout(desc).total;
    return MFT_OK;
}

mft_status mft_gated_linear_fwd(const mft_gated_linear_desc* desc, const void* x, const void* W_gate, const void* W_up,
                                void* h, void* gate, void* up, void* workspace, hipStream_t stream) {
    const char* who = "mft_gated_linear_fwd";
    const mft_status r = check(desc, who);
    if (r != MFT_OK) return r;
    if (desc->N == 0) return MFT_OK;
    if (!x || !W_gate || !W_up || !h)
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_fwd: x, W_gate, W_up and h must be non-NULL");
    if (!gate != !up) return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_fwd: gate and up are kept together");
    if (any_is(h, {x, W_gate, W_up, gate, up}) || any_is(gate, {x, W_gate, W_up, up}) || any_is(up, {x, W_gate, W_up}))
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_fwd: h, gate and up may not be one another or operands");
    const FwdLayout l = fwd_layout(desc);
    char* ws = static_cast<char*>(workspace);
    if (!ws && l.total > 0) return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_fwd: workspace must be non-NULL");
    mft::LinearProduct q = product_fwd(desc);
    q.P = x;
    q.Q = W_gate;
    q.Q2 = W_up;
    q.C = h;
    q.z = gate;
    q.z2 = up;
    q.partial = reinterpret_cast<float*>(ws);
    if (mft::few_rows(q)) return hip_status(mft::launch_gated_rows(q, is_bf(desc), stream), "mft_gated_linear_fwd launch");
    if (is_bf(desc)) return hip_status(mft::launch_gated_gemm(q, stream), "mft_gated_linear_fwd launch");
    mft::GemmF32 g = f_fwd(desc);
    float* first = gate ? static_cast<float*>(gate) : reinterpret_cast<float*>(ws + l.gate);
    g.partial = reinterpret_cast<float*>(ws + l.gemm);
    g.terms[0].A = static_cast<const float*>(x);
    g.terms[0].B = static_cast<const float*>(W_gate);
    g.C = first;
    hipError_t e = mft::launch_gemm_f32(g, stream);
    g.terms[0].B = static_cast<const float*>(W_up);
    g.C = static_cast<float*>(h);
    g.z = static_cast<float*>(up);
    g.gate = first;
    g.act = desc->activation;
    if (e == hipSuccess) e = mft::launch_gemm_f32(g, stream);
    return hip_status(e, "mft_gated_linear_fwd launch");
}

mft_status mft_gated_linear_bwd(const mft_gated_linear_desc* desc, const void* x, const void* W_gate, const void* W_up,
                                const void* gate, const void* up, const void* dh, void* dx, void* dW_gate, void* dW_up,
                                void* workspace, hipStream_t stream) {
    const char* who = "mft_gated_linear_bwd";
    const mft_status r = check(desc, who);
    if (r != MFT_OK) return r;
    const bool bf = is_bf(desc);
    void* const dW[2] = {dW_gate, dW_up};
    hipError_t e = hipSuccess;
    if (desc->N == 0) {
        for (void* w : dW)
            if (w && e == hipSuccess) e = mft::launch_fill_zero(w, (size_t)desc->in_dim * desc->ff_dim * (bf ? 2 : 4), stream);
        return hip_status(e, "mft_gated_linear_bwd launch");
    }
    if (!dx && !dW_gate && !dW_up) return MFT_OK;
    if (!gate || !up || !dh || !workspace || ((dW_gate || dW_up) && !x) || (dx && (!W_gate || !W_up)))
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_bwd: gate, up, dh, workspace, x (for the weights' gradients) "
                                         "and the weights (for dx) must be non-NULL");
    for (void* o : {dx, dW_gate, dW_up})
        if (any_is(o, {x, W_gate, W_up, gate, up, dh}))
            return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_bwd: a gradient may not be an operand");
    if (any_is(dx, {dW_gate, dW_up}) || any_is(dW_gate, {dW_up}))
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_bwd: the gradients may not be one another");
    const BwdLayout l = bwd_layout(desc);
    char* ws = static_cast<char*>(workspace);
    const int64_t ld = half_ld(desc);
    float* sums = reinterpret_cast<float*>(ws + l.gemm);
    const char* dz[2] = {ws + l.dz, ws + l.dz + ld * (bf ? 2 : 4)};
    e = mft::launch_gated_dz(gate, up, dh, ws + l.dz, desc->N, desc->ff_dim, ld, desc->activation, bf, stream);
    if (e == hipSuccess && dx) {
        if (bf) {
            mft::LinearProduct g = product_dx(desc);
            g.P = dz[0], g.Q = W_gate, g.Q2 = W_up, g.C = dx, g.partial = sums;
            e = mft::launch_joined_gemm(g, stream);
        } else {
            mft::GemmF32 g = f_dx(desc);
            const bool joins = f_joins(desc), kc = desc->w_transposed == 0;
            float* joined = reinterpret_cast<float*>(ws + l.join);
            const float* W[2] = {static_cast<const float*>(W_gate), static_cast<const float*>(W_up)};
            if (joins)
                e = mft::launch_join_weights(W[0], W[1], joined, kc ? desc->in_dim : desc->ff_dim,
                                             kc ? desc->ff_dim : desc->in_dim, kc, stream);
            g.C = static_cast<float*>(dx), g.partial = sums;
            for (int i = 0; i < (joins ? 1 : 2) && e == hipSuccess; ++i) {
                g.terms[0].A = reinterpret_cast<const float*>(dz[i]);
                g.terms[0].B = joins ? joined : W[i];
                g.add = i;
                e = mft::launch_gemm_f32(g, stream);
            }
        }
    }
    const bool both = may_be_both(desc) && dW_gate && dW_up;
    for (int i = 0; i < (both ? 1 : 2) && e == hipSuccess; ++i) {
        if (!dW[i]) continue;
        const void* rows = desc->w_transposed ? dz[i] : x;
        const void* cols = desc->w_transposed ? x : dz[i];
        if (bf) {
            mft::LinearProduct g = product_dw(desc);
            g.P = rows, g.Q = cols, g.C = dW[i], g.partial = sums;
            e = mft::launch_bf_gemm(g, stream);
        } else {
            mft::GemmF32 g = f_dw(desc, both);
            g.terms[0].A = static_cast<const float*>(rows), g.terms[0].B = static_cast<const float*>(cols);
            g.C = static_cast<float*>(dW[i]), g.partial = sums;
            if (both) g.C2 = static_cast<float*>(dW_up), g.rows = desc->ff_dim;
            e = mft::launch_gemm_f32(g, stream);
        }
    }
    return hip_status(e, "mft_gated_linear_bwd launch");
}

mft_status mft_gated_linear_e4m3_workspace_size(const mft_gated_linear_desc* desc, size_t* bytes) {
    const mft_status r = check(desc, "mft_gated_linear_e4m3_workspace_size", true);
    if (r != MFT_OK) return r;
    const mft::LinearProduct g = product_fwd(desc);
    if (bytes) *bytes = desc->N == 0 || mft::few_rows(g) ? 0 : mft::gated_e4m3_workspace(g);
    return MFT_OK;
}

mft_status mft_gated_linear_e4m3_fwd(const mft_gated_linear_desc* desc, const void* x, const float* x_scale,
                                     const void* W_gate, const float* gate_scale, const void* W_up,
                                     const float* up_scale, void* h, void* workspace, hipStream_t stream) {
    const char* who = "mft_gated_linear_e4m3_fwd";
    const mft_status r = check(desc, who, true);
    if (r != MFT_OK) return r;
    if (desc->N == 0) return MFT_OK;
    if (!x || !x_scale || !W_gate || !gate_scale || !W_up || !up_scale || !h)
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_e4m3_fwd: operands, scales and h must be non-NULL");
    if (any_is(h, {x, x_scale, W_gate, gate_scale, W_up, up_scale}))
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_e4m3_fwd: h may not be an operand");
    mft::LinearProduct g = product_fwd(desc);
    g.P = x;
    g.Q = W_gate;
    g.Q2 = W_up;
    g.C = h;
    g.partial = static_cast<float*>(workspace);
    if (mft::few_rows(g))
        return hip_status(mft::launch_gated_rows_e4m3(g, x_scale, gate_scale, up_scale, stream),
                          "mft_gated_linear_e4m3_fwd launch");
    if (!workspace && mft::gated_e4m3_workspace(g) > 0)
        return fail(MFT_ERR_INVALID_ARG, "mft_gated_linear_e4m3_fwd: workspace must be non-NULL");
    return hip_status(mft::launch_gated_e4m3(g, x_scale, gate_scale, up_scale, stream), "mft_gated_linear_e4m3_fwd launch");
}

}  // extern "C"
