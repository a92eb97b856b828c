// Launchers of the linear layer's kernels (linear_gemm.hip, linear_rows.hip,
// linear.hip; called by linear_capi.cpp) and of the gated linear layer's
// (gated_gemm.hip, gated_rows.hip, gated.hip; called by gated_linear_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mft {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU_TANH = 2, ACT_SILU = 3 };

// C[M, N] = act(sum_k P(m, k) Q(n, k) + bias[n]) + residual.  P is stored [M, K]
// (p_kc) or [K, M], Q [N, K] (q_kc) or [K, N], contiguous or, in bf16, with rows
// of ldp and ldq elements; all else contiguous.  All bf16, or all fp32, but bias
// (fp32).
struct LinearProduct {
    int64_t M, N, K;
    const void* P;
    const void* Q;
    int p_kc, q_kc;
    int64_t ldp, ldq;      // 0: contiguous
    void* C;
    // epilogue
    const float* bias;     // [N] or null
    const void* residual;  // [M, N] or null
    void* z;               // [M, N], before the activation, or null
    int act;
    float* partial;        // workspace of bf_gemm_workspace bytes
    // A second Q, stored as the first: of the gated product C = act(P Q^T) (P Q2^T), with z the first
    // sum and z2 the second, both or neither; or of a product joined along k, from `joint` on.
    const void* Q2;
    void* z2;
    int64_t joint;
};
// bf16, any sizes (linear_gemm.hip).
size_t bf_gemm_workspace(const LinearProduct& g);
hipError_t launch_bf_gemm(const LinearProduct& g, hipStream_t st);
// Few rows with p_kc (linear_rows.hip); no workspace.
bool few_rows(const LinearProduct& g);
hipError_t launch_few_rows(const LinearProduct& g, bool bf16, hipStream_t st);

// The gated product in bf16, any sizes (gated_gemm.hip): no bias, no residual.
size_t gated_gemm_workspace(const LinearProduct& g);
hipError_t launch_gated_gemm(const LinearProduct& g, hipStream_t st);
// sum_k P(m, k) Q(n, k) over k < joint plus the sum over the rest with Q2, P of rows of ldp elements: Q and Q2
// hold `joint` k each and K = 2 joint (gated_gemm.hip).
size_t joined_gemm_workspace(const LinearProduct& g);
hipError_t launch_joined_gemm(const LinearProduct& g, hipStream_t st);
// The gated product of e4m3 numbers with a scale for each row of P, Q and Q2, all with k contiguous, C in
// bf16 (gated_e4m3.hip).
size_t gated_e4m3_workspace(const LinearProduct& g);
hipError_t launch_gated_e4m3(const LinearProduct& g, const float* x_scale, const float* gate_scale,
                             const float* up_scale, hipStream_t st);
// The same and the gated product of either type for few rows (gated_rows.hip); no workspace.
hipError_t launch_gated_rows_e4m3(const LinearProduct& g, const float* x_scale, const float* gate_scale,
                                  const float* up_scale, hipStream_t st);
hipError_t launch_gated_rows(const LinearProduct& g, bool bf16, hipStream_t st);
// Two fp32 weights [rows, cols] beside one another, [rows, 2 cols], or one below the other (gated.hip).
hipError_t launch_join_weights(const float* a, const float* b, float* to, int64_t rows, int64_t cols, bool beside,
                               hipStream_t st);
// dz[N, 2 ld] = (dh up act'(gate) | dh act(gate)), either half padded with zeros from ff to ld columns
// (gated.hip).
hipError_t launch_gated_dz(const void* gate, const void* up, const void* dh, void* dz, int64_t N, int64_t ff, int64_t ld,
                           int act, bool bf16, hipStream_t st);

// dz = dy act'(z) ([N, out]; no act: dz is not written) and db[out] = the sums
// of dz's columns before rounding (null: left out).
size_t dz_workspace(int64_t N, int64_t out);
hipError_t launch_dz(const void* dy, const void* z, void* dz, float* db, int64_t N, int64_t out, int act, bool bf16,
                     float* workspace, hipStream_t st);
hipError_t launch_fill_zero(void* p, size_t bytes, hipStream_t st);  // bytes: a multiple of 2

}  // namespace mft
