// Launchers of the linear layer's kernels (linear_gemm.hip, linear_rows.hip,
// linear.hip; called by linear_capi.cpp).
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
};
// bf16, any sizes (linear_gemm.hip).
size_t bf_gemm_workspace(const LinearProduct& g);
hipError_t launch_bf_gemm(const LinearProduct& g, hipStream_t st);
// Few rows with p_kc (linear_rows.hip); no workspace.
bool few_rows(const LinearProduct& g);
hipError_t launch_few_rows(const LinearProduct& g, bool bf16, hipStream_t st);

// dz = dy act'(z) ([N, out]; no act: dz is not written) and db[out] = the sums
// of dz's columns before rounding (null: left out).
size_t dz_workspace(int64_t N, int64_t out);
hipError_t launch_dz(const void* dy, const void* z, void* dz, float* db, int64_t N, int64_t out, int act, bool bf16,
                     float* workspace, hipStream_t st);
hipError_t launch_fill_zero(void* p, size_t bytes, hipStream_t st);  // bytes: a multiple of 2

}  // namespace mft
