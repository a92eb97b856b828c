// The element-wise passes of the gated linear layer's backward (C ABI in
// include/mft/gated_linear.h): the gradients of both sums, and small weights laid
// beside one another.  Bound by memory.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.h"
#include "linear_act.h"
#include "row_util.h"

namespace mft {
namespace {

// A thread takes V columns of every gridDim.y-th row.  The gradients of both sums lie
// beside one another for dx, a product along both, and are stored in T, as the
// matrix units take them: in bf16 a rounding of half a step before the products, as
// the linear layer's dz has it (its comment has what more would cost).
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gated_dz(const T* gate, const T* up, const T* dh, T* dz, int64_t N, int64_t ff,
                                                int64_t ld) {
    constexpr int V = 16 / (int)sizeof(T);
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= ld) return;
#pragma unroll 2
    for (int64_t n = blockIdx.y; n < N; n += gridDim.y) {
        float g[V], u[V], d[V];
        load_part<T, V>(gate + n * ff, c, ff, g);
        load_part<T, V>(up + n * ff, c, ff, u);
        load_part<T, V>(dh + n * ff, c, ff, d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            u[e] *= d[e] * act_grad<ACT>(g[e]);
            d[e] *= act_value<ACT>(g[e]);
        }
        if (c + V > ff)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e >= ff) u[e] = d[e] = 0.f;
        store_part<T, V>(dz + n * 2 * ld, c, ld, u);
        store_part<T, V>(dz + n * 2 * ld + ld, c, ld, d);
    }
}

template <typename T>
void dz_t(const void* gate, const void* up, const void* dh, void* dz, int64_t N, int64_t ff, int64_t ld, int act,
          hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const int64_t cols = (ld + 256 * V - 1) / (256 * V);
    // about sixteen workgroups to a CU
    const dim3 grid((unsigned)cols, (unsigned)std::min<int64_t>({N, std::max<int64_t>(1, 16 * device_cus() / cols), 65535}));
#define MFT_GATED_DZ(ACT)                                                                                              \
    hipLaunchKernelGGL((gated_dz<T, ACT>), grid, dim3(256), 0, st, (const T*)gate, (const T*)up, (const T*)dh, (T*)dz, \
                       N, ff, ld)
    if (act == ACT_RELU) MFT_GATED_DZ(ACT_RELU);
    else if (act == ACT_SILU) MFT_GATED_DZ(ACT_SILU);
    else MFT_GATED_DZ(ACT_GELU_TANH);
#undef MFT_GATED_DZ
}

// Two weights [rows, cols] beside one another, [rows, 2 cols], or one below the other.
__global__ __launch_bounds__(256) void join_weights(const float* a, const float* b, float* to, int64_t rows, int64_t cols,
                                                    int beside) {
    const int64_t chunks = (cols + 3) / 4, n = rows * chunks, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += step) {
        const int64_t j = i < n ? i : i - n, r = j / chunks, c = (j - r * chunks) * 4;
        float v[4];
        load_part<float, 4>((i < n ? a : b) + r * cols, c, cols, v);
        float* row = beside ? to + (2 * r + (i >= n)) * cols : to + (r + (i < n ? 0 : rows)) * cols;
        store_part<float, 4>(row, c, cols, v);
    }
}

}  // namespace

hipError_t launch_join_weights(const float* a, const float* b, float* to, int64_t rows, int64_t cols, bool beside,
                               hipStream_t st) {
    const int64_t n = 2 * rows * ((cols + 3) / 4);
    hipLaunchKernelGGL(join_weights, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 16 * device_cus())), dim3(256), 0, st,
                       a, b, to, rows, cols, (int)beside);
    return hipGetLastError();
}

hipError_t launch_gated_dz(const void* gate, const void* up, const void* dh, void* dz, int64_t N, int64_t ff, int64_t ld,
                           int act, bool is_bf16, hipStream_t st) {
    if (N <= 0 || ff <= 0) return hipSuccess;
    if (is_bf16) dz_t<bf16>(gate, up, dh, dz, N, ff, ld, act, st);
    else dz_t<float>(gate, up, dh, dz, N, ff, ld, act, st);
    return hipGetLastError();
}

}  // namespace mft
