// Element-wise passes of the linear layer's backward (C ABI in
// include/mft/linear.h): dz = dy act'(z) and the bias gradient, its column sums.
// Bound by memory.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.h"
#include "linear_act.h"
#include "row_util.h"

namespace mft {
namespace {

// A workgroup takes 64 threads' columns (V each) and every strips-th row group:
// its four waves the rows in turn.  dz is stored in T, as the matrix units take it
// (the column sums are of the fp32 values).  In bf16 that is a rounding of half a
// step before both products: 8192 x 1024 -> 4096 with GELU, dx and dW are off by
// 2.35e-3 of their norm, 1.66e-3 without it by their own rounding.  Kept as the sum of
// two bf16 numbers dz would have the products run over twice their K: dx 63 -> 116 us
// and dW 77 -> 130 of 180.  fp32 tensors keep dz in fp32.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void dz_kernel(const T* dy, const T* z, T* dz, float* part, int64_t N, int64_t out) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float s[4][64 * V];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c0 = ((int64_t)blockIdx.x * 64 + lane) * V;
    float sum[V] = {};
    if (c0 < out)
#pragma unroll 4
        for (int64_t n = (int64_t)blockIdx.y * 4 + w; n < N; n += (int64_t)gridDim.y * 4) {
            float g[V], q[V];
            load_part<T, V>(dy + n * out, c0, out, g);
            if constexpr (ACT != ACT_NONE) {
                load_part<T, V>(z + n * out, c0, out, q);
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] *= act_grad<ACT>(q[e]);
                if (dz) store_part<T, V>(dz + n * out, c0, out, g);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += g[e];
        }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < V; ++e) s[w][lane * V + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * V; i += 256) {
        const int64_t c = (int64_t)blockIdx.x * 64 * V + i;
        if (c < out) part[(int64_t)blockIdx.y * out + c] = (s[0][i] + s[1][i]) + (s[2][i] + s[3][i]);
    }
}

// db[c] = the strips' sums, 64 columns to a workgroup, 16 waves in turn.
__global__ __launch_bounds__(1024) void db_kernel(const float* part, float* db, int64_t out, int64_t strips) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float v = 0.f;
    if (c < out)
#pragma unroll 8
        for (int64_t i = w; i < strips; i += 16) v += part[i * out + c];
    s[w][lane] = v;
    __syncthreads();
    if (w != 0 || c >= out) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += s[i][lane];
    db[c] = v;
}

// db[c] = the sums of dy's columns, in one launch: 32 columns to a workgroup, whose
// 32 rows of threads take dy's rows in turn.  1021 x 2304 in fp32 5 us for 9 as
// strips and their sums.
template <typename T>
__global__ __launch_bounds__(1024) void column_sums(const T* dy, float* db, int64_t N, int64_t out) {
    __shared__ float s[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < out)
#pragma unroll 8
        for (int64_t n = y; n < N; n += 32) v += (float)dy[n * out + c];
    s[y][x] = v;
    __syncthreads();
    if (y != 0 || c >= out) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][x];
    db[c] = v;
}

__global__ __launch_bounds__(256) void fill_zero_kernel(uint16_t* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

constexpr int64_t kFewRows = 2048;  // that 32 rows of threads add in a few rounds of loads

// Row strips: about four workgroups a CU, each of at least 32 rows.
int64_t dz_strips(int64_t N, int64_t out) {
    const int64_t cols = (out + 511) / 512;
    return std::max<int64_t>(1, std::min<int64_t>({N / 32, 4 * device_cus() / cols, 65535}));
}

template <typename T>
void launch_dz_t(const void* dy, const void* z, void* dz, float* part, int64_t N, int64_t out, int act, int64_t strips,
                 hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const dim3 grid((unsigned)((out + 64 * V - 1) / (64 * V)), (unsigned)strips);
#define MFT_DZ(ACT) \
    hipLaunchKernelGGL((dz_kernel<T, ACT>), grid, dim3(256), 0, st, (const T*)dy, (const T*)z, (T*)dz, part, N, out)
    switch (act) {
        case ACT_RELU: MFT_DZ(ACT_RELU); break;
        case ACT_GELU_TANH: MFT_DZ(ACT_GELU_TANH); break;
        case ACT_SILU: MFT_DZ(ACT_SILU); break;
        default: MFT_DZ(ACT_NONE); break;
    }
#undef MFT_DZ
}

}  // namespace

size_t dz_workspace(int64_t N, int64_t out) { return (size_t)dz_strips(N, out) * out * 4; }

hipError_t launch_dz(const void* dy, const void* z, void* dz, float* db, int64_t N, int64_t out, int act, bool is_bf16,
                     float* workspace, hipStream_t st) {
    if (act == ACT_NONE && !db) return hipSuccess;
    if (act == ACT_NONE && N <= kFewRows) {
        const dim3 grid((unsigned)((out + 31) / 32));
        if (is_bf16) hipLaunchKernelGGL((column_sums<bf16>), grid, dim3(1024), 0, st, (const bf16*)dy, db, N, out);
        else hipLaunchKernelGGL((column_sums<float>), grid, dim3(1024), 0, st, (const float*)dy, db, N, out);
        return hipGetLastError();
    }
    const int64_t strips = dz_strips(N, out);
    float* part = db ? workspace : nullptr;
    if (is_bf16) launch_dz_t<bf16>(dy, z, dz, part, N, out, act, strips, st);
    else launch_dz_t<float>(dy, z, dz, part, N, out, act, strips, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !db) return e;
    hipLaunchKernelGGL(db_kernel, dim3((unsigned)((out + 63) / 64)), dim3(1024), 0, st, part, db, out, strips);
    return hipGetLastError();
}

hipError_t launch_fill_zero(void* p, size_t bytes, hipStream_t st) {
    const size_t n = bytes / 2;
    if (n == 0) return hipSuccess;
    hipLaunchKernelGGL(fill_zero_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 4096)), dim3(256), 0, st,
                       static_cast<uint16_t*>(p), n);
    return hipGetLastError();
}

}  // namespace mft
