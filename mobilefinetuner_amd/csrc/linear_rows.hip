// The linear layer's products of few rows (a generated token, a handful of
// sequences; C ABI in include/mft/linear.h):
// C[M, N] = act(sum_k P(m, k) Q(n, k) + bias[n]) + residual, M <= kMaxRows.
//
// Q is read once and bounds it.  Each of its elements is multiplied by the M
// rows' in fp32 in the lane that has loaded it, 16 bytes a lane; sums meet in
// registers and, across waves, in LDS, in an order that the sizes fix.
//
// Q with k contiguous: a wave takes four rows of Q, or one where that leaves
// fewer than four waves to a CU, and its lanes share k.  Q with its rows
// contiguous: a workgroup takes 64 consecutive n or fewer (so that about 128
// workgroups run) and its lanes' groups share k.  bf16, one row, W out of cache:
// 1024 -> 4096 5.7 us (W [out, in]) and 6.2 ([in, out]), 4096 -> 1024 6.9 and 10.6;
// on 64 x 64 tiles of the matrix units 8.6, 8.9, 10.6 and 10.6.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_geometry.h"
#include "attn_kernels.h"
#include "linear_act.h"
#include "linear_epilogue.h"
#include "row_util.h"

namespace mft {
namespace {

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
// Against the tiles of the matrix units, on operands out of cache, eight layers of 768 to 8192: one row
// 4.5 to 13.5 us for 8 to 13, two 4.5 to 15.6 for 8 to 13 (over K of 4096 and more up to a quarter
// longer here, else shorter), three 11 to 21 for 9 to 13 with W [in, out].
constexpr int kMaxRows = 2;
constexpr int kThreads = 1024, kWaves = kThreads / 64;

template <typename T, int MR, int ACT, int COLS> __global__ __launch_bounds__(256) void rows_kc(LinearProduct g) {
    constexpr int V = kVec<T>;
    const int lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)xcd_block((int)blockIdx.x, (int)gridDim.x) * 4 + wave_id()) * COLS;
    if (n0 >= g.N) return;
    const T *P = (const T*)g.P, *Q = (const T*)g.Q;
    float acc[COLS][MR] = {};
#pragma unroll 4
    for (int64_t k = (int64_t)lane * V; k < g.K; k += 64 * V) {
        float q[COLS][V], p[MR][V];
#pragma unroll
        for (int c = 0; c < COLS; ++c) load_part<T, V>(Q + min(n0 + c, g.N - 1) * g.K, k, g.K, q[c]);
#pragma unroll
        for (int m = 0; m < MR; ++m) load_part<T, V>(P + min<int64_t>(m, g.M - 1) * g.K, k, g.K, p[m]);
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int m = 0; m < MR; ++m)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[c][m] = fmaf(q[c][e], p[m][e], acc[c][m]);
    }
    float out = 0.f;  // lane c + COLS m has column c of row m
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const float s = wave_sum_f(acc[c][m]);
            if (lane == c + COLS * m) out = s;
        }
    const int64_t n = n0 + lane % COLS, m = lane / COLS;
    if (m < min<int64_t>(MR, g.M) && n < g.N) linear_epilogue<T, ACT, 1>(g, m, n, &out);
}

// CH: lanes to a workgroup's columns (CH * V of them).
template <typename T, int MR, int ACT, int CH> __global__ __launch_bounds__(kThreads) void rows_nkc(LinearProduct g) {
    constexpr int V = kVec<T>, COLS = CH * V, GROUPS = kThreads / CH;
    __shared__ float part[kWaves][MR][COLS];
    const int lane = threadIdx.x & 63, w = wave_id(), c = threadIdx.x % CH;
    const int64_t n0 = (int64_t)xcd_block((int)blockIdx.x, (int)gridDim.x) * COLS, n = n0 + c * V;
    const T *P = (const T*)g.P, *Q = (const T*)g.Q;
    float acc[MR][V] = {};
    if (n < g.N) {
#pragma unroll 4
        for (int64_t k = threadIdx.x / CH; k < g.K; k += GROUPS) {
            float q[V];
            load_part<T, V>(Q + k * g.N, n, g.N, q);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const float p = (float)P[min<int64_t>(m, g.M - 1) * g.K + k];
#pragma unroll
                for (int e = 0; e < V; ++e) acc[m][e] = fmaf(q[e], p, acc[m][e]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int e = 0; e < V; ++e) {
#pragma unroll
            for (int o = 32; o >= CH; o >>= 1) acc[m][e] += __shfl_xor(acc[m][e], o, 64);
            if (lane < CH) part[w][m][lane * V + e] = acc[m][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < MR * COLS; i += kThreads) {
        const int m = i / COLS, col = i % COLS;
        float v = part[0][m][col];
#pragma unroll
        for (int j = 1; j < kWaves; ++j) v += part[j][m][col];
        if (m < g.M && n0 + col < g.N) linear_epilogue<T, ACT, 1>(g, m, n0 + col, &v);
    }
}

template <typename T, int MR, int ACT> void launch_m(const LinearProduct& g, hipStream_t st) {
    if (g.q_kc) {
        auto waves = [&](int cols) { return dim3((unsigned)((g.N + 4 * cols - 1) / (4 * cols))); };
        if (g.N >= 16 * device_cus()) hipLaunchKernelGGL((rows_kc<T, MR, ACT, 4>), waves(4), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((rows_kc<T, MR, ACT, 1>), waves(1), dim3(256), 0, st, g);
        return;
    }
    auto grid = [&](int ch) { return dim3((unsigned)((g.N + ch * kVec<T> - 1) / (ch * kVec<T>))); };
    const int64_t few = device_cus() / 2;
    if (g.N / (8 * kVec<T>) >= few)
        hipLaunchKernelGGL((rows_nkc<T, MR, ACT, 8>), grid(8), dim3(kThreads), 0, st, g);
    else if (g.N / (4 * kVec<T>) >= few)
        hipLaunchKernelGGL((rows_nkc<T, MR, ACT, 4>), grid(4), dim3(kThreads), 0, st, g);
    else
        hipLaunchKernelGGL((rows_nkc<T, MR, ACT, 2>), grid(2), dim3(kThreads), 0, st, g);
}
template <typename T, int ACT> void launch_a(const LinearProduct& g, hipStream_t st) {
    if (g.M == 1) launch_m<T, 1, ACT>(g, st);
    else launch_m<T, 2, ACT>(g, st);
}
template <typename T> void launch_t(const LinearProduct& g, hipStream_t st) {
    switch (g.act) {
        case ACT_RELU: launch_a<T, ACT_RELU>(g, st); break;
        case ACT_GELU_TANH: launch_a<T, ACT_GELU_TANH>(g, st); break;
        case ACT_SILU: launch_a<T, ACT_SILU>(g, st); break;
        default: launch_a<T, ACT_NONE>(g, st); break;
    }
}

}  // namespace

bool few_rows(const LinearProduct& g) { return g.p_kc && g.M <= kMaxRows; }

hipError_t launch_few_rows(const LinearProduct& g, bool is_bf16, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    if (!few_rows(g)) return hipErrorInvalidValue;
    if (is_bf16) launch_t<bf16>(g, st);
    else launch_t<float>(g, st);
    return hipGetLastError();
}

}  // namespace mft
