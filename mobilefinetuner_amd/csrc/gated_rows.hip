// The gated linear layer's products of few rows (a generated token, a handful of
// sequences; C ABI in include/mft/gated_linear.h):
// C[M, N] = act(sum_k P(m, k) Q(n, k)) (sum_k P(m, k) Q2(n, k)), M <= 2.
//
// Both weights are read once and bound it.  Each of their elements is multiplied
// by the M rows' in fp32 in the lane that has loaded it, 16 bytes a lane; sums meet
// in registers and, across waves, in LDS, in an order that the sizes fix.
//
// With k contiguous a wave takes one row of either weight, or two from 32 waves to a
// CU on, and its lanes share k.  bf16, one row, weights out of cache: 896 -> 4864 6.8 us
// (two rows 7.1), 1152 -> 6912 10.6 (10.2; 3.1 TB/s), 4096 -> 8192 25.9 (24.9; 5.4 TB/s).  With its rows
// contiguous a workgroup takes 64 consecutive n or fewer of both (so that about 128
// workgroups run) and its lanes' groups share k.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_geometry.h"
#include "attn_kernels.h"
#include "e4m3.h"
#include "linear_epilogue.h"
#include "row_util.h"

namespace mft {
namespace {

// The storage of e4m3 numbers, and what their product needs beside the weights.
struct e4m3 {
    uint8_t bits;
};
struct Scales {
    const float *x, *gate, *up;
};

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes of a row of K from element k on, zeros past its end.
template <typename T> __device__ __forceinline__ u32x4 load16(const T* row, int64_t k, int64_t K) {
    typedef u32x4 any16 __attribute__((aligned(1)));
    constexpr int V = kVec<T>;
    u32x4 v{};
    if (k + V <= K) {
        v = *reinterpret_cast<const any16*>(row + k);
    } else if (k < K) {
        T part[V] = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (k + e < K) part[e] = row[k + e];
        v = __builtin_bit_cast(u32x4, part);
    }
    return v;
}
template <typename T> __device__ __forceinline__ void unpack(u32x4 v, float* x) {
    if constexpr (std::is_same_v<T, e4m3>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e4m3_unpack4(v[i], x + 4 * i);
    } else if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
}
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kAhead = 4;

template <typename T, int MR, int COLS> __global__ __launch_bounds__(256) void gated_rows_kc(LinearProduct g, Scales s) {
    constexpr int V = kVec<T>, R = 2 * COLS;  // rows of the weights: gate's, then up's
    const int lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)xcd_block((int)blockIdx.x, (int)gridDim.x) * 4 + wave_id()) * COLS;
    if (n0 >= g.N) return;
    const T *P = (const T*)g.P, *Q[2] = {(const T*)g.Q, (const T*)g.Q2};
    float acc[R][MR] = {};
    // All loads of kAhead rounds go out before the first is used, whatever K is: one round at a time a row of
    // 1152 was three round trips, 13.5 us for 1 x 1152 -> 6912 in bf16.
    for (int64_t k0 = (int64_t)lane * V; k0 < g.K; k0 += kAhead * 64 * V) {
        u32x4 q[kAhead][R], p[kAhead][MR];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t k = k0 + u * 64 * V;
#pragma unroll
            for (int r = 0; r < R; ++r) q[u][r] = load16(Q[r / COLS] + min(n0 + r % COLS, g.N - 1) * g.K, k, g.K);
#pragma unroll
            for (int m = 0; m < MR; ++m) p[u][m] = load16(P + min<int64_t>(m, g.M - 1) * g.K, k, g.K);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float x[MR][V];
#pragma unroll
            for (int m = 0; m < MR; ++m) unpack<T>(p[u][m], x[m]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float w[V];
                unpack<T>(q[u][r], w);
#pragma unroll
                for (int m = 0; m < MR; ++m)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[r][m] = fmaf(w[e], x[m][e], acc[r][m]);
            }
        }
    }
    float gate = 0.f, up = 0.f;  // lane c + COLS m has column c of row m
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const float a = wave_sum_f(acc[c][m]), b = wave_sum_f(acc[COLS + c][m]);
            if (lane == c + COLS * m) gate = a, up = b;
        }
    const int64_t n = n0 + lane % COLS, m = lane / COLS;
    if (m >= min<int64_t>(MR, g.M) || n >= g.N) return;
    if constexpr (std::is_same_v<T, e4m3>) {
        gate = gate * s.x[m] * s.gate[n];
        up = up * s.x[m] * s.up[n];
        gated_epilogue<bf16, 1>(g, m, n, &gate, &up);
    } else {
        gated_epilogue<T, 1>(g, m, n, &gate, &up);
    }
}

// CH: lanes to a workgroup's columns (CH * V of them).
template <typename T, int MR, int CH> __global__ __launch_bounds__(kThreads) void gated_rows_nkc(LinearProduct g) {
    constexpr int V = kVec<T>, COLS = CH * V, GROUPS = kThreads / CH;
    __shared__ float part[kWaves][2][MR][COLS];
    const int lane = threadIdx.x & 63, w = wave_id(), c = threadIdx.x % CH;
    const int64_t n0 = (int64_t)xcd_block((int)blockIdx.x, (int)gridDim.x) * COLS, n = n0 + c * V;
    const T *P = (const T*)g.P, *Q[2] = {(const T*)g.Q, (const T*)g.Q2};
    float acc[2][MR][V] = {};
    if (n < g.N) {
#pragma unroll 4
        for (int64_t k = threadIdx.x / CH; k < g.K; k += GROUPS) {
            float q[2][V];
#pragma unroll
            for (int i = 0; i < 2; ++i) load_part<T, V>(Q[i] + k * g.N, n, g.N, q[i]);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const float p = (float)P[min<int64_t>(m, g.M - 1) * g.K + k];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[i][m][e] = fmaf(q[i][e], p, acc[i][m][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float v = acc[i][m][e];
#pragma unroll
                for (int o = 32; o >= CH; o >>= 1) v += __shfl_xor(v, o, 64);
                if (lane < CH) part[w][i][m][lane * V + e] = v;
            }
    __syncthreads();
    for (int i = threadIdx.x; i < MR * COLS; i += kThreads) {
        const int m = i / COLS, col = i % COLS;
        float gate = part[0][0][m][col], up = part[0][1][m][col];
#pragma unroll
        for (int j = 1; j < kWaves; ++j) gate += part[j][0][m][col], up += part[j][1][m][col];
        if (m < g.M && n0 + col < g.N) gated_epilogue<T, 1>(g, m, n0 + col, &gate, &up);
    }
}

template <typename T, int MR> void launch_kc(const LinearProduct& g, const Scales& s, hipStream_t st) {
    auto waves = [&](int cols) { return dim3((unsigned)((g.N + 4 * cols - 1) / (4 * cols))); };
    if (g.N >= 32 * device_cus()) hipLaunchKernelGGL((gated_rows_kc<T, MR, 2>), waves(2), dim3(256), 0, st, g, s);
    else hipLaunchKernelGGL((gated_rows_kc<T, MR, 1>), waves(1), dim3(256), 0, st, g, s);
}
template <typename T, int MR> void launch_m(const LinearProduct& g, hipStream_t st) {
    if (g.q_kc) return launch_kc<T, MR>(g, Scales{}, st);
    auto grid = [&](int ch) { return dim3((unsigned)((g.N + ch * kVec<T> - 1) / (ch * kVec<T>))); };
    const int64_t few = device_cus() / 2;
    if (g.N / (8 * kVec<T>) >= few) hipLaunchKernelGGL((gated_rows_nkc<T, MR, 8>), grid(8), dim3(kThreads), 0, st, g);
    else if (g.N / (4 * kVec<T>) >= few) hipLaunchKernelGGL((gated_rows_nkc<T, MR, 4>), grid(4), dim3(kThreads), 0, st, g);
    else hipLaunchKernelGGL((gated_rows_nkc<T, MR, 2>), grid(2), dim3(kThreads), 0, st, g);
}

}  // namespace

hipError_t launch_gated_rows(const LinearProduct& g, bool is_bf16, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    if (!few_rows(g)) return hipErrorInvalidValue;
    if (is_bf16) g.M == 1 ? launch_m<bf16, 1>(g, st) : launch_m<bf16, 2>(g, st);
    else g.M == 1 ? launch_m<float, 1>(g, st) : launch_m<float, 2>(g, st);
    return hipGetLastError();
}

hipError_t launch_gated_rows_e4m3(const LinearProduct& g, const float* x_scale, const float* gate_scale,
                                  const float* up_scale, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    if (!few_rows(g) || !g.q_kc) return hipErrorInvalidValue;
    const Scales s{x_scale, gate_scale, up_scale};
    g.M == 1 ? launch_kc<e4m3, 1>(g, s, st) : launch_kc<e4m3, 2>(g, s, st);
    return hipGetLastError();
}

}  // namespace mft
