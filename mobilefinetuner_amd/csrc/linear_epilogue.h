// The epilogues on fp32 sums.  The linear layer's: bias, z, activation, residual, y;
// the gated linear layer's: gate and up where they are kept, and act(gate) up.
#pragma once

#include "linear_act.h"
#include "linear_kernels.h"
#include "row_util.h"

namespace mft {

// y (and z) of V consecutive columns n of row m from their sums.
template <typename T, int ACT, int V>
__device__ __forceinline__ void linear_epilogue(const LinearProduct& g, int64_t m, int64_t n, float* v) {
    if (g.bias) {
        float b[V];
        load_part<float, V>(g.bias, n, g.N, b);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += b[e];
    }
    if (ACT != ACT_NONE && g.z) store_part<T, V>((T*)g.z + m * g.N, n, g.N, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = act_value<ACT>(v[e]);
    if (g.residual) {
        float r[V];
        load_part<T, V>((const T*)g.residual + m * g.N, n, g.N, r);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += r[e];
    }
    store_part<T, V>((T*)g.C + m * g.N, n, g.N, v);
}

template <typename T, int V>
__device__ __forceinline__ void gated_epilogue(const LinearProduct& g, int64_t m, int64_t n, float* gate, float* up) {
    if (g.z) {
        store_part<T, V>((T*)g.z + m * g.N, n, g.N, gate);
        store_part<T, V>((T*)g.z2 + m * g.N, n, g.N, up);
    }
    const Act act = Act::of(g.act);
#pragma unroll
    for (int e = 0; e < V; ++e) up[e] *= act.value(gate[e]);
    store_part<T, V>((T*)g.C + m * g.N, n, g.N, up);
}

// 32 rows of both sums from mw on in LDS rows of PITCH floats (gate's COLS, then
// up's), columns n = nw + lane % LPR * V of h: what a wave's lanes make of them.  xs
// and the columns' gs and us scale the sums (SCALED: e4m3).  Where no vector of V is
// cut by the rows' end and the activation is smooth, which the whole launch shares, the
// columns take the short way: the matrix units wait meanwhile.  8192 x 1152 -> 6912 on
// 256 x 256 tiles 345 us with a choice and an end for each column, 267 by this.
template <int COLS, int PITCH, bool SCALED>
__device__ __forceinline__ void gated_rows_out(const LinearProduct& g, int64_t mw, int64_t nw, const float* st, int lane,
                                               const float* xs, const float* gs, const float* us) {
    constexpr int V = 8, LPR = COLS / V;
    const int c = lane % LPR * V;
    const int64_t n = nw + c;
    if (n >= g.N) return;
    float scale[2][V];
    if constexpr (SCALED) {
        load_part<float, V>(gs, n, g.N, scale[0]);
        load_part<float, V>(us, n, g.N, scale[1]);
    }
    const Act act = Act::of(g.act);
    auto sums = [&](int row, float (&v)[2][V]) {
        const float x = SCALED ? xs[mw + row] : 1.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(st + row * PITCH + i * COLS + c + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][e + k] = SCALED ? u[k] * x * scale[i][e + k] : u[k];
            }
    };
    const int rows = (int)min<int64_t>(32, g.M - mw), first = lane / LPR;
    if (g.N % V == 0 && !act.relu) {
        const int64_t at = (mw + first) * g.N + n, step = 64 / LPR * g.N;
        bf16 *h = (bf16*)g.C + at, *z = (bf16*)g.z + at, *z2 = (bf16*)g.z2 + at;
#pragma unroll
        for (int r = 0; r < LPR / 2; ++r) {
            const int row = first + r * (64 / LPR);
            if (row >= rows) break;
            float v[2][V];
            sums(row, v);
            if (g.z) {
                AnyVec<bf16, V>::store(z + r * step, v[0]);
                AnyVec<bf16, V>::store(z2 + r * step, v[1]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) v[1][e] *= act.smooth(v[0][e]);
            AnyVec<bf16, V>::store(h + r * step, v[1]);
        }
    } else {
#pragma unroll 1
        for (int row = first; row < rows; row += 64 / LPR) {
            float v[2][V];
            sums(row, v);
            gated_epilogue<bf16, V>(g, mw + row, n, v[0], v[1]);
        }
    }
}

}  // namespace mft
