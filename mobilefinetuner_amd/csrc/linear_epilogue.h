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
#pragma unroll
    for (int e = 0; e < V; ++e) up[e] *= act_value_of(g.act, gate[e]);
    store_part<T, V>((T*)g.C + m * g.N, n, g.N, up);
}

}  // namespace mft
