// Launchers of the layer norm kernels (layer_norm.hip; called by
// layer_norm_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mft {

struct LayerNormArgs {
    int64_t N, D;
    int64_t sx, sy, sdy, sdx;  // elements from one row to the next
    float eps;
    const void* x;
    const float* w;            // [D] or null
    const float* b;            // [D] or null
    void* y;
    float* mean;               // [N] written by the forward (may be null)
    float* rstd;
    // backward
    const float* mean_in;
    const float* rstd_in;
    const void* dy;
    void* dx;                  // may be null
    float* dw;                 // may be null
    float* db;                 // may be null
    float* part;               // [groups][2][D] partial dw and db
    float2* sums;              // [N] (sum g, sum g h) of rows too long for registers
    int64_t groups;
};

hipError_t launch_layer_norm_fwd(const LayerNormArgs& a, bool bf16, hipStream_t st);
// Bytes of the backward's workspace (part, then sums).
size_t layer_norm_workspace(int64_t N, int64_t D, bool bf16);
hipError_t launch_layer_norm_bwd(LayerNormArgs a, bool bf16, void* workspace, hipStream_t st);

}  // namespace mft
