// Launchers of the root-mean-square norm's kernels (rms_norm.hip; called by
// rms_norm_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mft {

struct RmsNormArgs {
    int64_t N, D;
    int64_t sx, sr, st, sy, sdy, sdt, sdx;  // elements from one row to the next
    float eps;
    float one;               // what is added to the weight
    int norm;                // 0: y = s
    const void* x;           // backward: s
    const void* r;           // or null
    const float* w;          // [D] or null
    void* total;             // with r
    void* y;                 // e4m3 bytes with scale
    float* rstd;             // [N] or null
    float* scale;            // [N], the 8-bit output's; null: y in the rows' type
    // backward
    const float* rstd_in;
    const void* dy;
    const void* dt;          // or null
    void* dx;                // may be null
    float* dw;               // may be null
    float* part;             // [groups][D] partial dw
    float* sums;             // [N] sum g h of rows too long for registers
    int64_t groups;
};

hipError_t launch_rms_norm_fwd(const RmsNormArgs& a, bool bf16, hipStream_t st);
// Bytes of the backward's workspace (part, then sums).
size_t rms_norm_workspace(int64_t N, int64_t D, bool bf16);
hipError_t launch_rms_norm_bwd(RmsNormArgs a, bool bf16, void* workspace, hipStream_t st);

}  // namespace mft
