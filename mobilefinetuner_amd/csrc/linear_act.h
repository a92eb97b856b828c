// The activations of the linear layer's epilogue and their derivatives, in
// fp32.  The exponential form of GELU's tanh, z / (1 + exp(-2 u)), keeps the
// digits that 1 + tanh(u) loses below zero.
#pragma once

#include "attn_common.h"
#include "linear_kernels.h"

namespace mft {

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

template <int ACT> __device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == ACT_RELU) return z <= 0.f ? 0.f : z;  // a NaN stays
    if constexpr (ACT == ACT_GELU_TANH || ACT == ACT_SILU) {
        // exponent of 2 of exp(-2 u), or of exp(-z)
        const float x = ACT == ACT_SILU ? z * -kLog2e
                                        : z * fmaf(z * z, -2.f * kLog2e * kGeluC * kGeluA, -2.f * kLog2e * kGeluC);
        return z * __builtin_amdgcn_rcpf(1.f + fast_exp2(x));
    }
    return z;
}

template <int ACT> __device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == ACT_GELU_TANH || ACT == ACT_SILU) {
        // Past these the derivative is its limit to fp32, and powers of z overflow (a NaN stays).
        constexpr float kFar = ACT == ACT_SILU ? 80.f : 15.f;
        z = z < -kFar ? -kFar : z > kFar ? kFar : z;
        const float zz = z * z;
        const float x = ACT == ACT_SILU ? z * -kLog2e
                                        : z * fmaf(zz, -2.f * kLog2e * kGeluC * kGeluA, -2.f * kLog2e * kGeluC);
        const float e = fast_exp2(fminf(x, 120.f));  // e s below is then no inf * 0 (and a NaN's z s is NaN)
        const float s = __builtin_amdgcn_rcpf(1.f + e);
        // s + z s (1 - s) 2 u', 1 - s = e s
        const float du = ACT == ACT_SILU ? 1.f : fmaf(zz, 6.f * kGeluC * kGeluA, 2.f * kGeluC);
        return fmaf(z * s, e * s * du, s);
    }
    return 1.f;
}

}  // namespace mft
