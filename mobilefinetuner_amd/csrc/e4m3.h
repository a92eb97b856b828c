// Numbers in 8 bits on the device: e4m3 (OCP: 4 exponent and 3 mantissa bits,
// largest 448, smallest 2^-9, no infinity) next to an fp32 scale.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "row_util.h"

namespace mft {

constexpr float kE4m3Max = 448.f, kE4m3Min = 0x1p-9f;
constexpr float kScaleMin = 0x1p-126f;  // a scale's reciprocal stays finite

// The scale that takes a maximum of magnitudes (its bits; a NaN's are above
// infinity's, so it stays) to the largest e4m3 number: times 1 / 448 in fp32, as
// torch's kernels divide by a number, so that both hold the same numbers.
__device__ __forceinline__ float e4m3_scale(uint32_t max_bits) {
    const float s = __uint_as_float(max_bits) * (1.0f / kE4m3Max);
    return s < kScaleMin ? kScaleMin : s;  // a NaN stays
}

// Quotients by a scale, each x / scale rounded to nearest once, of which e4m3 numbers are then taken: by the
// reciprocal alone (x inv) 0.06 percent of a bf16 matrix's came out a number off, as its quotients often lie halfway
// between two.  Two corrections by exact remainders: the first leaves a number next to the quotient, and from there
// the second rounds it correctly (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990: inv is the nearest to 1 / scale, the remainder a float).  The remainder of a quotient from 2^-11 on
// is a float while the scale is above 2^-91; smaller quotients are zeros either way.  An infinite scale's finite values
// are 0.  8192 x 1152 with its norm 17.0 us, by the reciprocal 16.3, by the operator's own sequence throughout 18.6.
struct E4m3Divisor {
    float scale, inv;
    bool fast;
    __device__ __forceinline__ explicit E4m3Divisor(float s) : scale(s), inv(1.0f / s), fast(s >= 0x1p-80f && s < INFINITY) {}
    template <int V> __device__ __forceinline__ void divide(float* x) const {
        if (fast) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float q = x[e] * inv;
                q = fmaf(fmaf(-q, scale, x[e]), inv, q);
                x[e] = fmaf(fmaf(-q, scale, x[e]), inv, q);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] /= scale;
        }
    }
};

// Four values to nearest even.  Up to 448 (1 + 2^-22), which rounds to 448: no
// value of a group exceeds its scale's by more.
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ void e4m3_unpack4(uint32_t v, float* x) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}

// V values at a byte of any address, the first `n` of them where fewer than V are left.
template <int V> __device__ __forceinline__ void e4m3_store(uint8_t* p, int64_t n, const float* x) {
    typedef uint32_t raw __attribute__((ext_vector_type(V / 4), aligned(1)));
    raw r;
#pragma unroll
    for (int e = 0; e < V / 4; ++e) r[e] = e4m3_pack4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    if (n >= V) {
        *reinterpret_cast<raw*>(p) = r;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = (uint8_t)(r[e / 4] >> (8 * (e & 3)));
    }
}

// Maximum over the wave, in every lane.  All lanes must be active.
__device__ __forceinline__ uint32_t wave_max_u(uint32_t x, int lane) {
    x = max(x, lane_xor<1>(x, lane));
    x = max(x, lane_xor<2>(x, lane));
    x = max(x, lane_xor<7>(x, lane));   // the other quad of eight lanes
    x = max(x, lane_xor<15>(x, lane));  // the other eight of sixteen
    x = max(x, lane_xor<16>(x, lane));
    return max(x, lane_xor<32>(x, lane));
}

}  // namespace mft
