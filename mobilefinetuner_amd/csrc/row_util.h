// Device helpers of the row-wise passes: loads and stores of a few consecutive
// elements at any element address, and sums over a wave in registers.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "attn_common.h"

namespace mft {

// V consecutive elements of type T as floats.  The vector type has T's
// alignment: a wide access may start at any element (rows of odd length).
template <typename T, int V> struct AnyVec {
    typedef T raw __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    __device__ __forceinline__ static raw load_raw(const T* p) { return *reinterpret_cast<const raw*>(p); }
    __device__ __forceinline__ static void load(const T* p, float* x) {
        const raw r = load_raw(p);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (float)r[e];
    }
    __device__ __forceinline__ static void store(T* p, const float* x) {
        raw r;
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = (T)x[e];
        *reinterpret_cast<raw*>(p) = r;
    }
};

// Elements d0 .. d0 + V - 1 of a row of D elements, zero past its end.
template <typename T, int V>
__device__ __forceinline__ void load_part(const T* row, int64_t d0, int64_t D, float* x) {
    if (d0 + V <= D) {
        AnyVec<T, V>::load(row + d0, x);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = d0 + e < D ? (float)row[d0 + e] : 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_part(T* row, int64_t d0, int64_t D, const float* x) {
    if (d0 + V <= D) {
        AnyVec<T, V>::store(row + d0, x);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (d0 + e < D) row[d0 + e] = (T)x[e];
    }
}

// Sum of V values (a power of two) in pairs.
template <int V> __device__ __forceinline__ float sum_pairs(const float* x) {
    if constexpr (V == 1) return x[0];
    else return sum_pairs<V / 2>(x) + sum_pairs<V / 2>(x + V / 2);
}

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Sum over the wave, the same bits in every lane: pairs by DPP within rows of
// 16 lanes (quads by permutation, then mirrored halves and rows), then by lane
// swaps across them.  All lanes must be active.
__device__ __forceinline__ float wave_sum_f(float x) {
    x += dpp<0xB1>(x);   // quad_perm [1, 0, 3, 2]
    x += dpp<0x4E>(x);   // quad_perm [2, 3, 0, 1]
    x += dpp<0x141>(x);  // row_half_mirror
    x += dpp<0x140>(x);  // row_mirror
    x = row16_sum(x);
    return half_sum(x);
}

// x of lane (lane ^ O), in registers: quads, halves and rows of 16 by DPP, the
// rest by lane swaps.  All lanes must be active.
template <int O> __device__ __forceinline__ uint32_t lane_xor(uint32_t x, int lane) {
    auto dpp_u = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    if constexpr (O == 1) return dpp_u(x, std::integral_constant<int, 0xB1>{});
    if constexpr (O == 2) return dpp_u(x, std::integral_constant<int, 0x4E>{});
    if constexpr (O == 3) return dpp_u(x, std::integral_constant<int, 0x1B>{});
    if constexpr (O == 7) return dpp_u(x, std::integral_constant<int, 0x141>{});
    if constexpr (O == 4) return lane_xor<3>(lane_xor<7>(x, lane), lane);
    if constexpr (O == 8) return dpp_u(x, std::integral_constant<int, 0x128>{});   // row_ror 8
    if constexpr (O == 15) return dpp_u(x, std::integral_constant<int, 0x140>{});  // row_mirror
    if constexpr (O == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return lane & 16 ? s[0] : s[1];
    }
    if constexpr (O == 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return lane & 32 ? s[0] : s[1];
    }
    if constexpr (O == 63) return lane_xor<32>(lane_xor<16>(lane_xor<15>(x, lane), lane), lane);
}

}  // namespace mft
