// Layer norm over the last dimension, forward and backward (C ABI in
// include/mft/layer_norm.h).
//
// A row is held in registers, by one wave (WPR = 1), four or sixteen: one read
// of x, the mean, then the sums of d = x - mean and d^2 about it, so that a
// mean far above the deviation costs no digits: there d is exact, and its sum,
// zero but for the mean's rounding, corrects the mean.  A mean below the deviation
// is taken as it is: x - mean then rounds alike for all x of one binade, and the
// sum of d would carry that (mean of 8192 normal values: 8e-7 off with it).
// Longer rows are read once per sum.  All of it is bound by memory.
//
// Backward: the row sums of g = dy w and g h give dx in one pass over x and dy.
// The sums over rows, dw and db, stay in registers: a workgroup takes rows
// g, g + groups, ... and leaves one partial [2][D], and a second launch adds
// the partials in their order, so results do not depend on the schedule.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_kernels.h"
#include "layer_norm_kernels.h"
#include "row_util.h"

namespace mft {
namespace {

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

// Sums of two values over the WPR waves of a row, in every thread.  `s` is
// scratch of 2 * WPR floats that no other call in flight uses.
template <int WPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* s) {
    a = wave_sum_f(a);
    b = wave_sum_f(b);
    if constexpr (WPR > 1) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            s[2 * w] = a;
            s[2 * w + 1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            a += s[2 * i];
            b += s[2 * i + 1];
        }
    }
}

template <int WPR> constexpr int kThreads = WPR == 1 ? 256 : 64 * WPR;

template <typename T, int WPR, int CH>
__global__ __launch_bounds__(kThreads<WPR>) void ln_fwd(LayerNormArgs a) {
    constexpr int V = kVec<T>, TPR = 64 * WPR;
    __shared__ float s1[2 * WPR], s2[2 * WPR];
    const int t = threadIdx.x % TPR;
    const int64_t n = (int64_t)blockIdx.x * (kThreads<WPR> / TPR) + threadIdx.x / TPR;
    if (n >= a.N) return;  // whole waves: a workgroup of one row has n < N
    const T* xr = (const T*)a.x + n * a.sx;
    float x[CH][V];
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_part<T, V>(xr, (int64_t)(c * TPR + t) * V, a.D, x[c]);
    // Sums of a vector in pairs: a mean near zero is a small difference of its addends.
#pragma unroll
    for (int c = 0; c < CH; ++c) sum += sum_pairs<V>(x[c]);
    row_sum2<WPR>(sum, none, s1);
    const float inv = 1.0f / (float)a.D;
    float mean = sum * inv, d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = (int64_t)(c * TPR + t) * V + e < a.D ? x[c][e] - mean : 0.f;
            x[c][e] = d;
            q[e] = d * d;
        }
        d1 += sum_pairs<V>(x[c]);
        d2 += sum_pairs<V>(q);
    }
    row_sum2<WPR>(d1, d2, s2);
    const float off = mean * mean <= d2 * inv ? 0.f : d1 * inv;  // what the mean's rounding left; NaN stays
    const float rstd = 1.0f / sqrtf(fmaxf(fmaf(-off, off, d2 * inv), 0.f) + a.eps);
    T* yr = (T*)a.y + n * a.sy;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int64_t d0 = (int64_t)(c * TPR + t) * V;
        if (d0 >= a.D) break;
        float w[V], b[V];
        if (a.w) load_part<float, V>(a.w, d0, a.D, w);
        if (a.b) load_part<float, V>(a.b, d0, a.D, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float h = (x[c][e] - off) * rstd;
            x[c][e] = a.w ? (a.b ? fmaf(h, w[e], b[e]) : h * w[e]) : (a.b ? h + b[e] : h);
        }
        store_part<T, V>(yr, d0, a.D, x[c]);
    }
    if (t == 0) {
        if (a.mean) a.mean[n] = mean + off;
        if (a.rstd) a.rstd[n] = rstd;
    }
}

// Rows too long for registers: one workgroup reads the row once per sum and
// once to write.
constexpr int kLongThreads = 1024, kLongWaves = 16;
template <typename T> __global__ __launch_bounds__(kLongThreads) void ln_fwd_long(LayerNormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s1[2 * kLongWaves], s2[2 * kLongWaves];
    const int64_t n = blockIdx.x;
    const T* xr = (const T*)a.x + n * a.sx;
    const float inv = 1.0f / (float)a.D;
    float sum = 0.f, none = 0.f;
    for (int64_t d0 = (int64_t)threadIdx.x * V; d0 < a.D; d0 += kLongThreads * V) {
        float x[V];
        load_part<T, V>(xr, d0, a.D, x);
        sum += sum_pairs<V>(x);
    }
    row_sum2<kLongWaves>(sum, none, s1);
    const float mean = sum * inv;
    float d1 = 0.f, d2 = 0.f;
    for (int64_t d0 = (int64_t)threadIdx.x * V; d0 < a.D; d0 += kLongThreads * V) {
        float x[V], q[V];
        load_part<T, V>(xr, d0, a.D, x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[e] = d0 + e < a.D ? x[e] - mean : 0.f;
            q[e] = x[e] * x[e];
        }
        d1 += sum_pairs<V>(x);
        d2 += sum_pairs<V>(q);
    }
    row_sum2<kLongWaves>(d1, d2, s2);
    const float off = mean * mean <= d2 * inv ? 0.f : d1 * inv;
    const float rstd = 1.0f / sqrtf(fmaxf(fmaf(-off, off, d2 * inv), 0.f) + a.eps);
    T* yr = (T*)a.y + n * a.sy;
    for (int64_t d0 = (int64_t)threadIdx.x * V; d0 < a.D; d0 += kLongThreads * V) {
        float x[V], w[V], b[V];
        load_part<T, V>(xr, d0, a.D, x);
        if (a.w) load_part<float, V>(a.w, d0, a.D, w);
        if (a.b) load_part<float, V>(a.b, d0, a.D, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float h = ((x[e] - mean) - off) * rstd;
            x[e] = a.w ? (a.b ? fmaf(h, w[e], b[e]) : h * w[e]) : (a.b ? h + b[e] : h);
        }
        store_part<T, V>(yr, d0, a.D, x);
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[n] = mean + off;
        if (a.rstd) a.rstd[n] = rstd;
    }
}

// Waves of a backward workgroup: eight rows at once, or one row's waves.
template <int WPR> constexpr int kBwdThreads = WPR == 1 ? 512 : 64 * WPR;

// Workgroup g: rows in steps of groups * (rows a workgroup holds at once).  EVEN:
// D is a multiple of the vector, so that no element is looked at by itself.
// Keeping the next row's loads in flight as well takes more registers than it is
// worth: 16384 x 1024 in bf16 43 us, without and with 16 waves to a CU 31, and 20
// (4.9 TB/s) since the waves' sums meet in LDS by quads, in pairs of waves.
template <typename T, int WPR, int CH, bool PARAMS, bool EVEN>
__global__ __launch_bounds__(kBwdThreads<WPR>) void ln_bwd(LayerNormArgs a) {
    constexpr int V = kVec<T>, TPR = 64 * WPR, NT = kBwdThreads<WPR>, RPB = NT / TPR;
    __shared__ __attribute__((aligned(16))) float lds[PARAMS && RPB > 1 ? RPB * CH * V * 64 : 1];
    __shared__ float s[2][2 * WPR];
    const int t = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.D;
    // Elements from d0 on, 0 past the row's end (and with it all below).
    auto load = [&](auto* row, int64_t d0, float* x) {
        typedef std::remove_const_t<std::remove_pointer_t<decltype(row)>> E;
        if constexpr (EVEN) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = 0.f;
            if (d0 < a.D) AnyVec<E, V>::load(row + d0, x);
        } else {
            load_part<E, V>(row, d0, a.D, x);
        }
    };
    float dw[CH][V], db[CH][V], w[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = 0.f, w[c][e] = 1.f;
        if (a.w) load(a.w, (int64_t)(c * TPR + t) * V, w[c]);
    }
    int turn = 0;
    for (int64_t n = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; n < a.N; n += a.groups * RPB) {
        const T* xr = (const T*)a.x + n * a.sx;
        const T* gr = (const T*)a.dy + n * a.sdy;
        float h[CH][V], g[CH][V];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            load(xr, (int64_t)(c * TPR + t) * V, h[c]);
            load(gr, (int64_t)(c * TPR + t) * V, g[c]);
        }
        const float mean = a.mean_in[n], rstd = a.rstd_in[n];
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[c][e] = (h[c][e] - mean) * rstd;
                if constexpr (PARAMS) {
                    dw[c][e] = fmaf(g[c][e], h[c][e], dw[c][e]);
                    db[c][e] += g[c][e];
                }
                g[c][e] *= w[c][e];
                c1 += g[c][e];
                c2 = fmaf(g[c][e], h[c][e], c2);
            }
        if (a.dx) {
            row_sum2<WPR>(c1, c2, s[turn]);
            turn ^= 1;
            c1 *= inv;
            c2 *= inv;
            T* dr = (T*)a.dx + n * a.sdx;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t d0 = (int64_t)(c * TPR + t) * V;
                if (d0 >= a.D) break;
#pragma unroll
                for (int e = 0; e < V; ++e) g[c][e] = rstd * (g[c][e] - c1 - h[c][e] * c2);
                if constexpr (EVEN) AnyVec<T, V>::store(dr + d0, g[c]);
                else store_part<T, V>(dr, d0, a.D, g[c]);
            }
        }
    }
    if constexpr (PARAMS) {
        float* out = a.part + (int64_t)blockIdx.x * 2 * a.D;
        if constexpr (RPB > 1) {
            // The waves' sums meet in pairs, half of the waves handing theirs over at a time: quads of
            // columns, lane by lane, so that no bank is met twice.
            constexpr int QUADS = 2 * CH * V / 4, SLOT = QUADS * 64 * 4;  // floats of a wave: dw, then db
            const int wave = threadIdx.x / 64;
            auto quad = [&](int q) { return q < QUADS / 2 ? &dw[0][0] + 4 * q : &db[0][0] + 4 * (q - QUADS / 2); };
#pragma unroll
            for (int half = RPB / 2; half > 0; half /= 2) {
                if (wave >= half && wave < 2 * half)
#pragma unroll
                    for (int q = 0; q < QUADS; ++q)
                        *reinterpret_cast<f32x4*>(lds + (wave - half) * SLOT + (q * 64 + t) * 4) =
                            f32x4{quad(q)[0], quad(q)[1], quad(q)[2], quad(q)[3]};
                __syncthreads();
                if (wave < half)
#pragma unroll
                    for (int q = 0; q < QUADS; ++q) {
                        const f32x4 o = *reinterpret_cast<const f32x4*>(lds + wave * SLOT + (q * 64 + t) * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) quad(q)[e] += o[e];
                    }
                __syncthreads();
            }
            if (wave == 0)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int64_t d0 = (int64_t)(c * TPR + t) * V;
                    store_part<float, V>(out, d0, a.D, dw[c]);
                    store_part<float, V>(out + a.D, d0, a.D, db[c]);
                }
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t d0 = (int64_t)(c * TPR + t) * V;
                store_part<float, V>(out, d0, a.D, dw[c]);
                store_part<float, V>(out + a.D, d0, a.D, db[c]);
            }
        }
    }
}

// Rows too long for registers: their two sums, then dx and the partials of dw
// and db by columns.
template <typename T> __global__ __launch_bounds__(kLongThreads) void ln_bwd_sums(LayerNormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s[2 * kLongWaves];
    const int64_t n = blockIdx.x;
    const T* xr = (const T*)a.x + n * a.sx;
    const T* gr = (const T*)a.dy + n * a.sdy;
    const float mean = a.mean_in[n], rstd = a.rstd_in[n];
    float c1 = 0.f, c2 = 0.f;
    for (int64_t d0 = (int64_t)threadIdx.x * V; d0 < a.D; d0 += kLongThreads * V) {
        float x[V], g[V], w[V], p1 = 0.f, p2 = 0.f;
        load_part<T, V>(xr, d0, a.D, x);
        load_part<T, V>(gr, d0, a.D, g);
        if (a.w) load_part<float, V>(a.w, d0, a.D, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float q = a.w ? g[e] * w[e] : g[e];
            p1 += q;
            p2 = fmaf(q, (x[e] - mean) * rstd, p2);
        }
        c1 += p1;
        c2 += p2;
    }
    row_sum2<kLongWaves>(c1, c2, s);
    if (threadIdx.x == 0) a.sums[n] = make_float2(c1, c2);
}

template <typename T> __global__ __launch_bounds__(256) void ln_bwd_columns(LayerNormArgs a) {
    const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (d >= a.D) return;
    const float inv = 1.0f / (float)a.D, w = a.w ? a.w[d] : 1.f;
    float dw = 0.f, db = 0.f;
#pragma unroll 4
    for (int64_t n = blockIdx.y; n < a.N; n += a.groups) {
        const float rstd = a.rstd_in[n], h = ((float)((const T*)a.x)[n * a.sx + d] - a.mean_in[n]) * rstd;
        const float g = (float)((const T*)a.dy)[n * a.sdy + d];
        dw = fmaf(g, h, dw);
        db += g;
        if (a.dx) {
            const float2 c = a.sums[n];
            ((T*)a.dx)[n * a.sdx + d] = (T)(rstd * (g * w - c.x * inv - h * (c.y * inv)));
        }
    }
    if (a.part) {
        float* out = a.part + (int64_t)blockIdx.y * 2 * a.D;
        out[d] = dw;
        out[a.D + d] = db;
    }
}

// dw and db from column `first` of the two on: the groups' partials in order.  32
// columns (a line) to a workgroup; its 32 rows of threads take the groups in turn.
__global__ __launch_bounds__(1024) void ln_params(LayerNormArgs a, int64_t first) {
    __shared__ float s[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t c = first + (int64_t)blockIdx.x * 32 + x, C = 2 * a.D;
    float v = 0.f;
    if (c < C)
#pragma unroll 8
        for (int64_t g = y; g < a.groups; g += 32) v += a.part[g * C + c];
    s[y][x] = v;
    __syncthreads();
    if (y != 0 || c >= C) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][x];
    if (c < a.D) {
        if (a.dw) a.dw[c] = v;
    } else if (a.db) {
        a.db[c - a.D] = v;
    }
}

__global__ __launch_bounds__(256) void ln_zero_params(LayerNormArgs a) {
    const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (d >= a.D) return;
    if (a.dw) a.dw[d] = 0.f;
    if (a.db) a.db[d] = 0.f;
}

// Waves to a row and 16-byte chunks to a thread.  WPR 0: by memory.
struct Shape {
    int wpr, ch;
};
Shape fwd_shape(int64_t D, int vec) {
    for (const Shape s : {Shape{1, 1}, {1, 2}, {1, 4}, {1, 8}, {4, 4}, {4, 8}, {16, 4}, {16, 8}})
        if (D <= (int64_t)64 * s.wpr * s.ch * vec && s.ch * vec * s.wpr <= 512) return s;  // 16 waves: 128 registers
    return {0, 0};
}
Shape bwd_shape(int64_t D, int vec) {
    for (const Shape s : {Shape{1, 1}, {1, 2}, {1, 4}, {4, 2}, {4, 4}, {16, 2}})
        if (D <= (int64_t)64 * s.wpr * s.ch * vec && s.ch * vec <= 16 * (s.wpr == 4 ? 2 : 1)) return s;
    return {0, 0};
}
int64_t bwd_groups(int64_t N, int64_t D, int vec) {
    const Shape s = bwd_shape(D, vec);
    const int64_t at_once = s.wpr == 1 ? 8 : 1, most = s.wpr == 16 || s.wpr == 0 ? 1 : 2;
    // few rows, a wave to each: one workgroup to a CU, as each leaves a partial
    return std::max<int64_t>(1, std::min<int64_t>((N + at_once - 1) / at_once,
                                                  (s.wpr == 1 && N < 64 * device_cus() ? 1 : most) * device_cus()));
}
size_t up(size_t x) { return (x + 255) & ~size_t(255); }

// f(first row, rows) for as many rows at a time as a launch's 2^32 threads allow.
template <typename F> void row_slices(int64_t N, int wpr, F f) {
    const int64_t most = (int64_t(1) << 31) / (64 * (wpr ? wpr : kLongWaves));
    for (int64_t n = 0; n < N; n += most) f(n, std::min(most, N - n));
}

template <typename T> void fwd_rows(const LayerNormArgs& a, const Shape& s, hipStream_t st) {
    const dim3 grid((unsigned)(s.wpr == 1 ? (a.N + 3) / 4 : a.N));
#define MFT_LN_FWD(WPR, CH) \
    if (s.wpr == WPR && s.ch == CH) hipLaunchKernelGGL((ln_fwd<T, WPR, CH>), grid, dim3(kThreads<WPR>), 0, st, a)
    MFT_LN_FWD(1, 1);
    MFT_LN_FWD(1, 2);
    MFT_LN_FWD(1, 4);
    MFT_LN_FWD(1, 8);
    MFT_LN_FWD(4, 4);
    MFT_LN_FWD(4, 8);
    MFT_LN_FWD(16, 4);
    if constexpr (kVec<T> == 4) MFT_LN_FWD(16, 8);
#undef MFT_LN_FWD
    if (s.wpr == 0) hipLaunchKernelGGL((ln_fwd_long<T>), grid, dim3(kLongThreads), 0, st, a);
}
template <typename T> hipError_t fwd(const LayerNormArgs& a, hipStream_t st) {
    const Shape s = fwd_shape(a.D, kVec<T>);
    row_slices(a.N, s.wpr, [&](int64_t n, int64_t rows) {
        LayerNormArgs q = a;
        q.N = rows;
        q.x = (const T*)a.x + n * a.sx;
        q.y = (T*)a.y + n * a.sy;
        if (a.mean) q.mean = a.mean + n;
        if (a.rstd) q.rstd = a.rstd + n;
        fwd_rows<T>(q, s, st);
    });
    return hipGetLastError();
}

template <typename T> hipError_t bwd(const LayerNormArgs& a, hipStream_t st) {
    const Shape s = bwd_shape(a.D, kVec<T>);
    const bool params = a.dw || a.db;
    if (s.wpr == 0) {
        LayerNormArgs q = a;
        if (!params) q.part = nullptr;
        if (a.dx) {
            row_slices(a.N, 0, [&](int64_t n, int64_t rows) {
                LayerNormArgs r = a;
                r.x = (const T*)a.x + n * a.sx;
                r.dy = (const T*)a.dy + n * a.sdy;
                r.mean_in = a.mean_in + n;
                r.rstd_in = a.rstd_in + n;
                r.sums = a.sums + n;
                hipLaunchKernelGGL((ln_bwd_sums<T>), dim3((unsigned)rows), dim3(kLongThreads), 0, st, r);
            });
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL((ln_bwd_columns<T>), dim3((unsigned)((a.D + 255) / 256), (unsigned)a.groups), dim3(256), 0,
                           st, q);
    }
#define MFT_LN_BWD_E(WPR, CH, PARAMS)                                                                           \
    do {                                                                                                        \
        if (a.D % kVec<T> == 0)                                                                                 \
            hipLaunchKernelGGL((ln_bwd<T, WPR, CH, PARAMS, true>), grid, dim3(kBwdThreads<WPR>), 0, st, a);     \
        else                                                                                                    \
            hipLaunchKernelGGL((ln_bwd<T, WPR, CH, PARAMS, false>), grid, dim3(kBwdThreads<WPR>), 0, st, a);    \
    } while (0)
#define MFT_LN_BWD(WPR, CH)                                                                                     \
    if (s.wpr == WPR && s.ch == CH) {                                                                           \
        if (params) MFT_LN_BWD_E(WPR, CH, true);                                                                \
        else MFT_LN_BWD_E(WPR, CH, false);                                                                      \
    }
    const dim3 grid((unsigned)a.groups);
    MFT_LN_BWD(1, 1)
    MFT_LN_BWD(1, 2)
    if constexpr (kVec<T> == 4) {
        MFT_LN_BWD(1, 4)
    }
    MFT_LN_BWD(4, 2)
    MFT_LN_BWD(4, 4)
    MFT_LN_BWD(16, 2)
#undef MFT_LN_BWD_E
#undef MFT_LN_BWD
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !params) return e;
    // 32 threads to a column of the two, and fewer than 2^32 to a launch: 2^26 columns at a time
    constexpr int64_t kMost = int64_t(1) << 26;
    for (int64_t c = 0; c < 2 * a.D; c += kMost)
        hipLaunchKernelGGL(ln_params, dim3((unsigned)((std::min(kMost, 2 * a.D - c) + 31) / 32)), dim3(1024), 0, st, a, c);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm_fwd(const LayerNormArgs& a, bool is_bf16, hipStream_t st) {
    if (a.N == 0) return hipSuccess;
    return is_bf16 ? fwd<bf16>(a, st) : fwd<float>(a, st);
}

size_t layer_norm_workspace(int64_t N, int64_t D, bool is_bf16) {
    const int vec = is_bf16 ? kVec<bf16> : kVec<float>;
    size_t n = up((size_t)bwd_groups(N, D, vec) * 2 * D * 4);
    if (bwd_shape(D, vec).wpr == 0) n += up((size_t)N * sizeof(float2));
    return n;
}

hipError_t launch_layer_norm_bwd(LayerNormArgs a, bool is_bf16, void* workspace, hipStream_t st) {
    if (a.N == 0) {
        if (!a.dw && !a.db) return hipSuccess;
        hipLaunchKernelGGL(ln_zero_params, dim3((unsigned)((a.D + 255) / 256)), dim3(256), 0, st, a);
        return hipGetLastError();
    }
    if (!a.dx && !a.dw && !a.db) return hipSuccess;
    const int vec = is_bf16 ? kVec<bf16> : kVec<float>;
    a.groups = bwd_groups(a.N, a.D, vec);
    a.part = static_cast<float*>(workspace);
    a.sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + up((size_t)a.groups * 2 * a.D * 4));
    return is_bf16 ? bwd<bf16>(a, st) : bwd<float>(a, st);
}

}  // namespace mft
