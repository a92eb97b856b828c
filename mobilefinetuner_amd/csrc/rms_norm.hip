// Root-mean-square norm over the last dimension with the residual's addition in
// front of it, forward (in the rows' type or in 8 bits) and backward (C ABI in
// include/mft/rms_norm.h).
//
// A row is held in registers, by one wave (WPR = 1), four or sixteen: x and the
// residual are read once, the sum s = x + residual is rounded to the stream's
// type, stored and normed as it is stored, so that the backward's s is the
// forward's.  Longer rows go by memory.  All of it is bound by memory: 8192 x 1152 in
// bf16 with a residual and into 8 bits 17.0 us (3.9 TB/s; a copy reaches 4.75).
//
// Backward: the row's sum of g h gives dx in one pass over s, dy and the
// stream's gradient.  The sums over rows, dw, stay in registers: a workgroup takes
// rows g, g + groups, ... and leaves one partial [D], and a second launch adds
// the partials in their order, so results do not depend on the schedule.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_kernels.h"
#include "e4m3.h"
#include "rms_norm_kernels.h"
#include "row_util.h"

namespace mft {
namespace {

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

// A sum over the WPR waves of a row, in every thread.  `s` is scratch of WPR
// floats that no other call in flight uses.
template <int WPR> __device__ __forceinline__ float row_sum(float a, float* s) {
    a = wave_sum_f(a);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
        __syncthreads();
        a = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) a += s[i];
    }
    return a;
}
template <int WPR> __device__ __forceinline__ uint32_t row_max(uint32_t a, uint32_t* s) {
    a = wave_max_u(a, threadIdx.x & 63);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
        __syncthreads();
        a = 0;
#pragma unroll
        for (int i = 0; i < WPR; ++i) a = max(a, s[i]);
    }
    return a;
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int WPR> constexpr int kThreads = WPR == 1 ? 256 : 64 * WPR;

// Sum of squares of V values, in pairs.
template <int V> __device__ __forceinline__ float squares(const float* x) {
    float q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = x[e] * x[e];
    return sum_pairs<V>(q);
}

// V elements of s from d0 on (zeros past the end): x, or x + residual in T, which is stored.
template <typename T, int V>
__device__ __forceinline__ void stream(const RmsNormArgs& a, int64_t n, int64_t d0, float* x) {
    load_part<T, V>((const T*)a.x + n * a.sx, d0, a.D, x);
    if (!a.r) return;
    float r[V];
    load_part<T, V>((const T*)a.r + n * a.sr, d0, a.D, r);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = (float)(T)(x[e] + r[e]);
}
// y's values from s's: factors of V columns from d0 on.
template <int V> __device__ __forceinline__ void factors(const RmsNormArgs& a, int64_t d0, float* f) {
    if (a.w) load_part<float, V>(a.w, d0, a.D, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = a.w ? f[e] + a.one : 1.f;
}

template <typename T, int WPR, int CH, bool E4M3>
__global__ __launch_bounds__(kThreads<WPR>) void rms_fwd(RmsNormArgs a) {
    constexpr int V = kVec<T>, TPR = 64 * WPR;
    __shared__ float s1[WPR];
    __shared__ uint32_t s2[WPR];
    const int t = threadIdx.x % TPR;
    const int64_t n = (int64_t)blockIdx.x * (kThreads<WPR> / TPR) + threadIdx.x / TPR;
    if (n >= a.N) return;  // whole waves: a workgroup of one row has n < N
    float x[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) load_part<T, V>((const T*)a.x + n * a.sx, (int64_t)(c * TPR + t) * V, a.D, x[c]);
    if (a.r) {
        float r[CH][V];
#pragma unroll
        for (int c = 0; c < CH; ++c)
            load_part<T, V>((const T*)a.r + n * a.sr, (int64_t)(c * TPR + t) * V, a.D, r[c]);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t d0 = (int64_t)(c * TPR + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][e] = (float)(T)(x[c][e] + r[c][e]);
            if (d0 < a.D) store_part<T, V>((T*)a.total + n * a.st, d0, a.D, x[c]);
        }
    }
    float rstd = 1.f;
    if (!E4M3 || a.norm) {
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) sum += squares<V>(x[c]);
        rstd = 1.0f / sqrtf(row_sum<WPR>(sum, s1) / (float)a.D + a.eps);
        if (a.rstd && t == 0) a.rstd[n] = rstd;
    }
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int64_t d0 = (int64_t)(c * TPR + t) * V;
        if (d0 >= a.D) break;
        if (!E4M3 || a.norm) {
            float f[V];
            factors<V>(a, d0, f);
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][e] = x[c][e] * rstd * f[e];
        }
        if constexpr (E4M3) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (d0 + e < a.D) top = max(top, magnitude(x[c][e]));
        } else {
            store_part<T, V>((T*)a.y + n * a.sy, d0, a.D, x[c]);
        }
    }
    if constexpr (E4M3) {
        const float scale = e4m3_scale(row_max<WPR>(top, s2));
        const E4m3Divisor by(scale);
        if (t == 0) a.scale[n] = scale;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t d0 = (int64_t)(c * TPR + t) * V;
            if (d0 >= a.D) break;
            by.divide<V>(x[c]);
            e4m3_store<V>((uint8_t*)a.y + n * a.sy + d0, a.D - d0, x[c]);
        }
    }
}

// Rows too long for registers: one workgroup reads the row once per sum or
// maximum and once to write; each thread reads again what it has read before (or
// stored: the total may lie where x or the residual did).
constexpr int kLongThreads = 1024, kLongWaves = 16;
template <typename T, bool E4M3> __global__ __launch_bounds__(kLongThreads) void rms_fwd_long(RmsNormArgs a) {
    constexpr int V = kVec<T>, STEP = kLongThreads * V;
    __shared__ float s1[kLongWaves];
    __shared__ uint32_t s2[kLongWaves];
    const int64_t n = blockIdx.x, first = (int64_t)threadIdx.x * V;
    float sum = 0.f;
    for (int64_t d0 = first; d0 < a.D; d0 += STEP) {
        float x[V];
        stream<T, V>(a, n, d0, x);
        if (a.r) store_part<T, V>((T*)a.total + n * a.st, d0, a.D, x);
        sum += squares<V>(x);
    }
    const T* s = a.r ? (const T*)a.total + n * a.st : (const T*)a.x + n * a.sx;
    float rstd = 1.f;
    if (!E4M3 || a.norm) {
        rstd = 1.0f / sqrtf(row_sum<kLongWaves>(sum, s1) / (float)a.D + a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[n] = rstd;
    }
    auto values = [&](int64_t d0, float* x) {
        load_part<T, V>(s, d0, a.D, x);
        if (E4M3 && !a.norm) return;
        float f[V];
        factors<V>(a, d0, f);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = x[e] * rstd * f[e];
    };
    float scale = 1.f;
    if constexpr (E4M3) {
        uint32_t top = 0;
        for (int64_t d0 = first; d0 < a.D; d0 += STEP) {
            float x[V];
            values(d0, x);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (d0 + e < a.D) top = max(top, magnitude(x[e]));
        }
        scale = e4m3_scale(row_max<kLongWaves>(top, s2));
        if (threadIdx.x == 0) a.scale[n] = scale;
    }
    const E4m3Divisor by(scale);
    for (int64_t d0 = first; d0 < a.D; d0 += STEP) {
        float x[V];
        values(d0, x);
        if constexpr (E4M3) {
            by.divide<V>(x);
            e4m3_store<V>((uint8_t*)a.y + n * a.sy + d0, a.D - d0, x);
        } else {
            store_part<T, V>((T*)a.y + n * a.sy, d0, a.D, x);
        }
    }
}

// Waves of a backward workgroup: eight rows at once, or one row's waves.
template <int WPR> constexpr int kBwdThreads = WPR == 1 ? 512 : 64 * WPR;

// Workgroup g: rows in steps of groups * (rows a workgroup holds at once).  EVEN:
// D is a multiple of the vector, so that no element is looked at by itself.  A row
// stays in T between its two passes, over the sum and to dx: 16384 x 1152 in bf16 with
// the stream's gradient 34 us (4.4 TB/s); held as fp32 numbers, whose registers leave
// eight waves to a CU, it took 56.
template <typename T, int WPR, int CH, bool PARAMS, bool EVEN>
__global__ __launch_bounds__(kBwdThreads<WPR>, WPR == 4 ? 2 : 4) void rms_bwd(RmsNormArgs a) {
    constexpr int V = kVec<T>, TPR = 64 * WPR, NT = kBwdThreads<WPR>, RPB = NT / TPR;
    typedef typename AnyVec<T, V>::raw raw;
    __shared__ __attribute__((aligned(16))) float lds[PARAMS && RPB > 1 ? RPB / 2 * CH * V * 64 : 1];
    __shared__ float s[2][WPR];
    const int t = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.D;
    // Elements from d0 on, 0 past the row's end (and with it all below).
    auto load = [&](const T* row, int64_t d0) {
        raw x{};
        if (d0 + (EVEN ? 0 : V - 1) < a.D) {
            x = AnyVec<T, V>::load_raw(row + d0);
        } else if (!EVEN) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (d0 + e < a.D) x[e] = row[d0 + e];
        }
        return x;
    };
    float dw[CH][V], f[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        factors<V>(a, (int64_t)(c * TPR + t) * V, f[c]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[c][e] = 0.f;
    }
    int turn = 0;
    for (int64_t n = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; n < a.N; n += a.groups * RPB) {
        raw x[CH], g[CH], d[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t d0 = (int64_t)(c * TPR + t) * V;
            x[c] = load((const T*)a.x + n * a.sx, d0);
            g[c] = load((const T*)a.dy + n * a.sdy, d0);
            d[c] = a.dt ? load((const T*)a.dt + n * a.sdt, d0) : raw{};
        }
        const float rstd = a.rstd_in[n];
        float c2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float h = (float)x[c][e] * rstd, gh = (float)g[c][e] * h;
                if constexpr (PARAMS) dw[c][e] += gh;
                c2 = fmaf(gh, f[c][e], c2);
            }
        if (a.dx) {
            c2 = row_sum<WPR>(c2, s[turn]) * inv;
            turn ^= 1;
            T* dr = (T*)a.dx + n * a.sdx;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t d0 = (int64_t)(c * TPR + t) * V;
                if (d0 >= a.D) break;
                asm volatile("" : "+v"(x[c]), "+v"(g[c]));  // T's registers, not fp32's, from the first pass on
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    o[e] = rstd * ((float)g[c][e] * f[c][e] - (float)x[c][e] * rstd * c2);
                    if (a.dt) o[e] += (float)d[c][e];
                }
                if constexpr (EVEN) AnyVec<T, V>::store(dr + d0, o);
                else store_part<T, V>(dr, d0, a.D, o);
            }
        }
    }
    if constexpr (PARAMS) {
        float* out = a.part + (int64_t)blockIdx.x * a.D;
        if constexpr (RPB > 1) {
            // The waves' sums meet in pairs, half of the waves handing theirs over at a time: quads of
            // columns, lane by lane, so that no bank is met twice.
            constexpr int QUADS = CH * V / 4, SLOT = QUADS * 64 * 4;  // floats of a wave
            const int wave = threadIdx.x / 64;
#pragma unroll
            for (int half = RPB / 2; half > 0; half /= 2) {
                if (wave >= half && wave < 2 * half)
#pragma unroll
                    for (int q = 0; q < QUADS; ++q) {
                        const float* d = &dw[0][0] + 4 * q;
                        *reinterpret_cast<f32x4*>(lds + (wave - half) * SLOT + (q * 64 + t) * 4) =
                            f32x4{d[0], d[1], d[2], d[3]};
                    }
                __syncthreads();
                if (wave < half)
#pragma unroll
                    for (int q = 0; q < QUADS; ++q) {
                        const f32x4 o = *reinterpret_cast<const f32x4*>(lds + wave * SLOT + (q * 64 + t) * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) (&dw[0][0])[4 * q + e] += o[e];
                    }
                __syncthreads();
            }
            if (wave != 0) return;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t d0 = (int64_t)(c * TPR + t) * V;
            if (d0 < a.D) store_part<float, V>(out, d0, a.D, dw[c]);
        }
    }
}

// Rows too long for registers: their sum, then dx and the partials of dw by columns.
template <typename T> __global__ __launch_bounds__(kLongThreads) void rms_bwd_sums(RmsNormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s[kLongWaves];
    const int64_t n = blockIdx.x;
    const float rstd = a.rstd_in[n];
    float c2 = 0.f;
    for (int64_t d0 = (int64_t)threadIdx.x * V; d0 < a.D; d0 += kLongThreads * V) {
        float x[V], g[V], f[V], p = 0.f;
        load_part<T, V>((const T*)a.x + n * a.sx, d0, a.D, x);
        load_part<T, V>((const T*)a.dy + n * a.sdy, d0, a.D, g);
        factors<V>(a, d0, f);
#pragma unroll
        for (int e = 0; e < V; ++e) p = fmaf(g[e] * f[e], x[e] * rstd, p);
        c2 += p;
    }
    c2 = row_sum<kLongWaves>(c2, s);
    if (threadIdx.x == 0) a.sums[n] = c2;
}

template <typename T> __global__ __launch_bounds__(256) void rms_bwd_columns(RmsNormArgs a) {
    const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (d >= a.D) return;
    const float inv = 1.0f / (float)a.D, f = a.w ? a.w[d] + a.one : 1.f;
    float dw = 0.f;
#pragma unroll 4
    for (int64_t n = blockIdx.y; n < a.N; n += a.groups) {
        const float rstd = a.rstd_in[n], h = (float)((const T*)a.x)[n * a.sx + d] * rstd;
        const float g = (float)((const T*)a.dy)[n * a.sdy + d];
        dw = fmaf(g, h, dw);
        if (a.dx) {
            float dx = rstd * (g * f - h * (a.sums[n] * inv));
            if (a.dt) dx += (float)((const T*)a.dt)[n * a.sdt + d];
            ((T*)a.dx)[n * a.sdx + d] = (T)dx;
        }
    }
    if (a.part) a.part[(int64_t)blockIdx.y * a.D + d] = dw;
}

// dw from column `first` on: the groups' partials in order.  32 columns (a line) to a
// workgroup; its 32 rows of threads take the groups in turn.
__global__ __launch_bounds__(1024) void rms_params(RmsNormArgs a, int64_t first) {
    __shared__ float s[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t c = first + (int64_t)blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < a.D)
#pragma unroll 8
        for (int64_t g = y; g < a.groups; g += 32) v += a.part[g * a.D + c];
    s[y][x] = v;
    __syncthreads();
    if (y != 0 || c >= a.D) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][x];
    a.dw[c] = v;
}

__global__ __launch_bounds__(256) void rms_zero_params(RmsNormArgs a) {
    const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (d < a.D) a.dw[d] = 0.f;
}

// Waves to a row and 16-byte chunks to a thread.  WPR 0: by memory.
struct Shape {
    int wpr, ch;
};
Shape fwd_shape(int64_t D, int vec) {
    for (const Shape s : {Shape{1, 1}, {1, 2}, {1, 3}, {1, 4}, {4, 2}, {4, 4}, {16, 2}, {16, 4}})
        if (D <= (int64_t)64 * s.wpr * s.ch * vec) return s;
    return {0, 0};
}
Shape bwd_shape(int64_t D, int vec) {
    for (const Shape s : {Shape{1, 1}, {1, 2}, {1, 3}, {4, 2}, {16, 1}, {16, 2}})
        if (D <= (int64_t)64 * s.wpr * s.ch * vec) return s;
    return {0, 0};
}
// Workgroups of the backward, each of which leaves a partial.  One to a CU, or two of
// four waves from eight rows a CU on: 4096 x 1152 in fp32 23 us (one: 27, four: 22), 8192 x
// 2304 in bf16 40 (52, 38), while 1001 x 1153 in fp32 waits for the host either way; of eight
// waves a row each, 16384 x 1152 in bf16 36 (two: 37, four: 39), of sixteen, 2048 x 8192
// 33 (37, 43).  Calls over operands out of cache, with dtotal.
int64_t bwd_groups(int64_t N, int64_t D, int vec) {
    const Shape s = bwd_shape(D, vec);
    const int64_t at_once = s.wpr == 1 ? 8 : 1, cus = device_cus();
    return std::max<int64_t>(1, std::min<int64_t>((N + at_once - 1) / at_once, (s.wpr == 4 && N >= 8 * cus ? 2 : 1) * cus));
}
size_t up(size_t x) { return (x + 255) & ~size_t(255); }

// f(first row, rows) for as many rows at a time as a launch's 2^32 threads allow.
template <typename F> void row_slices(int64_t N, int wpr, F f) {
    const int64_t most = (int64_t(1) << 31) / (64 * (wpr ? wpr : kLongWaves));
    for (int64_t n = 0; n < N; n += most) f(n, std::min(most, N - n));
}

template <typename T, bool E4M3> void fwd_rows(const RmsNormArgs& a, const Shape& s, hipStream_t st) {
    const dim3 grid((unsigned)(s.wpr == 1 ? (a.N + 3) / 4 : a.N));
#define MFT_RMS_FWD(WPR, CH)        \
    if (s.wpr == WPR && s.ch == CH) \
    hipLaunchKernelGGL((rms_fwd<T, WPR, CH, E4M3>), grid, dim3(kThreads<WPR>), 0, st, a)
    MFT_RMS_FWD(1, 1);
    MFT_RMS_FWD(1, 2);
    MFT_RMS_FWD(1, 3);
    MFT_RMS_FWD(1, 4);
    MFT_RMS_FWD(4, 2);
    MFT_RMS_FWD(4, 4);
    MFT_RMS_FWD(16, 2);
    MFT_RMS_FWD(16, 4);
#undef MFT_RMS_FWD
    if (s.wpr == 0) hipLaunchKernelGGL((rms_fwd_long<T, E4M3>), grid, dim3(kLongThreads), 0, st, a);
}
template <typename T, bool E4M3> hipError_t fwd(const RmsNormArgs& a, hipStream_t st) {
    const Shape s = fwd_shape(a.D, kVec<T>);
    row_slices(a.N, s.wpr, [&](int64_t n, int64_t rows) {
        RmsNormArgs q = a;
        q.N = rows;
        q.x = (const T*)a.x + n * a.sx;
        if (a.r) q.r = (const T*)a.r + n * a.sr, q.total = (T*)a.total + n * a.st;
        q.y = (char*)a.y + n * a.sy * (E4M3 ? 1 : (int64_t)sizeof(T));
        if (a.rstd) q.rstd = a.rstd + n;
        if (a.scale) q.scale = a.scale + n;
        fwd_rows<T, E4M3>(q, s, st);
    });
    return hipGetLastError();
}

template <typename T> hipError_t bwd(const RmsNormArgs& a, hipStream_t st) {
    const Shape s = bwd_shape(a.D, kVec<T>);
    const bool params = a.dw != nullptr;
    if (s.wpr == 0) {
        RmsNormArgs q = a;
        if (!params) q.part = nullptr;
        if (a.dx) {
            row_slices(a.N, 0, [&](int64_t n, int64_t rows) {
                RmsNormArgs r = a;
                r.x = (const T*)a.x + n * a.sx;
                r.dy = (const T*)a.dy + n * a.sdy;
                r.rstd_in = a.rstd_in + n;
                r.sums = a.sums + n;
                hipLaunchKernelGGL((rms_bwd_sums<T>), dim3((unsigned)rows), dim3(kLongThreads), 0, st, r);
            });
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL((rms_bwd_columns<T>), dim3((unsigned)((a.D + 255) / 256), (unsigned)a.groups), dim3(256), 0,
                           st, q);
    }
#define MFT_RMS_BWD_E(WPR, CH, PARAMS)                                                                          \
    do {                                                                                                        \
        if (a.D % kVec<T> == 0)                                                                                 \
            hipLaunchKernelGGL((rms_bwd<T, WPR, CH, PARAMS, true>), grid, dim3(kBwdThreads<WPR>), 0, st, a);    \
        else                                                                                                    \
            hipLaunchKernelGGL((rms_bwd<T, WPR, CH, PARAMS, false>), grid, dim3(kBwdThreads<WPR>), 0, st, a);   \
    } while (0)
#define MFT_RMS_BWD(WPR, CH)                     \
    if (s.wpr == WPR && s.ch == CH) {            \
        if (params) MFT_RMS_BWD_E(WPR, CH, true); \
        else MFT_RMS_BWD_E(WPR, CH, false);      \
    }
    const dim3 grid((unsigned)a.groups);
    MFT_RMS_BWD(1, 1)
    MFT_RMS_BWD(1, 2)
    MFT_RMS_BWD(1, 3)
    MFT_RMS_BWD(4, 2)
    MFT_RMS_BWD(16, 1)
    MFT_RMS_BWD(16, 2)
#undef MFT_RMS_BWD_E
#undef MFT_RMS_BWD
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !params) return e;
    // 32 threads to a column, and fewer than 2^32 to a launch: 2^26 columns at a time
    constexpr int64_t kMost = int64_t(1) << 26;
    for (int64_t c = 0; c < a.D; c += kMost)
        hipLaunchKernelGGL(rms_params, dim3((unsigned)((std::min(kMost, a.D - c) + 31) / 32)), dim3(1024), 0, st, a, c);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm_fwd(const RmsNormArgs& a, bool is_bf16, hipStream_t st) {
    if (a.N == 0) return hipSuccess;
    if (a.scale) return is_bf16 ? fwd<bf16, true>(a, st) : fwd<float, true>(a, st);
    return is_bf16 ? fwd<bf16, false>(a, st) : fwd<float, false>(a, st);
}

size_t rms_norm_workspace(int64_t N, int64_t D, bool is_bf16) {
    const int vec = is_bf16 ? kVec<bf16> : kVec<float>;
    size_t n = up((size_t)bwd_groups(N, D, vec) * D * 4);
    if (bwd_shape(D, vec).wpr == 0) n += up((size_t)N * 4);
    return n;
}

hipError_t launch_rms_norm_bwd(RmsNormArgs a, bool is_bf16, void* workspace, hipStream_t st) {
    if (a.N == 0) {
        if (!a.dw) return hipSuccess;
        hipLaunchKernelGGL(rms_zero_params, dim3((unsigned)((a.D + 255) / 256)), dim3(256), 0, st, a);
        return hipGetLastError();
    }
    if (!a.dx && !a.dw) return hipSuccess;
    const int vec = is_bf16 ? kVec<bf16> : kVec<float>;
    a.groups = bwd_groups(a.N, a.D, vec);
    a.part = static_cast<float*>(workspace);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + up((size_t)a.groups * a.D * 4));
    return is_bf16 ? bwd<bf16>(a, st) : bwd<float>(a, st);
}

}  // namespace mft
