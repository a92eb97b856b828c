// The linear layer's bf16 products (C ABI in include/mft/linear.h) on the tiles of
// bf_gemm_tiles.h: which of them a product takes, and its launches.
#include "bf_gemm_tiles.h"

namespace mft {
namespace {

// The slices' partial products in their order, then the epilogue.
template <int ACT> __global__ __launch_bounds__(256) void bf_gemm_reduce(Args a) {
    const int64_t cols = (a.g.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / cols, n = (i - m * cols) * 4;
    if (m >= a.g.M) return;
    float v[4];
    load_part<float, 4>(a.g.partial + m * a.g.N, n, a.g.N, v);
#pragma unroll 4
    for (int s = 1; s < a.slices; ++s) {
        float p[4];
        load_part<float, 4>(a.g.partial + ((int64_t)s * a.g.M + m) * a.g.N, n, a.g.N, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
    linear_epilogue<bf16, ACT, 4>(a.g, m, n, v);
}

struct Plan {
    int shape;
    Args a;
};

// The tiles, and what each sustains over the whole GPU (TFLOP/s) with one
// workgroup to a CU and with more, and the k that its prologue and epilogue are
// worth (with an activation: `act` more).  Fitted to products of 16 to 8192 rows
// and 600 to 6912 columns, each timed on operands out of cache in every tile and
// cut into 1 to 16 slices: of 54 the choice by these is the fastest or within 6
// percent of it in 49, within 8 in 53, and 1.16 times it in one.
//   256 x 128, two workgroups to a CU: heavy epilogues over short K.  8192 x 1024
//     -> 4096 with GELU 88 us, 256 x 256 97, 128 x 128 104.
//   256 x 256, one wave to a SIMD with its accumulators in all of its registers:
//     least LDS and L2 traffic per product.  8192^3 844 us (1300 TFLOP/s), 256 x
//     128 923, 128 x 128 1025; W [out, in] 808, 128 x 128 946.
//   deep: 8192 x 1024 -> 4096's dW (256 tiles of 128 x 128 over K 8192) 78 us, 113
//     with one workgroup of 4 waves to a CU; its dx in 256 x 128 63 us for 74 in
//     128 x 128; 4096 x 6912 -> 1152 in 192 x 128 79 us (with a residual 85) for 98.
// With k contiguous in both operands the slabs of 256 x 128 do not leave a CU
// room for two; a slab of 192 rows has no whole direct loads without.
struct Shape {
    int bn, bm, deep;
    double one, more;
    int k, act;
};
constexpr Shape kShapes[] = {{256, 128, 0, 1000, 1350, 330, 190}, {128, 128, 0, 900, 1080, 345, 190},
                             {64, 64, 0, 400, 720, 200, 100},     {256, 256, 0, 1400, 1540, 704, 200},
                             {128, 128, 1, 1200, 1200, 380, 190}, {192, 128, 1, 1200, 1260, 345, 190},
                             {256, 128, 1, 1520, 1200, 380, 190}};
constexpr int kShapeCount = sizeof(kShapes) / sizeof(kShapes[0]);
bool has_shape(const LinearProduct& g, int s) {
    return s == 0 ? g.p_kc && !g.q_kc : s == 5 ? g.q_kc != 0 : true;
}

Plan plan(const LinearProduct& g) {
    Plan p{};
    const int cus = device_cus(), pairs = (int)(g.K / kSlab);
    double best = 1e300;
    int per = 1;
    for (int s = 0; s < kShapeCount; ++s) {
        if (!has_shape(g, s)) continue;
        const Shape& t = kShapes[s];
        const int64_t tiles = ((g.N + t.bn - 1) / t.bn) * ((g.M + t.bm - 1) / t.bm);
        for (int slices : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (slices > 1 && (slices > pairs || tiles * slices > 4 * cus)) break;
            const int per_slice = std::max(1, (pairs + slices - 1) / slices), n = std::max(1, (pairs + per_slice - 1) / per_slice);
            const double mean = (double)tiles * n / cus, most = std::ceil(mean);
            const double rate = (most <= 1 ? t.one : t.more) * (g.p_kc && g.q_kc ? 1.08 : 1.0) * cus / 256;
            double us = (most <= 1 ? 1 : t.deep ? most : (most + mean) / 2) * cus * t.bn * t.bm * 2 *
                        ((double)g.K / n + t.k + (g.act != ACT_NONE && n == 1 ? t.act : 0)) / rate / 1e6;
            if (n > 1) us += 1 + (double)n * g.M * g.N * 8 / 5.4e6;  // partials written and read, a launch
            if (us < best * 0.999) best = us, p.shape = s, per = per_slice;
        }
    }
    const Shape& t = kShapes[p.shape];
    p.a.g = g;
    p.a.tiles_m = (int)((g.M + t.bm - 1) / t.bm);
    p.a.tiles_n = (int)((g.N + t.bn - 1) / t.bn);
    p.a.halves = 2 * pairs;
    p.a.per_slice = 2 * per;
    p.a.slices = std::max(1, (pairs + per - 1) / per);
    p.a.whole = p.a.slices == 1;
    p.a.per_slice_tiles = FastDiv::make((uint32_t)(p.a.tiles_m * p.a.tiles_n));
    return p;
}

template <int BN, int BM, bool PKC, bool QKC, int ACT> void launch_t(const Args& a, bool dma, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices));
    if (dma) hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, PKC, QKC, true, ACT>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, PKC, QKC, false, ACT>), grid, dim3(kThreads), 0, st, a);
}
template <int BN, bool PKC, bool QKC, int ACT> void launch_deep(const Args& a, bool dma, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices));
    if (dma) hipLaunchKernelGGL((bf_gemm_deep<BN, 128, PKC, QKC, true, ACT>), grid, dim3(kDeepThreads), 0, st, a);
    else hipLaunchKernelGGL((bf_gemm_deep<BN, 128, PKC, QKC, false, ACT>), grid, dim3(kDeepThreads), 0, st, a);
}
template <bool PKC, bool QKC, int ACT> void launch_s(const Plan& p, bool dma, hipStream_t st) {
    if constexpr (PKC && !QKC) {
        if (p.shape == 0) launch_t<256, 128, PKC, QKC, ACT>(p.a, dma, st);
    }
    if (p.shape == 1) launch_t<128, 128, PKC, QKC, ACT>(p.a, dma, st);
    if (p.shape == 2) launch_t<64, 64, PKC, QKC, ACT>(p.a, dma, st);
    if (p.shape == 3) launch_t<256, 256, PKC, QKC, ACT>(p.a, dma, st);
    if (p.shape == 4) launch_deep<128, PKC, QKC, ACT>(p.a, dma, st);
    if constexpr (QKC) {
        if (p.shape == 5) launch_deep<192, PKC, QKC, ACT>(p.a, dma, st);
    }
    if (p.shape == 6) launch_deep<256, PKC, QKC, ACT>(p.a, dma, st);
}
template <int ACT> void launch_act_fwd(const Plan& p, bool dma, hipStream_t st) {
    if (p.a.g.q_kc) launch_s<true, true, ACT>(p, dma, st);
    else launch_s<true, false, ACT>(p, dma, st);
}

// Operands whose rows are off 16 bytes are first copied to rows of whole ones,
// where the product (of M N K pairs of numbers) is worth up to two more launches.
// 47 sizes, each product copied and through the registers, on operands out of
// cache: from 4e8 on copies take 0.3 to 1.1 times as long in most (4e8 to 1e9,
// at most 1.5), 2000 x 1153 -> 2001 41 -> 26 us, its dW 67 -> 28; under 3e8 1.1 to
// 1.9 times in most, 120 x 900 -> 1100's dW 7 -> 11.  With k contiguous in the
// operands that are off the registers' way is less slow: 1.0 to 1.3 times from
// 1e9 to 2e9, 0.7 to 1.1 above.
constexpr double kPackWorth = 4e8, kPackWorthKc = 2e9;
struct Packs {
    bool p, q;
    int64_t rows_p, cols_p, rows_q, cols_q;
    size_t at_p, at_q, total;
};
Packs packs(const LinearProduct& g, const Plan& plan) {
    Packs k{};
    k.rows_p = g.p_kc ? g.M : g.K, k.cols_p = g.p_kc ? g.K : g.M;
    k.rows_q = g.q_kc ? g.N : g.K, k.cols_q = g.q_kc ? g.K : g.N;
    const bool off_p = k.cols_p % 8 != 0 && g.ldp == 0, off_q = k.cols_q % 8 != 0 && g.ldq == 0;
    const bool worth = (double)g.M * g.N * g.K >= ((off_p && !g.p_kc) || (off_q && !g.q_kc) ? kPackWorth : kPackWorthKc);
    k.p = worth && off_p;
    k.q = worth && off_q;
    size_t o = plan.a.whole ? 0 : up((size_t)plan.a.slices * g.M * g.N * 4);
    k.at_p = o, o += k.p ? up((size_t)k.rows_p * whole_ld(k.cols_p) * 2) : 0;
    k.at_q = o, o += k.q ? up((size_t)k.rows_q * whole_ld(k.cols_q) * 2) : 0;
    k.total = o;
    return k;
}

}  // namespace

size_t bf_gemm_workspace(const LinearProduct& g) { return packs(g, plan(g)).total; }

hipError_t launch_bf_gemm(const LinearProduct& given, hipStream_t st) {
    LinearProduct g = given;
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    Plan p = plan(g);
    const Packs k = packs(g, p);
    if (g.ldp == 0) g.ldp = k.cols_p;
    if (g.ldq == 0) g.ldq = k.cols_q;
    char* ws = reinterpret_cast<char*>(g.partial);
    if (k.p) {
        const hipError_t e = pack(g.P, ws + k.at_p, k.rows_p, k.cols_p, st);
        if (e != hipSuccess) return e;
        g.P = ws + k.at_p, g.ldp = whole_ld(k.cols_p);
    }
    if (k.q) {
        const hipError_t e = pack(g.Q, ws + k.at_q, k.rows_q, k.cols_q, st);
        if (e != hipSuccess) return e;
        g.Q = ws + k.at_q, g.ldq = whole_ld(k.cols_q);
    }
    p.a.g = g;
    const int64_t ldp = g.ldp, ldq = g.ldq;
    // direct loads take 16 bytes whole, also at the end of a row
    const bool dma = ldp % 8 == 0 && ldq % 8 == 0 && on16(g.P) && on16(g.Q) && ldp <= (1 << 22) && ldq <= (1 << 22);
    // an epilogue after the slices' sum is the reduce kernel's
    const int act = p.a.whole ? g.act : ACT_NONE;
    if (!g.p_kc) {
        if (g.q_kc || g.act != ACT_NONE) return hipErrorInvalidValue;
        launch_s<false, false, ACT_NONE>(p, dma, st);
    } else if (act == ACT_RELU) {
        launch_act_fwd<ACT_RELU>(p, dma, st);
    } else if (act == ACT_GELU_TANH) {
        launch_act_fwd<ACT_GELU_TANH>(p, dma, st);
    } else if (act == ACT_SILU) {
        launch_act_fwd<ACT_SILU>(p, dma, st);
    } else {
        launch_act_fwd<ACT_NONE>(p, dma, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.a.whole) return e;
    const int64_t n = g.M * ((g.N + 3) / 4);
    const dim3 grid((unsigned)((n + 255) / 256)), block(256);
    switch (g.act) {
        case ACT_RELU: hipLaunchKernelGGL((bf_gemm_reduce<ACT_RELU>), grid, block, 0, st, p.a); break;
        case ACT_GELU_TANH: hipLaunchKernelGGL((bf_gemm_reduce<ACT_GELU_TANH>), grid, block, 0, st, p.a); break;
        case ACT_SILU: hipLaunchKernelGGL((bf_gemm_reduce<ACT_SILU>), grid, block, 0, st, p.a); break;
        default: hipLaunchKernelGGL((bf_gemm_reduce<ACT_NONE>), grid, block, 0, st, p.a); break;
    }
    return hipGetLastError();
}

}  // namespace mft
