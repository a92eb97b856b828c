// The gated linear layer's bf16 products (C ABI in include/mft/gated_linear.h) on
// the tiles of bf_gemm_tiles.h: gate and up in one kernel with act(gate) up in its
// epilogue, and the backward's dx = dgate W_gate^T + dup W_up^T as one product along
// both.  Which tile a product takes, and its launches.
#include "bf_gemm_tiles.h"

namespace mft {
namespace {

// The slices' partial sums of gate and up in their order, then the epilogue.
__global__ __launch_bounds__(256) void gated_reduce(Args a) {
    const int64_t cols = (a.g.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / cols, n = (i - m * cols) * 4;
    if (m >= a.g.M) return;
    float v[2][4] = {};
#pragma unroll 4
    for (int s = 0; s < a.slices; ++s)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float p[4];
            load_part<float, 4>(a.g.partial + (((int64_t)s * 2 + q) * a.g.M + m) * a.g.N, n, a.g.N, p);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] += p[e];
        }
    gated_epilogue<bf16, 4>(a.g, m, n, v[0], v[1]);
}
__global__ __launch_bounds__(256) void joined_reduce(Args a) {
    const int64_t cols = (a.g.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / cols, n = (i - m * cols) * 4;
    if (m >= a.g.M) return;
    float v[4] = {};
#pragma unroll 4
    for (int s = 0; s < a.slices; ++s) {
        float p[4];
        load_part<float, 4>(a.g.partial + ((int64_t)s * a.g.M + m) * a.g.N, n, a.g.N, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
    store_part<bf16, 4>((bf16*)a.g.C + m * a.g.N, n, a.g.N, v);
}

struct Plan {
    int shape;
    Args a;
};

// The tiles (columns of both sums together), and what each sustains over the whole
// GPU (TFLOP/s) with one workgroup to a CU and with more, and the k that its prologue
// and epilogue are worth (`act` of a gated tile: three outputs and the activation).
// Fitted to five (GATED) and four (JOINED) pairs of widths from 640 to 8192 and 16
// to 8192 rows, each timed in every tile and cut into 1 to 12 slices: the choice by
// these is within 6 percent of the fastest in 74 of 86 (10 in 82; 1.29 times it in one)
// and in 60 of 64 (10 in 63).
//   256 x 256, one wave to a SIMD: 8192 x 1152 -> 6912, both sums kept, 267 us, W [in,
//     ff] 268; 256 x 128 275, 128 x 128 320, the deep 256 x 128 340.  Its products
//     alone are 183 (1430 TFLOP/s, what the card's power allows); the rest is a
//     tile's beginning and its epilogue, which nothing hides.  Tiles of 128 x 192, two
//     workgroups to a CU, hide it but read LDS more: 280, and 92 for 97 without the sums
//     kept at K 640.
//   deep, and 128 x 64: few tiles.  512 rows of it 25 us in the deep 256 x 128, 33 in
//     256 x 256; 64 rows 13 us in the deep 128 x 128, 26.
struct Shape {
    int bn, bm, deep;
    double one, more;
    int k, act;
};
constexpr int kShapeCount = 6;
constexpr Shape kGated[kShapeCount] = {{256, 128, 0, 880, 1360, 200, 270}, {128, 128, 0, 970, 1120, 220, 250},
                                       {128, 64, 0, 580, 780, 180, 80},    {256, 256, 0, 1460, 1480, 370, 200},
                                       {128, 128, 1, 1330, 1010, 350, 80}, {256, 128, 1, 1440, 1520, 580, 420}};
constexpr Shape kJoined[kShapeCount] = {{256, 128, 0, 890, 1180, 140, 0}, {128, 128, 0, 880, 1000, 490, 0},
                                        {128, 64, 0, 490, 780, 170, 0},   {256, 256, 0, 1520, 1400, 430, 0},
                                        {128, 128, 1, 1210, 1000, 390, 0}, {256, 128, 1, 1250, 1520, 710, 0}};
// A second launch, and the partials written and read (bytes a us).
constexpr double kKcGated = 1.07, kKcJoined = 1.15, kCutGated = 3.9, kCutJoined = 1.0, kCutRate = 4.3e6, kCutRateJoined = 3e6;
// With k contiguous in both operands the slabs of 256 x 128 do not leave a CU room
// for two; 64 rows of a deep slab are not whole rows of its eight waves' loads without.
bool has_shape(const LinearProduct& g, int s, bool gated) {
    return s == 0 ? !g.q_kc : s == 4 ? !gated || g.q_kc : true;
}

Plan plan(const LinearProduct& g, bool gated) {
    Plan p{};
    const int cus = device_cus(), pairs = (int)(g.K / kSlab), nq = gated ? 2 : 1;
    double best = 1e300;
    int per = 1;
    for (int s = 0; s < kShapeCount; ++s) {
        if (!has_shape(g, s, gated)) continue;
        const Shape& t = (gated ? kGated : kJoined)[s];
        const int64_t tiles = ((g.N * nq + t.bn - 1) / t.bn) * ((g.M + t.bm - 1) / t.bm);
        for (int slices : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (slices > 1 && (slices > pairs || tiles * slices > 4 * cus)) break;
            const int per_slice = std::max(1, (pairs + slices - 1) / slices), n = std::max(1, (pairs + per_slice - 1) / per_slice);
            const double mean = (double)tiles * n / cus, most = std::ceil(mean);
            const double rate = (most <= 1 ? t.one : t.more) * (g.q_kc ? (gated ? kKcGated : kKcJoined) : 1.0) * cus / 256;
            double us = (most <= 1 ? 1 : t.deep ? most : (most + mean) / 2) * cus * t.bn * t.bm * 2 *
                        ((double)g.K / n + t.k + (n == 1 ? t.act : 0)) / rate / 1e6;
            if (n > 1) us += (gated ? kCutGated : kCutJoined) + (double)n * g.M * g.N * nq * 8 / (gated ? kCutRate : kCutRateJoined);
            if (us < best * 0.999) best = us, p.shape = s, per = per_slice;
        }
    }
    const Shape& t = (gated ? kGated : kJoined)[p.shape];
    p.a.g = g;
    p.a.tiles_m = (int)((g.M + t.bm - 1) / t.bm);
    p.a.tiles_n = (int)((g.N * nq + t.bn - 1) / t.bn);
    p.a.halves = 2 * pairs;
    p.a.per_slice = 2 * per;
    p.a.slices = std::max(1, (pairs + per - 1) / per);
    p.a.whole = p.a.slices == 1;
    p.a.per_slice_tiles = FastDiv::make((uint32_t)(p.a.tiles_m * p.a.tiles_n));
    return p;
}

template <int BN, int BM, bool QKC, int MODE> void launch_t(const Args& a, bool dma, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices));
    if (dma || MODE == JOINED)
        hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, true, QKC, true, ACT_NONE, MODE>), grid, dim3(kThreads), 0, st, a);
    else if constexpr (MODE != JOINED)
        hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, true, QKC, false, ACT_NONE, MODE>), grid, dim3(kThreads), 0, st, a);
}
template <int BN, bool QKC, int MODE> void launch_deep(const Args& a, bool dma, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices));
    if (dma || MODE == JOINED)
        hipLaunchKernelGGL((bf_gemm_deep<BN, 128, true, QKC, true, ACT_NONE, MODE>), grid, dim3(kDeepThreads), 0, st, a);
    else if constexpr (MODE != JOINED)
        hipLaunchKernelGGL((bf_gemm_deep<BN, 128, true, QKC, false, ACT_NONE, MODE>), grid, dim3(kDeepThreads), 0, st, a);
}
template <bool QKC, int MODE> void launch_s(const Plan& p, bool dma, hipStream_t st) {
    if constexpr (!QKC) {
        if (p.shape == 0) launch_t<256, 128, QKC, MODE>(p.a, dma, st);
    }
    if (p.shape == 1) launch_t<128, 128, QKC, MODE>(p.a, dma, st);
    if (p.shape == 2) launch_t<128, 64, QKC, MODE>(p.a, dma, st);
    if (p.shape == 3) launch_t<256, 256, QKC, MODE>(p.a, dma, st);
    if constexpr (QKC || MODE != GATED) {
        if (p.shape == 4) launch_deep<128, QKC, MODE>(p.a, dma, st);
    }
    if (p.shape == 5) launch_deep<256, QKC, MODE>(p.a, dma, st);
}

// Operands off 16 bytes are copied to whole rows where the product is worth up to
// three launches, as the linear layer's are (linear_gemm.hip has the figures).
constexpr double kPackWorth = 4e8, kPackWorthKc = 2e9;
struct Packs {
    bool p, q;
    int64_t rows_q, cols_q;
    size_t at_p, at_q, at_q2, total;
};
Packs packs(const LinearProduct& g, const Plan& plan) {
    Packs k{};
    k.rows_q = g.q_kc ? g.N : g.K, k.cols_q = g.q_kc ? g.K : g.N;
    const bool off_p = g.K % 8 != 0, off_q = k.cols_q % 8 != 0;
    const bool worth = 2.0 * g.M * g.N * g.K >= (off_q && !g.q_kc ? kPackWorth : kPackWorthKc);
    k.p = worth && off_p;
    k.q = worth && off_q;
    size_t o = plan.a.whole ? 0 : up((size_t)plan.a.slices * 2 * g.M * g.N * 4);
    k.at_p = o, o += k.p ? up((size_t)g.M * whole_ld(g.K) * 2) : 0;
    const size_t q = k.q ? up((size_t)k.rows_q * whole_ld(k.cols_q) * 2) : 0;
    k.at_q = o, o += q;
    k.at_q2 = o, o += q;
    k.total = o;
    return k;
}

// A product joined along k needs whole slabs of either part, and rows on 16 bytes;
// else both parts of Q are first copied behind one another.
bool joins(const LinearProduct& g) {
    return g.joint % kSlab == 0 && (g.q_kc || g.N % 8 == 0) && on16(g.Q) && on16(g.Q2) && g.ldp <= (1 << 22) &&
           (g.q_kc || g.N <= (1 << 22));
}
LinearProduct whole_product(const LinearProduct& g) {
    LinearProduct w = g;
    w.joint = 0;
    w.Q2 = nullptr;
    w.ldq = g.q_kc ? 2 * whole_ld(g.joint) : whole_ld(g.N);
    w.K = 2 * whole_ld(g.joint);
    return w;
}
size_t whole_bytes(const LinearProduct& g) {
    return up((g.q_kc ? (size_t)g.N * 2 * whole_ld(g.joint) : 2 * (size_t)whole_ld(g.joint) * whole_ld(g.N)) * 2);
}
// Q and Q2 behind one another along k, `joint` k each padded with zeros to whole ones.
__global__ __launch_bounds__(256) void join_q(const bf16* q, const bf16* q2, bf16* to, int64_t rows, int64_t cols,
                                              int64_t padded_rows, int64_t ld, int64_t second) {
    const int64_t chunks = ld / 8, n = padded_rows * chunks, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += step) {
        const int64_t j = i >= n ? i - n : i, r = j / chunks, c = (j - r * chunks) * 8;
        float v[8] = {};
        if (r < rows) load_part<bf16, 8>((i >= n ? q2 : q) + r * cols, c, cols, v);
        // along a row (second < ld of the whole), or below all rows
        AnyVec<bf16, 8>::store(to + (i >= n ? second : 0) + r * (second == ld ? 2 * ld : ld) + c, v);
    }
}

}  // namespace

size_t gated_gemm_workspace(const LinearProduct& g) { return packs(g, plan(g, true)).total; }

hipError_t launch_gated_gemm(const LinearProduct& given, hipStream_t st) {
    LinearProduct g = given;
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    Plan p = plan(g, true);
    const Packs k = packs(g, p);
    g.ldp = g.K;
    g.ldq = k.cols_q;
    char* ws = reinterpret_cast<char*>(g.partial);
    if (k.p) {
        const hipError_t e = pack(g.P, ws + k.at_p, g.M, g.K, st);
        if (e != hipSuccess) return e;
        g.P = ws + k.at_p, g.ldp = whole_ld(g.K);
    }
    if (k.q) {
        hipError_t e = pack(g.Q, ws + k.at_q, k.rows_q, k.cols_q, st);
        if (e == hipSuccess) e = pack(g.Q2, ws + k.at_q2, k.rows_q, k.cols_q, st);
        if (e != hipSuccess) return e;
        g.Q = ws + k.at_q, g.Q2 = ws + k.at_q2, g.ldq = whole_ld(k.cols_q);
    }
    p.a.g = g;
    // direct loads take 16 bytes whole, also at the end of a row
    const bool dma = g.ldp % 8 == 0 && g.ldq % 8 == 0 && on16(g.P) && on16(g.Q) && on16(g.Q2) && g.ldp <= (1 << 22) &&
                     g.ldq <= (1 << 22);
    if (g.q_kc) launch_s<true, GATED>(p, dma, st);
    else launch_s<false, GATED>(p, dma, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.a.whole) return e;
    const int64_t n = g.M * ((g.N + 3) / 4);
    hipLaunchKernelGGL(gated_reduce, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p.a);
    return hipGetLastError();
}

size_t joined_gemm_workspace(const LinearProduct& g) {
    const Plan p = plan(g, false);
    const size_t sums = p.a.whole ? 0 : up((size_t)p.a.slices * g.M * g.N * 4);
    return std::max(sums, whole_bytes(g) + bf_gemm_workspace(whole_product(g)));
}

hipError_t launch_joined_gemm(const LinearProduct& g, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    char* ws = reinterpret_cast<char*>(g.partial);
    if (!joins(g)) {
        LinearProduct w = whole_product(g);
        const int64_t rows = g.q_kc ? g.N : g.joint, cols = g.q_kc ? g.joint : g.N, ld = whole_ld(cols);
        const int64_t padded = g.q_kc ? rows : whole_ld(rows), n = 2 * padded * (ld / 8);
        hipLaunchKernelGGL(join_q, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 16 * device_cus())), dim3(256), 0, st,
                           (const bf16*)g.Q, (const bf16*)g.Q2, (bf16*)ws, rows, cols, padded, ld,
                           g.q_kc ? ld : padded * ld);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        w.Q = ws;
        w.partial = reinterpret_cast<float*>(ws + whole_bytes(g));
        return launch_bf_gemm(w, st);
    }
    LinearProduct q = g;
    q.ldq = g.q_kc ? g.joint : g.N;
    Plan p = plan(q, false);
    if (q.q_kc) launch_s<true, JOINED>(p, true, st);
    else launch_s<false, JOINED>(p, true, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.a.whole) return e;
    const int64_t n = q.M * ((q.N + 3) / 4);
    hipLaunchKernelGGL(joined_reduce, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p.a);
    return hipGetLastError();
}

}  // namespace mft
