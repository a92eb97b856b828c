// The linear layer's bf16 products (C ABI in include/mft/linear.h):
// C[M, N] = act(sum_k P(m, k) Q(n, k) + bias[n]) + residual.
//
// A workgroup of 2 x 2 waves owns a BN x BM tile of C^T = Q P^T, on
// v_mfma_f32_32x32x16_bf16: Q's rows are the instruction's rows, so that a lane
// holds four consecutive columns n of one row m of C.  Either operand is stored
// with k contiguous (a tile is [rows][BK], fragments are 16-byte reads) or with
// its rows contiguous (a tile is [BK][rows], fragments are transposing reads).
// A stage of BK values of k comes by direct loads into LDS where all rows and
// bases lie on 16 bytes (DMA), the stage after next while one is multiplied;
// else, and for the last stage where BK does not divide K, through registers
// with zeros past the end.
//
// Products of few tiles cut K into slices whose fp32 partials a second launch
// adds in their order and takes through the epilogue.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_common.h"
#include "attn_geometry.h"
#include "attn_kernels.h"
#include "linear_act.h"
#include "linear_kernels.h"
#include "prologue_kernels.h"
#include "row_util.h"

namespace mft {
namespace {

constexpr int kThreads = 256;

struct Args {
    BfGemm g;
    int tiles_m, tiles_n, slices, stages, per_slice;
    int whole;  // one slice: the epilogue in the product's launch
    FastDiv per_slice_tiles;
};

// 16-byte chunk c of row r in a tile with k contiguous: 16 rows' reads of one
// chunk meet no bank twice.
template <int BK> __device__ __forceinline__ constexpr int swz_kc(int r) {
    return BK == 32 ? (r >> 2) & 3 : (r >> 1) & 7;
}

// One operand of R rows a tile: its loads and its fragments.
template <int R, int BK, bool KC> struct Operand {
    static constexpr int kBytes = R * BK * 2, PER = kBytes / 1024 / 4;  // 1 KiB loads of a wave
    static constexpr int ROW = KC ? BK : R, CPR = ROW / 8, RPL = 64 / CPR;  // LDS row, chunks of it, rows of a load
    static_assert(PER >= 1 && PER * 4096 == kBytes && RPL >= 1, "whole loads");
    // Tile row (KC: the operand's row, else k) and chunk of this lane's load j.
    __device__ __forceinline__ static int load_row(int w, int j, int lane) { return (w * PER + j) * RPL + lane / CPR; }
    __device__ __forceinline__ static int load_chunk(int row, int lane) {
        const int p = lane % CPR;
        return KC ? p ^ swz_kc<BK>(row) : p ^ swz_tr<CPR>(row);
    }
    // Direct loads: this lane's byte offsets from the tile's first element.
    uint32_t off[PER];
    __device__ __forceinline__ void init(int w, int lane, int64_t r0, int64_t rows, int64_t ld) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = load_row(w, j, lane), c = load_chunk(r, lane);
            if (KC)  // rows past the end are read again from the last one, and not stored
                off[j] = (uint32_t)((min(r0 + r, rows - 1) - r0) * ld * 2) + 16u * c;
            else
                off[j] = (uint32_t)(r * ld * 2) + (uint32_t)(min(r0 + 8 * c, rows - 8) - r0) * 2u;
        }
    }
    __device__ __forceinline__ void issue(const char* tile, uint32_t lds, int w) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) load_lds_16_s(tile, off[j], lds + (uint32_t)(w * PER + j) * 1024u);
    }
    // The same loads through registers, anywhere and with zeros past the ends.
    typedef bf16 any8 __attribute__((ext_vector_type(8), aligned(2)));
    __device__ __forceinline__ static bf16x8 fetch(const bf16* p, int64_t ld, int64_t r0, int64_t rows, int64_t k0,
                                                   int64_t K, int w, int j, int lane) {
        const int r = load_row(w, j, lane), c = load_chunk(r, lane);
        const int64_t row = KC ? min(r0 + r, rows - 1) : k0 + r;       // storage row
        const int64_t col = KC ? k0 + 8 * c : r0 + 8 * c, end = KC ? K : rows;
        bf16x8 v = zero_vec<bf16x8>();
        if (!KC && row >= K) return v;
        const bf16* q = p + row * ld + col;
        if (col + 8 <= end) {
            v = __builtin_bit_cast(bf16x8, *reinterpret_cast<const any8*>(q));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < end) v[e] = q[e];
        }
        return v;
    }
    __device__ __forceinline__ static void store(char* lds, int w, int j, int lane, bf16x8 v) {
        *reinterpret_cast<bf16x8*>(lds + (w * PER + j) * 1024 + lane * 16) = v;
    }
};

// Fragments of T 32-row tiles from row `first` on, k step ks of a stage.
template <int R, int BK, bool KC, int T> struct Fragments {
    uint32_t at[KC ? BK / 16 : T];
    __device__ __forceinline__ void init(int first, int lane) {
        const int n = lane & 31, hh = lane >> 5;
        if constexpr (KC) {
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks)
                at[ks] = (uint32_t)((first + n) * BK * 2 + ((2 * ks + hh) ^ swz_kc<BK>(n)) * 16);
        } else {
            const int j = lane & 15, k = 8 * hh + j / 4;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int col = first + 32 * t + 16 * (lane >> 4 & 1) + 4 * (j & 3);
                at[t] = (uint32_t)(k * R * 2 + ((col >> 3) ^ swz_tr<R / 8>(k)) * 16 + (col & 7) * 2);
            }
        }
    }
    __device__ __forceinline__ bf16x8 read(const char* lds, int ks, int t) const {
        if constexpr (KC) {
            return *reinterpret_cast<const bf16x8*>(lds + at[ks] + t * 32 * BK * 2);
        } else {
            const char* p = lds + at[t] + ks * 16 * R * 2;
            const bf16x4 a = ds_read_tr4(reinterpret_cast<const bf16*>(p));
            const bf16x4 b = ds_read_tr4(reinterpret_cast<const bf16*>(p + 4 * R * 2));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    static constexpr int kReads = KC ? T : 2 * T;
};

// y (and z) of V consecutive columns n of row m from their sums.
template <int ACT, int V>
__device__ __forceinline__ void epilogue(const BfGemm& g, int64_t m, int64_t n, float* v) {
    if (g.bias) {
        float b[V];
        load_part<float, V>(g.bias, n, g.N, b);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += b[e];
    }
    if (ACT != ACT_NONE && g.z) store_part<bf16, V>((bf16*)g.z + m * g.N, n, g.N, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = act_value<ACT>(v[e]);
    if (g.residual) {
        float r[V];
        load_part<bf16, V>((const bf16*)g.residual + m * g.N, n, g.N, r);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += r[e];
    }
    store_part<bf16, V>((bf16*)g.C + m * g.N, n, g.N, v);
}

template <int BN, int BM, int BK, bool PKC, bool QKC, bool DMA, int ACT>
__global__ __launch_bounds__(kThreads, 2) void bf_gemm_kernel(Args a) {
    constexpr int TN = BN / 64, TM = BM / 64;  // 32 x 32 tiles of a wave
    typedef Operand<BM, BK, PKC> OpP;
    typedef Operand<BN, BK, QKC> OpQ;
    constexpr int kStage = OpP::kBytes + OpQ::kBytes, kBufs = DMA ? 3 : 2;
    __shared__ __attribute__((aligned(1024))) char smem[kBufs * kStage];  // [buffer][Q, P]
    const int lane = threadIdx.x & 63, w = wave_id(), hh = lane >> 5;
    const int wn = w & 1, wm = w >> 1;

    int i = xcd_block((int)blockIdx.x, (int)gridDim.x);
    const int slice = __builtin_amdgcn_readfirstlane((int)a.per_slice_tiles.div(i));
    i -= slice * a.tiles_m * a.tiles_n;
    // Eight rows of tiles at a time, column by column.
    constexpr int kBand = 8;
    const int band = i / (kBand * a.tiles_n), in = i - band * kBand * a.tiles_n;
    const int high = min(kBand, a.tiles_m - band * kBand), col = in / high;
    // scalars, whatever unit divides: the direct loads take their bases from them
    const int tn = __builtin_amdgcn_readfirstlane(col), tm = __builtin_amdgcn_readfirstlane(band * kBand + in - col * high);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int s0 = slice * a.per_slice, s1 = min(s0 + a.per_slice, a.stages);

    const int64_t ldp = PKC ? a.g.K : a.g.M, ldq = QKC ? a.g.K : a.g.N;
    const bf16 *P = (const bf16*)a.g.P, *Q = (const bf16*)a.g.Q;
    Fragments<BM, BK, PKC, TM> fp;
    Fragments<BN, BK, QKC, TN> fq;
    fp.init(wm * BM / 2, lane);
    fq.init(wn * BN / 2, lane);
    f32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int k = 0; k < TM; ++k) {
            acc[j][k] = zero16();
            asm volatile("" : "+v"(acc[j][k]));  // not a literal zero (see mfma_v_first)
        }
    auto multiply = [&](const char* q, const char* p) {
        struct Ops {
            bf16x8 q[TN], p[TM];
        };
        auto read = [&](int ks) {
            Ops o;
#pragma unroll
            for (int t = 0; t < TN; ++t) o.q[t] = fq.read(q, ks, t);
#pragma unroll
            for (int t = 0; t < TM; ++t) o.p[t] = fp.read(p, ks, t);
            return o;
        };
        Ops cur = read(0);
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            Ops next;
            if (ks + 1 < BK / 16) next = read(ks + 1);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int k = 0; k < TM; ++k) acc[j][k] = mfma_bf16(cur.q[j], cur.p[k], acc[j][k]);
            if (ks + 1 < BK / 16) cur = next;
        }
        pin_read_ahead<BK / 16, 1, Fragments<BM, BK, PKC, TM>::kReads + Fragments<BN, BK, QKC, TN>::kReads, TN * TM>();
    };
    bf16x8 rp[OpP::PER], rq[OpQ::PER];
    auto fetch = [&](int s) {
        const int64_t k0 = (int64_t)s * BK;
#pragma unroll
        for (int j = 0; j < OpQ::PER; ++j) rq[j] = OpQ::fetch(Q, ldq, n0, a.g.N, k0, a.g.K, w, j, lane);
#pragma unroll
        for (int j = 0; j < OpP::PER; ++j) rp[j] = OpP::fetch(P, ldp, m0, a.g.M, k0, a.g.K, w, j, lane);
    };
    auto store = [&](char* stage) {
#pragma unroll
        for (int j = 0; j < OpQ::PER; ++j) OpQ::store(stage, w, j, lane, rq[j]);
#pragma unroll
        for (int j = 0; j < OpP::PER; ++j) OpP::store(stage + OpQ::kBytes, w, j, lane, rp[j]);
    };

    if constexpr (DMA) {
        OpP op;
        OpQ oq;
        op.init(w, lane, m0, a.g.M, ldp);
        oq.init(w, lane, n0, a.g.N, ldq);
        const char* tp = reinterpret_cast<const char*>(P + (PKC ? m0 * ldp : m0));
        const char* tq = reinterpret_cast<const char*>(Q + (QKC ? n0 * ldq : n0));
        const int64_t step_p = (int64_t)BK * 2 * (PKC ? 1 : ldp), step_q = (int64_t)BK * 2 * (QKC ? 1 : ldq);
        const uint32_t base = lds_addr(smem);
        auto issue = [&](int s, int buf) {
            oq.issue(tq + s * step_q, base + (uint32_t)(buf * kStage), w);
            op.issue(tp + s * step_p, base + (uint32_t)(buf * kStage + OpQ::kBytes), w);
        };
        const int sf = min(s1, (int)(a.g.K / BK));  // whole stages
        if (s0 < sf) issue(s0, 0);
        if (s0 + 1 < sf) issue(s0 + 1, 1);
        int buf = 0;
        for (int s = s0; s < sf; ++s) {
            // Stage s has landed in every wave's share, and every wave is done
            // with stage s - 1, whose buffer stage s + 2 takes.
            if (s + 1 < sf) wait_vmcnt<OpP::PER + OpQ::PER>();
            else wait_vmcnt<0>();
            lds_barrier();
            if (s + 2 < sf) issue(s + 2, buf == 0 ? 2 : buf - 1);
            multiply(smem + buf * kStage, smem + buf * kStage + OpQ::kBytes);
            buf = buf == 2 ? 0 : buf + 1;
        }
        if (sf < s1) {  // the last, partial stage
            fetch(sf);
            lds_barrier();
            store(smem);
            lds_barrier();
            multiply(smem, smem + OpQ::kBytes);
        }
    } else {
        fetch(s0);
        store(smem);
        lds_barrier();
        int buf = 0;
        for (int s = s0; s < s1; ++s) {
            if (s + 1 < s1) fetch(s + 1);
            multiply(smem + buf * kStage, smem + buf * kStage + OpQ::kBytes);
            buf ^= 1;
            if (s + 1 < s1) store(smem + buf * kStage);
            lds_barrier();
        }
    }

    const int64_t mw = m0 + wm * (BM / 2) + (lane & 31), nw = n0 + wn * (BN / 2) + 4 * hh;
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        const int64_t m = mw + 32 * k;
        if (m >= a.g.M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t n = nw + 32 * j + 8 * q;
                if (n >= a.g.N) continue;
                float v[4] = {acc[j][k][4 * q], acc[j][k][4 * q + 1], acc[j][k][4 * q + 2], acc[j][k][4 * q + 3]};
                if (a.whole) epilogue<ACT, 4>(a.g, m, n, v);
                else store_part<float, 4>(a.g.partial + ((int64_t)slice * a.g.M + m) * a.g.N, n, a.g.N, v);
            }
    }
}

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
    epilogue<ACT, 4>(a.g, m, n, v);
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Plan {
    int shape;  // 0: 256 x 128 (n x m), 1: 128 x 128, 2: 64 x 64
    Args a;
};
constexpr int kBN[3] = {256, 128, 64}, kBM[3] = {128, 128, 64}, kBK[3] = {32, 32, 64};

Plan plan(const BfGemm& g) {
    Plan p{};
    const int cus = device_cus();
    auto tiles = [&](int s) { return ((g.N + kBN[s] - 1) / kBN[s]) * ((g.M + kBM[s] - 1) / kBM[s]); };
    p.shape = tiles(0) >= cus ? 0 : tiles(1) >= cus ? 1 : 2;
    int64_t slices = 1;
    if (p.shape == 2) {
        if (tiles(1) * (g.K / 512) >= cus) p.shape = 1;
        const int64_t t = tiles(p.shape);
        if (2 * t < cus * 2) slices = std::max<int64_t>(1, std::min<int64_t>(2 * cus / t, g.K / 256));
    }
    const int s = p.shape;
    p.a.g = g;
    p.a.tiles_m = (int)((g.M + kBM[s] - 1) / kBM[s]);
    p.a.tiles_n = (int)((g.N + kBN[s] - 1) / kBN[s]);
    p.a.stages = (int)((g.K + kBK[s] - 1) / kBK[s]);
    p.a.per_slice = (int)((p.a.stages + slices - 1) / slices);
    p.a.slices = (p.a.stages + p.a.per_slice - 1) / p.a.per_slice;
    p.a.whole = p.a.slices == 1;
    p.a.per_slice_tiles = FastDiv::make((uint32_t)(p.a.tiles_m * p.a.tiles_n));
    return p;
}

template <int BN, int BM, int BK, bool PKC, bool QKC, int ACT>
void launch_t(const Args& a, bool dma, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices));
    if (dma) hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, BK, PKC, QKC, true, ACT>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((bf_gemm_kernel<BN, BM, BK, PKC, QKC, false, ACT>), grid, dim3(kThreads), 0, st, a);
}
template <bool PKC, bool QKC, int ACT> void launch_s(const Plan& p, bool dma, hipStream_t st) {
    if (p.shape == 0) launch_t<256, 128, 32, PKC, QKC, ACT>(p.a, dma, st);
    else if (p.shape == 1) launch_t<128, 128, 32, PKC, QKC, ACT>(p.a, dma, st);
    else launch_t<64, 64, 64, PKC, QKC, ACT>(p.a, dma, st);
}
template <int ACT> void launch_act_fwd(const Plan& p, bool dma, hipStream_t st) {
    if (p.a.g.q_kc) launch_s<true, true, ACT>(p, dma, st);
    else launch_s<true, false, ACT>(p, dma, st);
}

}  // namespace

size_t bf_gemm_workspace(const BfGemm& g) {
    const Plan p = plan(g);
    return p.a.whole ? 0 : (size_t)p.a.slices * g.M * g.N * 4;
}

hipError_t launch_bf_gemm(const BfGemm& g, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    const Plan p = plan(g);
    const int64_t ldp = g.p_kc ? g.K : g.M, ldq = g.q_kc ? g.K : g.N;
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
