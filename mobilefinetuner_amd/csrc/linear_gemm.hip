// The linear layer's bf16 products (C ABI in include/mft/linear.h):
// C[M, N] = act(sum_k P(m, k) Q(n, k) + bias[n]) + residual.
//
// A workgroup of 2 x 2 waves owns a BN x BM tile of C^T = Q P^T, on
// v_mfma_f32_32x32x16_bf16: Q's rows are the instruction's rows, so that a lane
// holds four consecutive columns n of one row m of C.
//
// Operands.  With k contiguous (KC) an operand lies in LDS as slabs [rows][64]
// and its fragments are 16-byte reads; a slab's rows are whole 128-byte lines
// (slabs of 32 took every line from L2 twice: 25 M requests for 13 M at 4096^3,
// and 157 us for 124).  With its rows contiguous it lies as slabs [32][rows] and
// its fragments are transposing reads.  Either way by direct loads into LDS
// where all rows and bases lie on 16 bytes (DMA), else through registers.
//
// Pipeline (DMA), in halves of 32 k: two slabs of 64 or three of 32 are in LDS.
// A wave reads the fragments of a half's second step while it multiplies the
// first; then one barrier tells that everybody has read the half and that the
// next has landed, the loads of the half three on go out into the freed slabs,
// and the next half's first fragments are read while the second step
// multiplies.  Two workgroups share a CU: one multiplies while the other waits
// or runs its epilogue.
//
// Epilogue.  The accumulators go through LDS, 32 rows of m at a time and wave by
// wave, so that y, z and the residual move in whole lines.
//
// Products of few tiles cut K into slices whose fp32 partials a second launch
// adds in their order and takes through the epilogue.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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

constexpr int kHalf = 32, kSlab = 64;  // k of a pipeline step, and of a slab with k contiguous

struct Args {
    BfGemm g;
    int tiles_m, tiles_n, slices;
    int halves, per_slice;  // whole halves that go in pairs; of one slice (even)
    int whole;              // one slice: the epilogue in the product's launch
    FastDiv per_slice_tiles;
};

__device__ __forceinline__ constexpr int swz_kc(int r) { return (r >> 1) & 7; }  // 16 rows' reads of a chunk: 16 banks' groups

// One operand of R rows a tile.
template <int R, bool KC> struct Operand {
    static constexpr int kSlabBytes = KC ? R * kSlab * 2 : R * kHalf * 2, kRing = KC ? 2 : 3;
    static constexpr int kBytes = kRing * kSlabBytes;
    static constexpr int ROW = KC ? kSlab : R, CPR = ROW / 8;  // elements and chunks of an LDS row
    static constexpr int PER = kSlabBytes / 4096;              // direct loads (1 KiB) of a wave per slab
    static constexpr int HALF = R / 64;                        // 16-byte chunks of a thread per half
    // The slab that holds half h (an offset in the operand's LDS).
    __device__ __forceinline__ static int slab(int h) {
        return KC ? (h >> 1 & 1) * kSlabBytes : (int)((unsigned)h % 3u) * kSlabBytes;
    }
    __device__ __forceinline__ static int swz_of(int r) { return KC ? swz_kc(r) : swz_tr<CPR>(r); }

    // Direct loads: this lane's byte offsets from a slab's first element.
    struct Dma {
        uint32_t off[PER];
        __device__ __forceinline__ void init(int w, int lane, int64_t r0, int64_t rows, int64_t ld) {
            static_assert(PER * 4096 == kSlabBytes && 64 % CPR == 0, "whole loads of whole rows");
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int r = (w * PER + j) * (64 / CPR) + lane / CPR, c = lane % CPR ^ swz_of(r);
                if (KC)  // rows past the end are read again from the last one, and not stored
                    off[j] = (uint32_t)((min(r0 + r, rows - 1) - r0) * ld * 2) + 16u * c;
                else
                    off[j] = (uint32_t)(r * ld * 2) + (uint32_t)(min(r0 + 8 * c, rows - 8) - r0) * 2u;
            }
        }
        // Load j of the slab whose first element is `from`, into the slab at LDS address `to`.
        __device__ __forceinline__ void issue(const char* from, uint32_t to, int w, int j) const {
            load_lds_16_s(from, off[j], to + (uint32_t)(w * PER + j) * 1024u);
        }
    };

    // A half through registers, from anywhere and with zeros past the ends.
    typedef bf16 any8 __attribute__((ext_vector_type(8), aligned(2)));
    __device__ __forceinline__ static int half_row(int j, int tid) { return KC ? (j * kThreads + tid) / 4 : (j * kThreads + tid) / CPR; }
    __device__ __forceinline__ static int half_chunk(int j, int tid) { return KC ? tid % 4 : (j * kThreads + tid) % CPR; }
    __device__ __forceinline__ static bf16x8 fetch(const bf16* p, int64_t ld, int64_t r0, int64_t rows, int64_t k0,
                                                   int64_t K, int j, int tid) {
        const int r = half_row(j, tid), c = half_chunk(j, tid);
        const int64_t row = KC ? min(r0 + r, rows - 1) : k0 + r;  // storage row
        const int64_t col = (KC ? k0 : r0) + 8 * c, end = KC ? K : rows;
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
    __device__ __forceinline__ static void store(char* lds, int h, int j, int tid, bf16x8 v) {  // h even
        const int r = half_row(j, tid), c = half_chunk(j, tid);
        *reinterpret_cast<bf16x8*>(lds + slab(h) + r * ROW * 2 + (c ^ swz_of(r)) * 16) = v;
    }
};

// Fragments of T 32-row tiles from row `first` on.
template <int R, bool KC, int T> struct Fragments {
    uint32_t at[KC ? kSlab / 16 : T];
    __device__ __forceinline__ void init(int first, int lane) {
        const int n = lane & 31, hh = lane >> 5;
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < kSlab / 16; ++i)
                at[i] = (uint32_t)((first + n) * kSlab * 2 + ((2 * i + hh) ^ swz_kc(n)) * 16);
        } else {
            const int j = lane & 15, k = 8 * hh + j / 4;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int col = first + 32 * t + 16 * (lane >> 4 & 1) + 4 * (j & 3);
                at[t] = (uint32_t)(k * R * 2 + ((col >> 3) ^ swz_tr<R / 8>(k)) * 16 + (col & 7) * 2);
            }
        }
    }
    // Tile t, step ks (0, 1) of a half, the second of its pair if `odd`, in the slab at `lds`.
    __device__ __forceinline__ bf16x8 read(const char* lds, bool odd, int ks, int t) const {
        if constexpr (KC) {
            return *reinterpret_cast<const bf16x8*>(lds + at[2 * odd + ks] + t * 32 * kSlab * 2);
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

template <int BN, int BM, bool PKC, bool QKC, bool DMA, int ACT>
__global__ __launch_bounds__(kThreads, 2) void bf_gemm_kernel(Args a) {
    constexpr int TN = BN / 64, TM = BM / 64;  // 32 x 32 tiles of a wave
    typedef Operand<BM, PKC> OpP;
    typedef Operand<BN, QKC> OpQ;
    constexpr int WN = BN / 2, kPitch = WN + 4;  // the epilogue's rows of fp32, a bank group apart
    constexpr int kStaged = 4 * 32 * kPitch * 4, kSlabs = OpQ::kBytes + OpP::kBytes;
    __shared__ __attribute__((aligned(1024))) char smem[kSlabs > kStaged ? kSlabs : kStaged];  // [Q slabs][P slabs]
    char* const lds_p = smem + OpQ::kBytes;
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
    const bool last = slice == a.slices - 1;
    // Halves of this slice, and where the last one's k end (the rest of K goes through registers).
    const int h0 = slice * a.per_slice, h1 = last ? a.halves : h0 + a.per_slice;

    const int64_t ldp = PKC ? a.g.K : a.g.M, ldq = QKC ? a.g.K : a.g.N;
    const bf16 *P = (const bf16*)a.g.P, *Q = (const bf16*)a.g.Q;
    Fragments<BM, PKC, TM> fp;
    Fragments<BN, QKC, TN> fq;
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
    struct Ops {
        bf16x8 q[TN], p[TM];
    };
    auto read = [&](int h, bool odd, int ks) {
        Ops o;
        const char *q = smem + OpQ::slab(h), *p = lds_p + OpP::slab(h);
#pragma unroll
        for (int t = 0; t < TN; ++t) o.q[t] = fq.read(q, odd, ks, t);
#pragma unroll
        for (int t = 0; t < TM; ++t) o.p[t] = fp.read(p, odd, ks, t);
        return o;
    };
    constexpr int kTiles = TN * TM;
    auto multiply = [&](const Ops& o, int t0 = 0, int t1 = 1 << 10) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
            if (t >= t0 && t < t1) acc[t / TM][t % TM] = mfma_bf16(o.q[t / TM], o.p[t % TM], acc[t / TM][t % TM]);
    };
    constexpr int kReads = Fragments<BM, PKC, TM>::kReads + Fragments<BN, QKC, TN>::kReads;

    if constexpr (DMA) {
        if (h0 < h1) {
            typename OpP::Dma dp;
            typename OpQ::Dma dq;
            dp.init(w, lane, m0, a.g.M, ldp);
            dq.init(w, lane, n0, a.g.N, ldq);
            const char* tp = reinterpret_cast<const char*>(P + (PKC ? m0 * ldp : m0));
            const char* tq = reinterpret_cast<const char*>(Q + (QKC ? n0 * ldq : n0));
            const int64_t step_p = (int64_t)kHalf * 2 * (PKC ? 1 : ldp), step_q = (int64_t)kHalf * 2 * (QKC ? 1 : ldq);
            const uint32_t base = lds_addr(smem);
            // The loads of half h, ODD its place in its pair (a slab of 64 comes with its even half).
            auto issue = [&](int h, auto odd_t) {
                constexpr bool ODD = decltype(odd_t)::value;
                if constexpr (!(QKC && ODD)) {
                    const char* from = tq + h * step_q;
                    const uint32_t to = base + (uint32_t)OpQ::slab(h);
#pragma unroll
                    for (int j = 0; j < OpQ::PER; ++j) dq.issue(from, to, w, j);
                }
                if constexpr (!(PKC && ODD)) {
                    const char* from = tp + h * step_p;
                    const uint32_t to = base + (uint32_t)(OpQ::kBytes + OpP::slab(h));
#pragma unroll
                    for (int j = 0; j < OpP::PER; ++j) dp.issue(from, to, w, j);
                }
            };
            constexpr std::false_type even{};
            constexpr std::true_type odd{};
            constexpr int kEven = OpQ::PER + OpP::PER, kOdd = (QKC ? 0 : OpQ::PER) + (PKC ? 0 : OpP::PER);
            issue(h0, even);
            issue(h0 + 1, odd);
            if (h0 + 2 < h1) {
                issue(h0 + 2, even);
                wait_vmcnt<kEven + kOdd>();
            } else {
                wait_vmcnt<kOdd>();
            }
            lds_barrier();
            Ops cur = read(h0, false, 0);
            // N MFMAs with R LDS reads between them, in this order.
            auto spread = [](auto n_t, auto r_t) {
                constexpr int N = decltype(n_t)::value, R = decltype(r_t)::value, E = (R + N - 1) / N;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
                    if (i * E < R) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, E, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            // One half, ODD its place in its pair; LEFT: halves after it (3: at least three).
            auto half = [&](int h, auto odd_t, auto left_t) {
                constexpr bool ODD = decltype(odd_t)::value;
                constexpr int LEFT = decltype(left_t)::value;
                const Ops nxt = read(h, ODD, 1);
                multiply(cur);
                spread(std::integral_constant<int, kTiles>{}, std::integral_constant<int, kReads>{});
                if constexpr (LEFT >= 1) {
                    // Half h + 1 has landed (h + 2 may be on its way), and all of half h is read.
                    wait_vmcnt<LEFT == 1 ? 0 : ODD ? kOdd : kEven>();
                    lds_barrier();
                    constexpr int kFirst = (kTiles + 1) / 2;
                    cur = read(h + 1, !ODD, 0);
                    multiply(nxt, 0, kFirst);
                    spread(std::integral_constant<int, kFirst>{}, std::integral_constant<int, kReads>{});
                    if constexpr (LEFT >= 3) issue(h + 3, std::bool_constant<!ODD>{});
                    __builtin_amdgcn_sched_barrier(0);
                    multiply(nxt, kFirst);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    multiply(nxt);
                }
            };
            constexpr std::integral_constant<int, 0> left0{};
            constexpr std::integral_constant<int, 1> left1{};
            constexpr std::integral_constant<int, 2> left2{};
            constexpr std::integral_constant<int, 3> left3{};
            int h = h0;
            for (; h + 4 < h1; h += 2) {
                half(h, even, left3);
                half(h + 1, odd, left3);
            }
            if (h + 2 < h1) {
                half(h, even, left3);
                half(h + 1, odd, left2);
                h += 2;
            }
            half(h, even, left1);
            half(h + 1, odd, left0);
        }
    }
    // What is left of K in pairs of halves, or all of it, half by half through registers.
    const int from = DMA ? a.halves : h0, to = DMA || last ? (int)((a.g.K + kHalf - 1) / kHalf) : h1;
    if (!DMA || last) {
        bf16x8 rp[OpP::HALF], rq[OpQ::HALF];
        auto fetch = [&](int h) {
            const int64_t k0 = (int64_t)h * kHalf;
#pragma unroll
            for (int j = 0; j < OpQ::HALF; ++j) rq[j] = OpQ::fetch(Q, ldq, n0, a.g.N, k0, a.g.K, j, threadIdx.x);
#pragma unroll
            for (int j = 0; j < OpP::HALF; ++j) rp[j] = OpP::fetch(P, ldp, m0, a.g.M, k0, a.g.K, j, threadIdx.x);
        };
        if (from < to) {
            fetch(from);
            if (DMA) lds_barrier();  // everybody has read the last pair
        }
        for (int h = from; h < to; ++h) {
            // Two are in LDS at a time, each the even half of its slab: a wave stores one once all
            // have read the one before the last.
            const int i = 2 * (h - from);
#pragma unroll
            for (int j = 0; j < OpQ::HALF; ++j) OpQ::store(smem, i, j, threadIdx.x, rq[j]);
#pragma unroll
            for (int j = 0; j < OpP::HALF; ++j) OpP::store(lds_p, i, j, threadIdx.x, rp[j]);
            lds_barrier();
            if (h + 1 < to) fetch(h + 1);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) multiply(read(i, false, ks));
        }
    }

    // The accumulators, 32 rows of m at a time, through this wave's part of LDS.
    lds_barrier();
    float* st = reinterpret_cast<float*>(smem) + w * 32 * kPitch;
    constexpr int V = 8, LPR = WN / V;  // lanes to a row
    const int64_t nw = n0 + wn * WN;
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        const int64_t mw = m0 + wm * (BM / 2) + 32 * k;
        if (mw >= a.g.M) break;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4*>(st + (lane & 31) * kPitch + 32 * j + 8 * q + 4 * hh) =
                    f32x4{acc[j][k][4 * q], acc[j][k][4 * q + 1], acc[j][k][4 * q + 2], acc[j][k][4 * q + 3]};
        asm volatile("" ::: "memory");  // a wave's LDS accesses stay in order
#pragma unroll
        for (int r = 0; r < LPR / 2; ++r) {
            const int at = r * 64 + lane, row = at / LPR, c = at % LPR * V;
            const int64_t m = mw + row, n = nw + c;
            if (m >= a.g.M || n >= a.g.N) continue;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(st + row * kPitch + c + e);
                v[e] = u[0], v[e + 1] = u[1], v[e + 2] = u[2], v[e + 3] = u[3];
            }
            if (a.whole) epilogue<ACT, V>(a.g, m, n, v);
            else store_part<float, V>(a.g.partial + ((int64_t)slice * a.g.M + m) * a.g.N, n, a.g.N, v);
        }
        asm volatile("" ::: "memory");
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
    int shape;
    Args a;
};
constexpr int kShapes = 3;
constexpr int kBN[kShapes] = {256, 128, 64}, kBM[kShapes] = {128, 128, 64};

Plan plan(const BfGemm& g) {
    Plan p{};
    const int cus = device_cus();
    auto tiles = [&](int s) { return ((g.N + kBN[s] - 1) / kBN[s]) * ((g.M + kBM[s] - 1) / kBM[s]); };
    p.shape = tiles(0) >= cus ? 0 : tiles(1) >= cus ? 1 : 2;
    if (p.shape == 0 && g.p_kc && g.q_kc) p.shape = 1;
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
    const int pairs = (int)(g.K / kSlab);
    p.a.halves = 2 * pairs;
    const int per = std::max<int>(1, (int)((pairs + slices - 1) / slices));
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
template <bool PKC, bool QKC, int ACT> void launch_s(const Plan& p, bool dma, hipStream_t st) {
    if (p.shape == 2) {
        launch_t<64, 64, PKC, QKC, ACT>(p.a, dma, st);
        return;
    }
    if constexpr (!(PKC && QKC)) {
        if (p.shape == 0) {
            launch_t<256, 128, PKC, QKC, ACT>(p.a, dma, st);
            return;
        }
    }
    launch_t<128, 128, PKC, QKC, ACT>(p.a, dma, st);
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
