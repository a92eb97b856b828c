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
#include <cmath>
#include <type_traits>

#include "attn_common.h"
#include "attn_geometry.h"
#include "attn_kernels.h"
#include "linear_epilogue.h"
#include "prologue_kernels.h"
#include "row_util.h"

namespace mft {
namespace {

constexpr int kThreads = 256;
constexpr int kHalf = 32, kSlab = 64;  // k of a pipeline step, and of a slab with k contiguous

struct Args {
    LinearProduct g;
    int tiles_m, tiles_n, slices;
    int halves, per_slice;  // whole halves that go in pairs; of one slice (even)
    int whole;              // one slice: the epilogue in the product's launch
    FastDiv per_slice_tiles;
};

// 16 rows' reads of one chunk of a slab of 64 meet no bank twice.
__device__ __forceinline__ constexpr int swz_kc(int r) { return (r >> 1) & 7; }

// One operand of R rows a tile, for a workgroup of W waves: RING slabs of SK k.
template <int R, bool KC, int W = 4, int SK = KC ? kSlab : kHalf, int RING = KC ? 2 : 3> struct Operand {
    static_assert(!KC || SK == kSlab, "whole lines");
    static_assert(KC || R * 4 % (64 * W) == 0, "every thread's chunks are rows of the slab");
    static constexpr int kSlabBytes = R * SK * 2, kBytes = RING * kSlabBytes;
    static constexpr int ROW = KC ? kSlab : R, CPR = ROW / 8;  // elements and chunks of an LDS row
    static constexpr int PER = kSlabBytes / 1024 / W;          // direct loads (1 KiB) of a wave per slab
    static constexpr int HALF = (R * 4 + 64 * W - 1) / (64 * W);  // 16-byte chunks of a thread per half, at most
    // The slab that holds half h (an offset in the operand's LDS).
    __device__ __forceinline__ static int slab(int h) {
        return KC ? (h >> 1 & 1) * kSlabBytes : (int)((unsigned)h % 3u) * kSlabBytes;
    }
    __device__ __forceinline__ static int swz_of(int r) { return KC ? swz_kc(r) : swz_tr<CPR>(r); }

    // Direct loads: this lane's byte offsets from a slab's first element.
    struct Dma {
        uint32_t off[PER];
        __device__ __forceinline__ void init(int w, int lane, int64_t r0, int64_t rows, int64_t ld) {
            static_assert(PER * W * 1024 == kSlabBytes && 64 % CPR == 0, "whole loads of whole rows");
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int r = (w * PER + j) * (64 / CPR) + lane / CPR, c = lane % CPR ^ swz_of(r);
                if (KC)  // rows past the end are read again from the last one, and not stored
                    off[j] = (uint32_t)((min(r0 + r, rows - 1) - r0) * ld * 2) + 16u * c;
                else  // whole chunks, the last of them again past the end
                    off[j] = (uint32_t)(r * ld * 2) + (uint32_t)(min(r0 + 8 * c, (rows - 1) / 8 * 8) - r0) * 2u;
            }
        }
        // Load j of the slab whose first element is `from`, into the slab at LDS address `to`.
        __device__ __forceinline__ void issue(const char* from, uint32_t to, int w, int j) const {
            load_lds_16_s(from, off[j], to + (uint32_t)(w * PER + j) * 1024u);
        }
    };

    // A half through registers, from anywhere and with zeros past the ends.
    typedef bf16 any8 __attribute__((ext_vector_type(8), aligned(2)));
    __device__ __forceinline__ static int half_row(int j, int tid) { return (j * 64 * W + tid) / (KC ? 4 : CPR); }
    __device__ __forceinline__ static int half_chunk(int j, int tid) { return (j * 64 * W + tid) % (KC ? 4 : CPR); }
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
    // The first half of the slab at `to`, or with SK = 64 the second one.
    __device__ __forceinline__ static void store(char* to, int second, int j, int tid, bf16x8 v) {
        if (R * 4 % (64 * W) != 0 && j * 64 * W + tid >= R * 4) return;
        const int r = half_row(j, tid) + (KC ? 0 : kHalf * second), c = half_chunk(j, tid) + (KC ? 4 * second : 0);
        *reinterpret_cast<bf16x8*>(to + r * ROW * 2 + (c ^ swz_of(r)) * 16) = v;
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
};

// This workgroup's slice and tile.
template <int BN, int BM> __device__ __forceinline__ void place(const Args& a, int* slice, int64_t* m0, int64_t* n0) {
    int i = xcd_block((int)blockIdx.x, (int)gridDim.x);
    *slice = __builtin_amdgcn_readfirstlane((int)a.per_slice_tiles.div(i));
    i -= *slice * a.tiles_m * a.tiles_n;
    // Four rows of tiles at a time (of 256, eight), column by column: 8192 x 1024 -> 4096 with GELU, 256 x
    // 128, 98 us with eight, 92 with four (its plain y 76 and 78, dW 71 and 69); of 13 other products none
    // is off by over 1 percent either way.
    constexpr int kBand = BM > 128 ? 8 : 4;
    const int band = i / (kBand * a.tiles_n), in = i - band * kBand * a.tiles_n;
    const int high = min(kBand, a.tiles_m - band * kBand), col = in / high;
    // scalars, whatever unit divides: the direct loads take their bases from them
    *n0 = (int64_t)__builtin_amdgcn_readfirstlane(col) * BN;
    *m0 = (int64_t)__builtin_amdgcn_readfirstlane(band * kBand + in - col * high) * BM;
}

// 32 rows of C from mw on, 32 TN columns from nw on, through this wave's LDS (32
// rows of 32 TN + 4 fp32: a bank group apart).
template <int TN, int ACT>
__device__ __forceinline__ void write_rows(const Args& a, int slice, int64_t mw, int64_t nw, const f32x16 (&acc)[TN],
                                           float* st, int lane) {
    constexpr int V = 8, LPR = 32 * TN / V, kPitch = 32 * TN + 4;  // lanes to a row
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(st + (lane & 31) * kPitch + 32 * j + 8 * q + 4 * (lane >> 5)) =
                f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
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
        if (a.whole) linear_epilogue<bf16, ACT, V>(a.g, m, n, v);
        else store_part<float, V>(a.g.partial + ((int64_t)slice * a.g.M + m) * a.g.N, n, a.g.N, v);
    }
    asm volatile("" ::: "memory");
}

template <int BN, int BM, bool PKC, bool QKC, bool DMA, int ACT>
__global__ __launch_bounds__(kThreads, BN * BM > 32768 ? 1 : 2) void bf_gemm_kernel(Args a) {
    constexpr int TN = BN / 64, TM = BM / 64;  // 32 x 32 tiles of a wave
    typedef Operand<BM, PKC> OpP;
    typedef Operand<BN, QKC> OpQ;
    constexpr int WN = BN / 2, kPitch = WN + 4;  // the epilogue's rows of fp32, a bank group apart
    constexpr int kStaged = 4 * 32 * kPitch * 4, kSlabs = OpQ::kBytes + OpP::kBytes;
    __shared__ __attribute__((aligned(1024))) char smem[kSlabs > kStaged ? kSlabs : kStaged];  // [Q slabs][P slabs]
    char* const lds_p = smem + OpQ::kBytes;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wn = w & 1, wm = w >> 1;

    int slice;
    int64_t m0, n0;
    place<BN, BM>(a, &slice, &m0, &n0);
    const bool last = slice == a.slices - 1;
    // Halves of this slice, and where the last one's k end (the rest of K goes through registers).
    const int h0 = slice * a.per_slice, h1 = last ? a.halves : h0 + a.per_slice;

    const int64_t ldp = a.g.ldp, ldq = a.g.ldq;
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
            // not a literal zero (see mfma_v_first)
            if constexpr (TN * TM > 8) asm volatile("" : "+a"(acc[j][k]));
            else asm volatile("" : "+v"(acc[j][k]));
        }
    struct Ops {
        bf16x8 q[TN], p[TM];
    };
    constexpr int kTiles = TN * TM, kFrags = TN + TM;
    // Fragment f of step ks of half h (the second of its pair if `odd`).
    auto read_one = [&](Ops& o, int h, bool odd, int ks, int f) {
        if (f < TM) o.p[f] = fp.read(lds_p + OpP::slab(h), odd, ks, f);
        else o.q[f - TM] = fq.read(smem + OpQ::slab(h), odd, ks, f - TM);
    };
    auto read = [&](int h, bool odd, int ks) {
        Ops o;
#pragma unroll
        for (int f = 0; f < kFrags; ++f) read_one(o, h, odd, ks, f);
        return o;
    };
    auto multiply_one = [&](const Ops& o, int t) {
        acc[t / TM][t % TM] = mfma_bf16(o.q[t / TM], o.p[t % TM], acc[t / TM][t % TM]);
    };
    auto multiply = [&](const Ops& o) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) multiply_one(o, t);
    };

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
            // Load j of half h, ODD its place in its pair (a slab of 64 comes with its even half).
            auto issue_one = [&](int h, auto odd_t, int j) {
                constexpr bool ODD = decltype(odd_t)::value;
                constexpr int NQ = QKC && ODD ? 0 : OpQ::PER;
                if (j < NQ) dq.issue(tq + h * step_q, base + (uint32_t)OpQ::slab(h), w, j);
                else dp.issue(tp + h * step_p, base + (uint32_t)(OpQ::kBytes + OpP::slab(h)), w, j - NQ);
            };
            constexpr std::false_type even{};
            constexpr std::true_type odd{};
            constexpr int kEven = OpQ::PER + OpP::PER, kOdd = (QKC ? 0 : OpQ::PER) + (PKC ? 0 : OpP::PER);
            auto issue = [&](int h, auto odd_t) {
#pragma unroll
                for (int j = 0; j < (decltype(odd_t)::value ? kOdd : kEven); ++j) issue_one(h, odd_t, j);
            };
            issue(h0, even);
            issue(h0 + 1, odd);
            wait_vmcnt<kOdd>();
            lds_barrier();
            Ops cur = read(h0, false, 0);
            // A step's MFMAs, with the next step's fragment reads and a share of the loads of a
            // half between them: one after the other in this order, as a wave that issues many
            // loads at once waits for them with nothing to multiply.
            auto weave = [&](const Ops& o, auto&& reads, auto&& loads) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
#pragma unroll
                    for (int f = t * kFrags / kTiles; f < (t + 1) * kFrags / kTiles; ++f) reads(f);
                    multiply_one(o, t);
                    loads(t);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // Share t of kTiles of a part (0: the first, 1: the second) of half h's loads.
            auto share = [&](int h, auto odd_t, int part, int t) {
                constexpr int n = decltype(odd_t)::value ? kOdd : kEven, first = (n + 1) / 2;
                const int from = part ? first : 0, count = part ? n - first : first;
#pragma unroll
                for (int j = 0; j < n; ++j)
                    if (j >= from + t * count / kTiles && j < from + (t + 1) * count / kTiles) issue_one(h, odd_t, j);
            };
            // One half, ODD its place in its pair; LEFT: halves after it (3: at least three).  The
            // loads of half h + 3 go out behind the barrier, when half h's slabs are free, and in half h + 1.
            auto half = [&](int h, auto odd_t, auto left_t) {
                constexpr bool ODD = decltype(odd_t)::value;
                constexpr int LEFT = decltype(left_t)::value;
                constexpr std::bool_constant<!ODD> other{};
                Ops nxt;
                weave(cur, [&](int f) { read_one(nxt, h, ODD, 1, f); },
                      [&](int t) {
                          if constexpr (LEFT >= 2) share(h + 2, odd_t, 1, t);
                      });
                if constexpr (LEFT >= 1) {
                    // Half h + 1 has landed (h + 2 may be on its way), and all of half h is read.
                    wait_vmcnt<LEFT == 1 ? 0 : ODD ? kOdd : kEven>();
                    lds_barrier();
                    weave(nxt, [&](int f) { read_one(cur, h + 1, !ODD, 0, f); },
                          [&](int t) {
                              if constexpr (LEFT >= 3) share(h + 3, other, 0, t);
                          });
                } else {
                    multiply(nxt);
                }
            };
            if (h0 + 2 < h1) {  // the first part of half h0 + 2, as if by the half before
#pragma unroll
                for (int t = 0; t < kTiles; ++t) share(h0 + 2, even, 0, t);
            }
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
            for (int j = 0; j < OpQ::HALF; ++j) OpQ::store(smem + OpQ::slab(i), 0, j, threadIdx.x, rq[j]);
#pragma unroll
            for (int j = 0; j < OpP::HALF; ++j) OpP::store(lds_p + OpP::slab(i), 0, j, threadIdx.x, rp[j]);
            lds_barrier();
            if (h + 1 < to) fetch(h + 1);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) multiply(read(i, false, ks));
        }
    }

    lds_barrier();  // the slabs have been read
    float* st = reinterpret_cast<float*>(smem) + w * 32 * kPitch;
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        const int64_t mw = m0 + wm * (BM / 2) + 32 * k;
        if (mw >= a.g.M) break;
        f32x16 rows[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) rows[j] = acc[j][k];
        write_rows<TN, ACT>(a, slice, mw, n0 + wn * WN, rows, st, lane);
    }
}

// A tile for a CU of its own: two groups of 2 x 2 waves take the halves of each
// pair of halves, three or four pairs are in LDS, and the groups' sums meet there
// at the end.
constexpr int kDeepThreads = 512;
template <int BN, int BM, bool PKC, bool QKC, bool DMA, int ACT>
__global__ __launch_bounds__(kDeepThreads, 2) void bf_gemm_deep(Args a) {
    constexpr int TN = BN / 64, TM = BM / 64, kTiles = TN * TM, kFrags = TN + TM;
    static_assert(TM == 2, "each group writes one of a wave's two rows of tiles");
    constexpr int kRing = (160 << 10) / ((BN + BM) * kSlab * 2) < 4 ? 3 : 4;
    typedef Operand<BM, PKC, 8, kSlab, kRing> OpP;
    typedef Operand<BN, QKC, 8, kSlab, kRing> OpQ;
    constexpr int kPair = OpQ::kSlabBytes + OpP::kSlabBytes, PER = OpQ::PER + OpP::PER;
    constexpr int kPitch = 32 * TN + 4;
    static_assert(8 * 32 * kPitch * 4 <= kRing * kPair && 8 * TN * 16 * 64 * 4 <= kRing * kPair, "fits the slabs");
    __shared__ __attribute__((aligned(1024))) char smem[kRing * kPair];  // [pair][Q, P]
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wn = w & 1, wm = w >> 1 & 1, group = w >> 2;
    int slice;
    int64_t m0, n0;
    place<BN, BM>(a, &slice, &m0, &n0);
    const int p0 = slice * a.per_slice / 2, p1 = min(p0 + a.per_slice / 2, a.halves / 2);  // pairs
    const int64_t ldp = a.g.ldp, ldq = a.g.ldq;
    const bf16 *P = (const bf16*)a.g.P, *Q = (const bf16*)a.g.Q;
    Fragments<BM, PKC, TM> fp;
    Fragments<BN, QKC, TN> fq;
    fp.init(wm * BM / 2, lane);
    fq.init(wn * BN / 2, lane);
    // This group's half of a slab.
    const int half_p = group * (PKC ? 0 : OpP::kSlabBytes / 2), half_q = group * (QKC ? 0 : OpQ::kSlabBytes / 2);
    if (PKC && group)
#pragma unroll
        for (int i = 0; i < 2; ++i) fp.at[i] = fp.at[2 + i];
    if (QKC && group)
#pragma unroll
        for (int i = 0; i < 2; ++i) fq.at[i] = fq.at[2 + i];
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
    auto read_one = [&](Ops& o, int slot, int ks, int f) {
        const char* at = smem + slot * kPair;
        if (f < TM) o.p[f] = fp.read(at + OpQ::kSlabBytes + half_p, false, ks, f);
        else o.q[f - TM] = fq.read(at + half_q, false, ks, f - TM);
    };
    auto read = [&](int slot, int ks) {
        Ops o;
#pragma unroll
        for (int f = 0; f < kFrags; ++f) read_one(o, slot, ks, f);
        return o;
    };
    auto multiply_one = [&](const Ops& o, int t) { acc[t / TM][t % TM] = mfma_bf16(o.q[t / TM], o.p[t % TM], acc[t / TM][t % TM]); };
    if (DMA && p0 < p1) {
        typename OpP::Dma dp;
        typename OpQ::Dma dq;
        dp.init(w, lane, m0, a.g.M, ldp);
        dq.init(w, lane, n0, a.g.N, ldq);
        const char* tp = reinterpret_cast<const char*>(P + (PKC ? m0 * ldp : m0));
        const char* tq = reinterpret_cast<const char*>(Q + (QKC ? n0 * ldq : n0));
        const int64_t step_p = (int64_t)kSlab * 2 * (PKC ? 1 : ldp), step_q = (int64_t)kSlab * 2 * (QKC ? 1 : ldq);
        const uint32_t base = lds_addr(smem);
        auto issue_one = [&](int p, int slot, int j) {
            const uint32_t to = base + (uint32_t)(slot * kPair);
            if (j < OpQ::PER) dq.issue(tq + p * step_q, to, w, j);
            else dp.issue(tp + p * step_p, to + OpQ::kSlabBytes, w, j - OpQ::PER);
        };
#pragma unroll
        for (int i = 0; i < kRing; ++i)
            if (p0 + i < p1)
#pragma unroll
                for (int j = 0; j < PER; ++j) issue_one(p0 + i, i, j);
        if (p0 + kRing <= p1) wait_vmcnt<(kRing - 1) * PER>();
        else wait_vmcnt<0>();
        lds_barrier();
        Ops cur = read(0, 0);
        // MORE: pair p + kRing exists.
        auto pair = [&](int p, int slot, auto more_t) {
            constexpr bool MORE = decltype(more_t)::value;
            const int after = slot + 1 == kRing ? 0 : slot + 1;
            Ops nxt;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
#pragma unroll
                for (int f = t * kFrags / kTiles; f < (t + 1) * kFrags / kTiles; ++f) read_one(nxt, slot, 1, f);
                multiply_one(cur, t);
                __builtin_amdgcn_sched_barrier(0);
            }
            // Pair p + 1 has landed, and everybody has read pair p.
            if constexpr (MORE) wait_vmcnt<(kRing - 2) * PER>();
            else wait_vmcnt<0>();
            lds_barrier();
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                if (MORE || p + 1 < p1) {
#pragma unroll
                    for (int f = t * kFrags / kTiles; f < (t + 1) * kFrags / kTiles; ++f) read_one(cur, after, 0, f);
                }
                multiply_one(nxt, t);
                if constexpr (MORE) {
#pragma unroll
                    for (int j = t * PER / kTiles; j < (t + 1) * PER / kTiles; ++j) issue_one(p + kRing, slot, j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        int p = p0, slot = 0;
        for (; p + kRing < p1; ++p) {
            pair(p, slot, std::true_type{});
            slot = slot + 1 == kRing ? 0 : slot + 1;
        }
        for (; p < p1; ++p) {
            pair(p, slot, std::false_type{});
            slot = slot + 1 == kRing ? 0 : slot + 1;
        }
    }
    // What is left of K in pairs, or all of it, half by half through registers, the groups in turn.
    const bool last = slice == a.slices - 1;
    const int from = DMA ? a.halves : 2 * p0, to = !last ? (DMA ? from : 2 * p1) : (int)((a.g.K + kHalf - 1) / kHalf);
    bf16x8 rp[OpP::HALF], rq[OpQ::HALF];
    auto fetch = [&](int h) {
        const int64_t k0 = (int64_t)h * kHalf;
#pragma unroll
        for (int j = 0; j < OpQ::HALF; ++j) rq[j] = OpQ::fetch(Q, ldq, n0, a.g.N, k0, a.g.K, j, threadIdx.x);
#pragma unroll
        for (int j = 0; j < OpP::HALF; ++j) rp[j] = OpP::fetch(P, ldp, m0, a.g.M, k0, a.g.K, j, threadIdx.x);
    };
    if (from < to) fetch(from);
    for (int h = from; h < to; ++h) {
        lds_barrier();  // everybody has read what was there
#pragma unroll
        for (int j = 0; j < OpQ::HALF; ++j) OpQ::store(smem, h & 1, j, threadIdx.x, rq[j]);
#pragma unroll
        for (int j = 0; j < OpP::HALF; ++j) OpP::store(smem + OpQ::kSlabBytes, h & 1, j, threadIdx.x, rp[j]);
        lds_barrier();
        if (h + 1 < to) fetch(h + 1);
        if ((h & 1) == group) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const Ops o = read(0, ks);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) multiply_one(o, t);
            }
        }
    }
    // Each group hands the other one half of its rows of m.
    lds_barrier();
    float* give = reinterpret_cast<float*>(smem) + (w ^ 4) * TN * 16 * 64;
    const float* got = reinterpret_cast<float*>(smem) + w * TN * 16 * 64;
    f32x16 rows[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        rows[j] = group ? acc[j][1] : acc[j][0];
        const f32x16 other = group ? acc[j][0] : acc[j][1];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(give + ((j * 4 + q) * 64 + lane) * 4) =
                f32x4{other[4 * q], other[4 * q + 1], other[4 * q + 2], other[4 * q + 3]};
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(got + ((j * 4 + q) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) rows[j][4 * q + e] += o[e];
        }
    lds_barrier();
    const int64_t mw = m0 + wm * (BM / 2) + 32 * group;
    if (mw < a.g.M)
        write_rows<TN, ACT>(a, slice, mw, n0 + wn * (BN / 2), rows, reinterpret_cast<float*>(smem) + w * 32 * kPitch, lane);
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
    linear_epilogue<bf16, ACT, 4>(a.g, m, n, v);
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

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
size_t up(size_t x) { return (x + 255) & ~size_t(255); }
int64_t whole_ld(int64_t cols) { return (cols + 7) / 8 * 8; }
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

// rows x cols of bf16 into rows of ld (a multiple of 8), zeros behind them.
__global__ __launch_bounds__(256) void pack_rows(const bf16* from, bf16* to, int64_t rows, int64_t cols, int64_t ld) {
    const int64_t chunks = ld / 8, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * chunks; i += step) {
        const int64_t r = i / chunks, c = (i - r * chunks) * 8;
        float v[8];
        load_part<bf16, 8>(from + r * cols, c, cols, v);
        AnyVec<bf16, 8>::store(to + r * ld + c, v);
    }
}
hipError_t pack(const void* from, void* to, int64_t rows, int64_t cols, hipStream_t st) {
    const int64_t ld = whole_ld(cols), n = rows * (ld / 8);
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 16 * device_cus()));
    hipLaunchKernelGGL(pack_rows, grid, dim3(256), 0, st, (const bf16*)from, (bf16*)to, rows, cols, ld);
    return hipGetLastError();
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
