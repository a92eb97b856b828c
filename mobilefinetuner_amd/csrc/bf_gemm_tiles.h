// The kernels of the bf16 products of the linear layer (linear_gemm.hip) and of
// the gated linear layer (gated_gemm.hip):
// C[M, N] = act(sum_k P(m, k) Q(n, k) + bias[n]) + residual, and the forms of Q
// below.
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
#pragma once

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

// What a kernel makes of Q.  PLAIN: one operand.  GATED: two of N rows each, Q and
// Q2, half of a tile's columns from either, so that a lane holds both sums of an
// output column; C = act(P Q^T) (P Q2^T).  JOINED: k up to `joint` from Q and from there on
// from Q2 (whole pairs of halves, direct loads).
enum { PLAIN, GATED, JOINED };

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

// 32 rows of C from mw on, 32 TN columns from nw on (GATED: half as many of
// either sum), through this wave's LDS (32 rows of 32 TN + 4 fp32: a bank group apart).
template <int TN, int ACT, int MODE>
__device__ __forceinline__ void write_rows(const Args& a, int slice, int64_t mw, int64_t nw, const f32x16 (&acc)[TN],
                                           float* st, int lane) {
    constexpr int NQ = MODE == GATED ? 2 : 1, COLS = 32 * TN / NQ;
    constexpr int V = 8, LPR = COLS / V, kPitch = 32 * TN + 4;  // lanes to a row
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(st + (lane & 31) * kPitch + 32 * j + 8 * q + 4 * (lane >> 5)) =
                f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    asm volatile("" ::: "memory");  // a wave's LDS accesses stay in order
    if constexpr (MODE == GATED) {
        if (a.whole) {
            gated_rows_out<COLS, kPitch, false>(a.g, mw, nw, st, lane, nullptr, nullptr, nullptr);
            asm volatile("" ::: "memory");
            return;
        }
    }
#pragma unroll
    for (int r = 0; r < LPR / 2; ++r) {
        const int at = r * 64 + lane, row = at / LPR, c = at % LPR * V;
        const int64_t m = mw + row, n = nw + c;
        if (m >= a.g.M || n >= a.g.N) continue;
        float v[NQ][V];
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(st + row * kPitch + i * COLS + c + e);
                v[i][e] = u[0], v[i][e + 1] = u[1], v[i][e + 2] = u[2], v[i][e + 3] = u[3];
            }
        if (MODE != GATED && a.whole) {
            linear_epilogue<bf16, ACT, V>(a.g, m, n, v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                store_part<float, V>(a.g.partial + (((int64_t)slice * NQ + i) * a.g.M + m) * a.g.N, n, a.g.N, v[i]);
        }
    }
    asm volatile("" ::: "memory");
}

template <int BN, int BM, bool PKC, bool QKC, bool DMA, int ACT, int MODE = PLAIN>
__global__ __launch_bounds__(kThreads, BN * BM > 32768 ? 1 : 2) void bf_gemm_kernel(Args a) {
    static_assert(MODE != JOINED || DMA, "whole pairs of halves");
    constexpr int TN = BN / 64, TM = BM / 64;  // 32 x 32 tiles of a wave
    constexpr int NQ = MODE == GATED ? 2 : 1, TQ = TN / NQ;
    typedef Operand<BM, PKC> OpP;
    typedef Operand<BN / NQ, QKC> OpQ;
    constexpr int WN = BN / 2, kPitch = WN + 4;  // the epilogue's rows of fp32, a bank group apart
    constexpr int kStaged = 4 * 32 * kPitch * 4, kSlabs = NQ * OpQ::kBytes + OpP::kBytes;
    // [Q slabs][Q2 slabs][P slabs]
    __shared__ __attribute__((aligned(1024))) char smem[kSlabs > kStaged ? kSlabs : kStaged];
    char* const lds_p = smem + NQ * OpQ::kBytes;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wn = w & 1, wm = w >> 1;

    int slice;
    int64_t m0, n0;
    place<BN / NQ, BM>(a, &slice, &m0, &n0);
    const bool last = slice == a.slices - 1;
    // Halves of this slice, and where the last one's k end (the rest of K goes through registers).
    const int h0 = slice * a.per_slice, h1 = last ? a.halves : h0 + a.per_slice;

    const int64_t ldp = a.g.ldp, ldq = a.g.ldq;
    const bf16 *P = (const bf16*)a.g.P, *Q = (const bf16*)a.g.Q, *Q2 = (const bf16*)a.g.Q2;
    Fragments<BM, PKC, TM> fp;
    Fragments<BN / NQ, QKC, TQ> fq;
    fp.init(wm * BM / 2, lane);
    fq.init(wn * BN / NQ / 2, lane);
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
        else o.q[f - TM] = fq.read(smem + (f - TM) / TQ * OpQ::kBytes + OpQ::slab(h), odd, ks, (f - TM) % TQ);
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
            const char* tq2 = reinterpret_cast<const char*>(Q2 + (QKC ? n0 * ldq : n0));
            const int joint = (int)(a.g.joint / kHalf);
            const int64_t step_p = (int64_t)kHalf * 2 * (PKC ? 1 : ldp), step_q = (int64_t)kHalf * 2 * (QKC ? 1 : ldq);
            const uint32_t base = lds_addr(smem);
            // Load j of half h, ODD its place in its pair (a slab of 64 comes with its even half).
            auto issue_one = [&](int h, auto odd_t, int j) {
                constexpr bool ODD = decltype(odd_t)::value;
                constexpr int LQ = QKC && ODD ? 0 : NQ * OpQ::PER;
                if (j >= LQ) {
                    dp.issue(tp + h * step_p, base + (uint32_t)(NQ * OpQ::kBytes + OpP::slab(h)), w, j - LQ);
                } else {
                    const char* from = tq + h * step_q;
                    if (MODE == GATED && j >= OpQ::PER) from = tq2 + h * step_q;
                    if (MODE == JOINED && h >= joint) from = tq2 + (h - joint) * step_q;
                    dq.issue(from, base + (uint32_t)(j / OpQ::PER * OpQ::kBytes + OpQ::slab(h)), w, j % OpQ::PER);
                }
            };
            constexpr std::false_type even{};
            constexpr std::true_type odd{};
            constexpr int kEven = NQ * OpQ::PER + OpP::PER, kOdd = (QKC ? 0 : NQ * OpQ::PER) + (PKC ? 0 : OpP::PER);
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
        bf16x8 rp[OpP::HALF], rq[NQ][OpQ::HALF];
        auto fetch = [&](int h) {
            const int64_t k0 = (int64_t)h * kHalf;
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int j = 0; j < OpQ::HALF; ++j)
                    rq[i][j] = OpQ::fetch(i ? Q2 : Q, ldq, n0, a.g.N, k0, a.g.K, j, threadIdx.x);
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
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < OpQ::HALF; ++j)
                    OpQ::store(smem + q * OpQ::kBytes + OpQ::slab(i), 0, j, threadIdx.x, rq[q][j]);
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
        write_rows<TN, ACT, MODE>(a, slice, mw, n0 + wn * WN / NQ, rows, st, lane);
    }
}

// A tile for a CU of its own: two groups of 2 x 2 waves take the halves of each
// pair of halves, three or four pairs are in LDS, and the groups' sums meet there
// at the end.
constexpr int kDeepThreads = 512;
template <int BN, int BM, bool PKC, bool QKC, bool DMA, int ACT, int MODE = PLAIN>
__global__ __launch_bounds__(kDeepThreads, 2) void bf_gemm_deep(Args a) {
    static_assert(MODE != JOINED || DMA, "whole pairs of halves");
    constexpr int TN = BN / 64, TM = BM / 64, kTiles = TN * TM, kFrags = TN + TM;
    constexpr int NQ = MODE == GATED ? 2 : 1, TQ = TN / NQ;
    static_assert(TM == 2, "each group writes one of a wave's two rows of tiles");
    constexpr int kRing = (160 << 10) / ((BN + BM) * kSlab * 2) < 4 ? 3 : 4;
    typedef Operand<BM, PKC, 8, kSlab, kRing> OpP;
    typedef Operand<BN / NQ, QKC, 8, kSlab, kRing> OpQ;
    constexpr int kPair = NQ * OpQ::kSlabBytes + OpP::kSlabBytes, PER = NQ * OpQ::PER + OpP::PER;
    constexpr int kPitch = 32 * TN + 4;
    static_assert(8 * 32 * kPitch * 4 <= kRing * kPair && 8 * TN * 16 * 64 * 4 <= kRing * kPair, "fits the slabs");
    __shared__ __attribute__((aligned(1024))) char smem[kRing * kPair];  // [pair][Q, Q2, P]
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wn = w & 1, wm = w >> 1 & 1, group = w >> 2;
    int slice;
    int64_t m0, n0;
    place<BN / NQ, BM>(a, &slice, &m0, &n0);
    const int p0 = slice * a.per_slice / 2, p1 = min(p0 + a.per_slice / 2, a.halves / 2);  // pairs
    const int64_t ldp = a.g.ldp, ldq = a.g.ldq;
    const bf16 *P = (const bf16*)a.g.P, *Q = (const bf16*)a.g.Q, *Q2 = (const bf16*)a.g.Q2;
    Fragments<BM, PKC, TM> fp;
    Fragments<BN / NQ, QKC, TQ> fq;
    fp.init(wm * BM / 2, lane);
    fq.init(wn * BN / NQ / 2, lane);
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
        if (f < TM) o.p[f] = fp.read(at + NQ * OpQ::kSlabBytes + half_p, false, ks, f);
        else o.q[f - TM] = fq.read(at + (f - TM) / TQ * OpQ::kSlabBytes + half_q, false, ks, (f - TM) % TQ);
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
        const char* tq2 = reinterpret_cast<const char*>(Q2 + (QKC ? n0 * ldq : n0));
        const int joint = (int)(a.g.joint / kSlab);
        const int64_t step_p = (int64_t)kSlab * 2 * (PKC ? 1 : ldp), step_q = (int64_t)kSlab * 2 * (QKC ? 1 : ldq);
        const uint32_t base = lds_addr(smem);
        auto issue_one = [&](int p, int slot, int j) {
            const uint32_t to = base + (uint32_t)(slot * kPair);
            if (j >= NQ * OpQ::PER) {
                dp.issue(tp + p * step_p, to + NQ * OpQ::kSlabBytes, w, j - NQ * OpQ::PER);
            } else {
                const char* from = tq + p * step_q;
                if (MODE == GATED && j >= OpQ::PER) from = tq2 + p * step_q;
                if (MODE == JOINED && p >= joint) from = tq2 + (p - joint) * step_q;
                dq.issue(from, to + (uint32_t)(j / OpQ::PER * OpQ::kSlabBytes), w, j % OpQ::PER);
            }
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
    bf16x8 rp[OpP::HALF], rq[NQ][OpQ::HALF];
    auto fetch = [&](int h) {
        const int64_t k0 = (int64_t)h * kHalf;
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int j = 0; j < OpQ::HALF; ++j)
                rq[i][j] = OpQ::fetch(i ? Q2 : Q, ldq, n0, a.g.N, k0, a.g.K, j, threadIdx.x);
#pragma unroll
        for (int j = 0; j < OpP::HALF; ++j) rp[j] = OpP::fetch(P, ldp, m0, a.g.M, k0, a.g.K, j, threadIdx.x);
    };
    if (from < to) fetch(from);
    for (int h = from; h < to; ++h) {
        lds_barrier();  // everybody has read what was there
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int j = 0; j < OpQ::HALF; ++j)
                OpQ::store(smem + i * OpQ::kSlabBytes, h & 1, j, threadIdx.x, rq[i][j]);
#pragma unroll
        for (int j = 0; j < OpP::HALF; ++j) OpP::store(smem + NQ * OpQ::kSlabBytes, h & 1, j, threadIdx.x, rp[j]);
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
        write_rows<TN, ACT, MODE>(a, slice, mw, n0 + wn * (BN / NQ / 2), rows,
                                  reinterpret_cast<float*>(smem) + w * 32 * kPitch, lane);
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t up(size_t x) { return (x + 255) & ~size_t(255); }
int64_t whole_ld(int64_t cols) { return (cols + 7) / 8 * 8; }

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
}  // namespace mft
