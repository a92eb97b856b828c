// The gated linear layer on e4m3 numbers with a scale a row (C ABI in
// include/mft/gated_linear.h): h = act(x_scale gate_scale x W_gate^T) (x_scale up_scale
// x W_up^T), all with k contiguous, in bf16.
//
// A workgroup of 2 x 2 waves owns a tile of BM rows by BN / 2 columns of h, both
// sums of a column in one lane, on v_mfma_f32_32x32x64_f8f6f4 (without block scales:
// a row's scale leaves the sum).  It multiplies 64 k in the time of 32 in bf16, so in
// bytes loads, LDS and matrix units are in the ratio of bf_gemm_tiles.h, whose slabs
// these are: [rows][128 bytes], direct loads, two of them in LDS.  The 32 bytes of a
// lane's fragment are two 16-byte reads; which k they hold is the same for all
// operands.
//
// A pair of halves of 64 k to a slab: while a half is multiplied the next one's
// fragments are read.  Behind the barrier after a slab's last reads the loads of the
// slab after the next go out into it.
//
// What the matrix unit keeps.  It adds the products of eight consecutive k first, each
// cut towards zero to a multiple of 2^-13 of 2^(a + b), a and b the exponents of the
// factors of the largest of them (measured; v_mfma_f32_32x32x16_fp8_fp8 does the
// same), and these sums and the accumulator in fp32.  A product is off by at most
// 2^-13 of its group's largest, where e4m3 itself rounds each factor by up to 2^-4;
// the bf16 units would keep all of it at half the rate.
//
// What is left of K after whole slabs, and operands off 16 bytes, go through
// registers.
#include "bf_gemm_tiles.h"
#include "e4m3.h"

namespace mft {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kRow = 128;  // bytes of a slab's row

struct E4m3Args {
    Args a;
    const float* x_scale;
    const float* gate_scale;
    const float* up_scale;
    int slabs;  // whole ones, by direct loads
};

// One operand of R rows in slabs of kRow bytes.
template <int R> struct Rows {
    static constexpr int kBytes = R * kRow, PER = kBytes / 1024 / 4;  // direct loads of a wave per slab
    uint32_t off[PER];  // this lane's bytes from a slab's first
    __device__ __forceinline__ void init(int w, int lane, int64_t r0, int64_t rows, int64_t ld) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = (w * PER + j) * 8 + lane / 8, c = lane % 8 ^ swz_kc(r);
            // rows past the end are read again from the last one, and not stored
            off[j] = (uint32_t)((min(r0 + r, rows - 1) - r0) * ld) + 16u * c;
        }
    }
    __device__ __forceinline__ void issue(const char* from, uint32_t to, int w, int j) const {
        load_lds_16_s(from, off[j], to + (uint32_t)(w * PER + j) * 1024u);
    }
    // The slab of bytes k0 .. k0 + 127 through registers, from anywhere and with zeros past K.
    __device__ __forceinline__ static void copy(char* to, const char* p, int64_t r0, int64_t rows, int64_t K, int64_t k0,
                                                int tid) {
        typedef i32x4 any16 __attribute__((aligned(1)));
#pragma unroll 4
        for (int i = tid; i < R * 8; i += kThreads) {
            const int r = i / 8, c = i % 8;
            const char* q = p + min(r0 + r, rows - 1) * K + k0 + 16 * c;
            const int64_t left = K - k0 - 16 * c;
            i32x4 v{};
            if (left >= 16) {
                v = *reinterpret_cast<const any16*>(q);
            } else {
                for (int e = 0; e < left; ++e) v[e / 4] |= (int)((uint32_t)(uint8_t)q[e] << (8 * (e & 3)));
            }
            *reinterpret_cast<i32x4*>(to + r * kRow + (c ^ swz_kc(r)) * 16) = v;
        }
    }
};

// 32 rows of h from mw on, 16 TN columns from nw on, through this wave's LDS.
template <int TN>
__device__ __forceinline__ void write_h(const E4m3Args& a, int64_t mw, int64_t nw, const f32x16 (&acc)[TN], float* st,
                                        int lane) {
    constexpr int COLS = 16 * TN, kPitch = 2 * COLS + 4;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(st + (lane & 31) * kPitch + 32 * j + 8 * q + 4 * (lane >> 5)) =
                f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    asm volatile("" ::: "memory");  // a wave's LDS accesses stay in order
    gated_rows_out<COLS, kPitch, true>(a.a.g, mw, nw, st, lane, a.x_scale, a.gate_scale, a.up_scale);
    asm volatile("" ::: "memory");
}

template <int BN, int BM>
__global__ __launch_bounds__(kThreads, BN * BM > 32768 ? 1 : 2) void gated_e4m3_kernel(E4m3Args a) {
    constexpr int RING = 2;
    constexpr int TN = BN / 64, TM = BM / 64, TQ = TN / 2, kTiles = TN * TM, kFrags = TN + TM;
    typedef Rows<BM> OpP;
    typedef Rows<BN / 2> OpQ;
    constexpr int kSlabBytes = 2 * OpQ::kBytes + OpP::kBytes, PER = 2 * OpQ::PER + OpP::PER;
    constexpr int kPitch = 32 * TN + 4, kStaged = 4 * 32 * kPitch * 4;
    // [slab][W_gate, W_up, x]
    __shared__ __attribute__((aligned(1024))) char smem[RING * kSlabBytes > kStaged ? RING * kSlabBytes : kStaged];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wn = w & 1, wm = w >> 1;
    int slice;
    int64_t m0, n0;
    place<BN / 2, BM>(a.a, &slice, &m0, &n0);
    const LinearProduct& g = a.a.g;
    const char *P = (const char*)g.P, *Q = (const char*)g.Q, *Q2 = (const char*)g.Q2;
    // Chunk i of 16 bytes of this lane's two a half: its place in the first of its rows.
    uint32_t at_p[4], at_q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = lane & 31, c = ((2 * i + (lane >> 5)) ^ swz_kc(n)) * 16;
        at_p[i] = (uint32_t)((wm * BM / 2 + n) * kRow + c);
        at_q[i] = (uint32_t)((wn * BN / 4 + n) * kRow + c);
    }
    f32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int k = 0; k < TM; ++k) {
            acc[j][k] = zero16();
            // not a literal zero (see mfma_v_first)
            if constexpr (kTiles > 8) asm volatile("" : "+a"(acc[j][k]));
            else asm volatile("" : "+v"(acc[j][k]));
        }
    struct Ops {
        i32x8 q[TN], p[TM];
    };
    // Fragment f of the half `odd` of a slab.
    auto read_one = [&](Ops& o, int slot, int odd, int f) {
        const char* s = smem + slot * kSlabBytes;
        const bool is_p = f < TM;
        const int t = is_p ? f : f - TM;
        const char* r = is_p ? s + 2 * OpQ::kBytes + t * 32 * kRow : s + t / TQ * OpQ::kBytes + t % TQ * 32 * kRow;
        const i32x4 lo = *reinterpret_cast<const i32x4*>(r + (is_p ? at_p : at_q)[2 * odd]);
        const i32x4 hi = *reinterpret_cast<const i32x4*>(r + (is_p ? at_p : at_q)[2 * odd + 1]);
        (is_p ? o.p[t] : o.q[t]) = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto multiply_one = [&](const Ops& o, int t) {
        acc[t / TM][t % TM] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(o.q[t / TM], o.p[t % TM],
                                                                              acc[t / TM][t % TM], 0, 0, 0, 0, 0, 0);
    };
    // A half's MFMAs, with the next half's fragment reads and a slab's loads between them.
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
    const int slabs = a.slabs;
    if (slabs > 0) {
        OpP dp;
        OpQ dq;
        dp.init(w, lane, m0, g.M, g.K);
        dq.init(w, lane, n0, g.N, g.K);
        const char *tp = P + m0 * g.K, *tq = Q + n0 * g.K, *tq2 = Q2 + n0 * g.K;
        const uint32_t base = lds_addr(smem);
        auto issue_one = [&](int p, int slot, int j) {
            const uint32_t to = base + (uint32_t)(slot * kSlabBytes);
            if (j < OpQ::PER) dq.issue(tq + (int64_t)p * kRow, to, w, j);
            else if (j < 2 * OpQ::PER) dq.issue(tq2 + (int64_t)p * kRow, to + OpQ::kBytes, w, j - OpQ::PER);
            else dp.issue(tp + (int64_t)p * kRow, to + 2 * OpQ::kBytes, w, j - 2 * OpQ::PER);
        };
#pragma unroll
        for (int i = 0; i < RING; ++i)
            if (i < slabs)
#pragma unroll
                for (int j = 0; j < PER; ++j) issue_one(i, i, j);
        if (slabs >= RING) wait_vmcnt<(RING - 1) * PER>();
        else wait_vmcnt<0>();
        lds_barrier();
        Ops cur, nxt;
#pragma unroll
        for (int f = 0; f < kFrags; ++f) read_one(cur, 0, 0, f);
        // MORE: slab p + RING exists.
        auto slab = [&](int p, int slot, auto more_t) {
            constexpr bool MORE = decltype(more_t)::value;
            const int after = slot + 1 == RING ? 0 : slot + 1;
            weave(cur, [&](int f) { read_one(nxt, slot, 1, f); }, [](int) {});
            // Slab p + 1 has landed, and everybody has read slab p.
            if constexpr (MORE) wait_vmcnt<(RING - 2) * PER>();
            else wait_vmcnt<0>();
            lds_barrier();
            weave(nxt, [&](int f) { if (MORE || p + 1 < slabs) read_one(cur, after, 0, f); },
                  [&](int t) {
                      if constexpr (MORE) {
#pragma unroll
                          for (int j = t * PER / kTiles; j < (t + 1) * PER / kTiles; ++j) issue_one(p + RING, slot, j);
                      }
                  });
        };
        int p = 0, slot = 0;
        for (; p + RING < slabs; ++p) {
            slab(p, slot, std::true_type{});
            slot = slot + 1 == RING ? 0 : slot + 1;
        }
        for (; p < slabs; ++p) {
            slab(p, slot, std::false_type{});
            slot = slot + 1 == RING ? 0 : slot + 1;
        }
    }
    for (int64_t k0 = (int64_t)slabs * kRow; k0 < g.K; k0 += kRow) {
        lds_barrier();  // everybody has read what was there
        OpQ::copy(smem, Q, n0, g.N, g.K, k0, threadIdx.x);
        OpQ::copy(smem + OpQ::kBytes, Q2, n0, g.N, g.K, k0, threadIdx.x);
        OpP::copy(smem + 2 * OpQ::kBytes, P, m0, g.M, g.K, k0, threadIdx.x);
        lds_barrier();
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            Ops o;
#pragma unroll
            for (int f = 0; f < kFrags; ++f) read_one(o, 0, odd, f);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) multiply_one(o, t);
        }
    }
    lds_barrier();  // the slabs have been read
    float* st = reinterpret_cast<float*>(smem) + w * 32 * kPitch;
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        const int64_t mw = m0 + wm * (BM / 2) + 32 * k;
        if (mw >= g.M) break;
        f32x16 rows[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) rows[j] = acc[j][k];
        write_h<TN>(a, mw, n0 + wn * (BN / 4), rows, st, lane);
    }
}

// The tiles (columns of both sums together), the workgroups that a CU holds, and
// what one takes in us: with one to a CU at, and with more, a + b K.  Fitted to 41
// sizes of 16 to 8192 rows and 640 to 8192 columns.  8192 x 1152 -> 6912 151 us in 128 x
// 192, 169 in 128 x 128, 182 in 256 x 256, whose epilogue nothing hides; 4096 x 4096
// -> 8192 254, 294 and 236: over long k it reads LDS least.  256 rows of it 25 us in 128 x
// 64, 28 in 128 x 128, 45 in 256 x 256.
struct Shape {
    int bn, bm, at_once;
    double one_a, one_b, a, b;
};
constexpr Shape kShapes[] = {{256, 256, 1, 14, 0.0109, 14, 0.0109}, {128, 192, 2, 7.5, 0.0080, 7.5, 0.0091},
                             {128, 128, 2, 6, 0.0054, 4.4, 0.0079}, {128, 64, 3, 5.4, 0.0047, 2.5, 0.0071}};
int shape_of(const LinearProduct& g) {
    const double cus = device_cus();
    int best = 0;
    double least = 1e300;
    for (int i = 0; i < 4; ++i) {
        const Shape& t = kShapes[i];
        const double tiles = (double)((2 * g.N + t.bn - 1) / t.bn) * ((g.M + t.bm - 1) / t.bm);
        const double rounds = std::max(1.0, tiles / (cus * t.at_once));
        const double us = tiles <= cus ? t.one_a + t.one_b * g.K : (std::ceil(rounds) + rounds) / 2 * (t.a + t.b * g.K);
        if (us < least) least = us, best = i;
    }
    return best;
}

template <int BN, int BM> hipError_t launch_t(E4m3Args a, hipStream_t st) {
    a.a.tiles_m = (int)((a.a.g.M + BM - 1) / BM);
    a.a.tiles_n = (int)((2 * a.a.g.N + BN - 1) / BN);
    a.a.per_slice_tiles = FastDiv::make((uint32_t)(a.a.tiles_m * a.a.tiles_n));
    hipLaunchKernelGGL((gated_e4m3_kernel<BN, BM>), dim3((unsigned)(a.a.tiles_m * a.a.tiles_n)), dim3(kThreads), 0,
                       st, a);
    return hipGetLastError();
}

// rows of K bytes into rows of ld (a multiple of 16), zeros behind them.
__global__ __launch_bounds__(256) void pack_bytes(const uint8_t* from, uint8_t* to, int64_t rows, int64_t K, int64_t ld) {
    typedef uint32_t word __attribute__((ext_vector_type(4)));
    typedef word any16 __attribute__((aligned(1)));
    const int64_t chunks = ld / 16, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * chunks; i += step) {
        const int64_t r = i / chunks, c = (i - r * chunks) * 16;
        word v{};
        if (c + 16 <= K) {
            v = *reinterpret_cast<const any16*>(from + r * K + c);
        } else {
            for (int e = 0; c + e < K; ++e) v[e / 4] |= (uint32_t)from[r * K + c + e] << (8 * (e & 3));
        }
        *reinterpret_cast<word*>(to + r * ld + c) = v;
    }
}

int64_t whole_row(int64_t K) { return (K + kRow - 1) / kRow * kRow; }
bool off_rows(const LinearProduct& g) { return g.K % 16 != 0; }

}  // namespace

size_t gated_e4m3_workspace(const LinearProduct& g) {
    return off_rows(g) ? up((size_t)g.M * whole_row(g.K)) + 2 * up((size_t)g.N * whole_row(g.K)) : 0;
}

hipError_t launch_gated_e4m3(const LinearProduct& given, const float* x_scale, const float* gate_scale,
                             const float* up_scale, hipStream_t st) {
    LinearProduct g = given;
    if (g.M <= 0 || g.N <= 0 || g.K <= 0) return hipSuccess;
    if (off_rows(g)) {  // rows off 16 bytes are copied to whole slabs
        const int64_t ld = whole_row(g.K);
        const void** from[3] = {&g.P, &g.Q, &g.Q2};
        uint8_t* to = reinterpret_cast<uint8_t*>(g.partial);
        for (int i = 0; i < 3; ++i) {
            const int64_t rows = i ? g.N : g.M, n = rows * (ld / 16);
            hipLaunchKernelGGL(pack_bytes, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 16 * device_cus())), dim3(256),
                               0, st, (const uint8_t*)*from[i], to, rows, g.K, ld);
            *from[i] = to;
            to += up((size_t)rows * ld);
        }
        g.K = ld;
    }
    E4m3Args a{};
    a.a.g = g;
    a.x_scale = x_scale, a.gate_scale = gate_scale, a.up_scale = up_scale;
    a.slabs = on16(g.P) && on16(g.Q) && on16(g.Q2) && g.K <= (1 << 23) ? (int)(g.K / kRow) : 0;
    switch (shape_of(g)) {
        case 0: return launch_t<256, 256>(a, st);
        case 1: return launch_t<128, 192>(a, st);
        case 2: return launch_t<128, 128>(a, st);
        default: return launch_t<128, 64>(a, st);
    }
}

}  // namespace mft
