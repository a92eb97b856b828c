// Log probabilities of given tokens, entropy and top alternatives (C ABI in
// include/mft/logprobs.h).
//
// Forward: one pass over a row keeps, per thread, the running maximum m and the
// sums S = sum exp(z - m) and T = sum exp(z - m) (z - m); then
//   log p(t) = (z_t - m) - log S,  entropy = log S - T / S.
// T is never positive and log S never negative, so nothing cancels.
//
// Alternatives.  The same pass gives each thread the first of its vectors that
// holds its maximum.  Ordered by value and then by place, the k-th of the
// threads' maxima bounds the row's k-th value from below, and only the k threads
// at or above it can hold one of the row's k largest.  Their vectors are read
// again (from the caches, by all threads of the workgroup), the values at or
// above the bound collected in LDS and sorted by one wave.  A value is a 64-bit
// key of its own, its bits in order above its complemented index, so the result
// does not depend on the order of collection.  A list of 64 keys, one per lane
// in falling order, merges with another by taking the larger of lane i of one
// and lane 63 - i of the other, which leaves the 64 largest in a bitonic order.
//
// Few rows are cut into parts, each a workgroup's, that a second launch joins.
// Bound by the one read of the logits (backward: one read, one write).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.h"
#include "logprobs_kernels.h"
#include "row_util.h"

namespace mft {
namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
// Vectors in flight per thread: 2048 rows of 50257 in fp32 with five alternatives, a
// tenth of them ignored and not read, 87 us with 2, 86 with 4, 79 with 8 (4.7 TB/s);
// 1000 of 262144 in bf16 103, 100 and 101.
constexpr int kUnroll = 8;
constexpr int kBwdVecs = 4;  // of a thread of the backward's workgroups
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
constexpr float kLowest = -1e30f;  // in place of -inf in a product with a probability of 0
constexpr float kGone = -1e6f;     // exp is 0 from here down, and its product with a sum (at most 2^30) finite

struct Sums {
    float m = -INFINITY, s = 0.f, t = 0.f;
    // The sums about a larger maximum.  Logits excluded by a type's lowest value are up to
    // 3.4e38 below it: their s (m - to) would overflow, and f = 0 make NaN of that.
    __device__ __forceinline__ void move_to(float to) {
        if (m != -INFINITY) {  // else s and t are 0, or the NaN of a value
            const float f = __expf(m - to);
            t = f * fmaf(s, fmaxf(m - to, kGone), t);
            s *= f;
        }
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        const float d = x - (m == -INFINITY ? 0.f : m), e = __expf(d);
        s += e;
        t = fmaf(e, fmaxf(d, kLowest), t);
    }
    __device__ __forceinline__ void join(Sums o) {
        const float to = fmaxf(m, o.m);
        move_to(to);
        o.move_to(to);
        s += o.s;
        t += o.t;
    }
};
// The sums of all lanes, in every lane.
__device__ __forceinline__ Sums join_wave(Sums x, int lane) {
    auto with = [&](auto o) {
        constexpr int O = decltype(o)::value;
        Sums r;
        r.m = __uint_as_float(lane_xor<O>(__float_as_uint(x.m), lane));
        r.s = __uint_as_float(lane_xor<O>(__float_as_uint(x.s), lane));
        r.t = __uint_as_float(lane_xor<O>(__float_as_uint(x.t), lane));
        x.join(r);
    };
    with(std::integral_constant<int, 32>{});
    with(std::integral_constant<int, 16>{});
    with(std::integral_constant<int, 8>{});
    with(std::integral_constant<int, 4>{});
    with(std::integral_constant<int, 2>{});
    with(std::integral_constant<int, 1>{});
    return x;
}

// Value and place as a key: larger values first, then lower places.  0: none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t place) {
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~place;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return ~(uint32_t)key; }

template <int O> __device__ __forceinline__ uint64_t key_xor(uint64_t x, int lane) {
    const uint32_t lo = lane_xor<O>((uint32_t)x, lane), hi = lane_xor<O>((uint32_t)(x >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
// Lanes O apart in order, the larger first where `falling`.
template <int O> __device__ __forceinline__ uint64_t exchange(uint64_t x, int lane, bool falling) {
    const uint64_t y = key_xor<O>(x, lane);
    return (((lane & O) == 0) == falling) == (x > y) ? x : y;
}
// Runs of 2 N lanes that are bitonic, in falling order or (`falling` false in some lanes' run) rising.
template <int N> __device__ __forceinline__ uint64_t sort_runs(uint64_t x, int lane, bool falling) {
    x = exchange<N>(x, lane, falling);
    if constexpr (N > 1) x = sort_runs<N / 2>(x, lane, falling);
    return x;
}
// Bitonic keys of a wave in falling order.
__device__ __forceinline__ uint64_t sort_bitonic(uint64_t x, int lane) { return sort_runs<32>(x, lane, true); }
// The wave's keys in falling order.
__device__ __forceinline__ uint64_t sort_wave(uint64_t x, int lane) {
    x = sort_runs<1>(x, lane, (lane & 2) == 0);
    x = sort_runs<2>(x, lane, (lane & 4) == 0);
    x = sort_runs<4>(x, lane, (lane & 8) == 0);
    x = sort_runs<8>(x, lane, (lane & 16) == 0);
    x = sort_runs<16>(x, lane, (lane & 32) == 0);
    return sort_runs<32>(x, lane, true);
}
// The 64 largest of a list in falling order and of other[0 .. n - 1], in falling order as well.
__device__ __forceinline__ uint64_t merge_list(uint64_t x, const uint64_t* other, int n, int lane) {
    const uint64_t y = 63 - lane < n ? other[63 - lane] : 0;
    return sort_bitonic(x > y ? x : y, lane);
}

// Elements from p to the next 16-byte boundary.
template <typename T> __device__ __forceinline__ int to_boundary(const T* p) {
    return (int)(-(reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (kVec<T> - 1));
}

// The row's results from its sums and its alternatives' keys (lane i of the
// calling wave holds the i-th).
template <typename T>
__device__ __forceinline__ void finish_row(const LogprobsArgs& a, int64_t n, const Sums& r, uint64_t best, int lane) {
    const float log_s = logf(r.s);
    if (lane == 0) {
        const int y = a.tokens[n];
        const bool in = y >= 0 && y < a.V;
        a.logprob[n] = in ? ((float)((const T*)a.z)[n * a.ld + y] - r.m) - log_s : NAN;
        if (!in && a.status) *a.status = 1;
        if (a.entropy) a.entropy[n] = log_s - r.t / r.s;
        if (a.stats) a.stats[n] = make_float2(r.m, log_s);
    }
    if (lane < a.top) {
        a.top_logprobs[n * a.top + lane] = best ? (value_of(best) - r.m) - log_s : NAN;
        a.top_ids[n * a.top + lane] = best ? (int32_t)place_of(best) : -1;
    }
}
__device__ __forceinline__ void skip_row(const LogprobsArgs& a, int64_t n, int lane) {
    if (lane == 0) {
        a.logprob[n] = 0.f;
        if (a.entropy) a.entropy[n] = 0.f;
        if (a.stats) a.stats[n] = make_float2(0.f, 0.f);
    }
    if (lane < a.top) {
        a.top_logprobs[n * a.top + lane] = -INFINITY;
        a.top_ids[n * a.top + lane] = -1;
    }
}

// One workgroup to a row, or (SPLIT) to a part of one.
template <typename T, bool TOP, bool SPLIT>
__global__ __launch_bounds__(kLpThreads) void lp_fwd(LogprobsArgs a) {
    constexpr int V = kVec<T>, NT = kLpThreads, kRound = NT * V, kCand = kRound + 256;
    typedef typename AnyVec<T, V>::raw raw;
    __shared__ float sm[kLpWaves], ss[kLpWaves], st[kLpWaves];
    __shared__ uint64_t lists[TOP ? kLpWaves : 1][64], cand[TOP ? kCand : 1], bound;
    __shared__ int owners[kLogprobsMaxTop], n_owners, n_cand;
    const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
    const int64_t n = SPLIT ? blockIdx.x / (unsigned)a.parts : blockIdx.x;
    const int part = SPLIT ? (int)(blockIdx.x % (unsigned)a.parts) : 0;
    if (a.tokens[n] == a.ignore) {
        if (!SPLIT && w == 0) skip_row(a, n, lane);
        return;
    }
    const int64_t lo = SPLIT ? part * a.per_part : 0;
    const T* row = (const T*)a.z + n * a.ld + lo;
    const int len = (int)((SPLIT ? min(lo + a.per_part, a.V) : a.V) - lo);
    const int nvec = len / V, rest = len - nvec * V;  // vectors from the row's first element on, and what is left
    auto vec_place = [&](int j) { return (uint32_t)(lo + j * V); };
    auto rest_at = [&](int i) { return nvec * V + i; };

    Sums r;
    int at = -1;  // the first vector with the thread's maximum
    auto take = [&](const raw& q, int j) {
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (float)q[e];
        float vm = x[0];
#pragma unroll
        for (int e = 1; e < V; ++e) vm = fmaxf(vm, x[e]);
        if (vm > r.m || (TOP && at < 0 && vm == r.m)) {
            r.move_to(vm);
            at = j;
        }
        const float base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = x[e] - base, p = __expf(d);
            r.s += p;
            r.t = fmaf(p, fmaxf(d, kLowest), r.t);
        }
    };
    int j = tid;
    for (; j + (kUnroll - 1) * NT < nvec; j += kUnroll * NT) {
        raw q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = *reinterpret_cast<const raw*>(row + (j + u * NT) * (int64_t)V);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) take(q[u], j + u * NT);
    }
    for (; j < nvec; j += NT) take(*reinterpret_cast<const raw*>(row + j * (int64_t)V), j);
    uint64_t best = at >= 0 ? key_of(r.m, vec_place(at)) : 0;
    if (tid < rest) {
        const float x = (float)row[rest_at(tid)];
        if (x > r.m) r.move_to(x);
        r.add(x);
        if (x == x) best = max(best, key_of(x, (uint32_t)(lo + rest_at(tid))));
    }

    r = join_wave(r, lane);
    if (lane == 0) sm[w] = r.m, ss[w] = r.s, st[w] = r.t;
    if constexpr (TOP) {
        if (tid == 0) n_owners = n_cand = 0;
        uint64_t k = sort_wave(best, lane);
        lists[w][lane] = k;
        __syncthreads();
        if (w < 2) k = merge_list(k, lists[w + 2], 64, lane);
        if (w == 1) lists[1][lane] = k;
        __syncthreads();
        if (w == 0) {
            k = merge_list(k, lists[1], 64, lane);
            if (lane == a.top - 1) bound = k;
        }
    }
    __syncthreads();
    r = Sums{};
#pragma unroll
    for (int i = 0; i < kLpWaves; ++i) {
        Sums o;
        o.m = sm[i], o.s = ss[i], o.t = st[i];
        r.join(o);
    }

    uint64_t list = 0;
    if constexpr (TOP) {
        const uint64_t least = bound;
        if (best != 0 && best >= least) owners[atomicAdd(&n_owners, 1)] = tid;  // at most `top`: keys are distinct
        __syncthreads();
        const int per = (nvec + NT - 1) / NT + 1, items = n_owners * per;  // a thread's vectors, and its single element
        for (int i0 = 0; i0 < items; i0 += NT) {
            const int i = i0 + tid;
            if (i < items) {
                const int o = owners[i / per], step = i % per, v = o + step * NT;
                if (step < per - 1) {
                    if (v < nvec) {
                        float x[V];
                        AnyVec<T, V>::load(row + v * (int64_t)V, x);
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (x[e] == x[e] && key_of(x[e], vec_place(v)) >= least)
                                cand[atomicAdd(&n_cand, 1)] = key_of(x[e], vec_place(v) + e);
                    }
                } else if (o < rest) {
                    const float x = (float)row[rest_at(o)];
                    const uint64_t k = key_of(x, (uint32_t)(lo + rest_at(o)));
                    if (x == x && k >= least) cand[atomicAdd(&n_cand, 1)] = k;
                }
            }
            __syncthreads();
            const int got = n_cand;
            if (got > kCand - kRound || i0 + NT >= items) {
                if (w == 0)
                    for (int c = 0; c < got; c += 64) {
                        const uint64_t y = sort_wave(c + lane < got ? cand[c + lane] : 0, lane), z = key_xor<63>(y, lane);
                        list = sort_bitonic(list > z ? list : z, lane);
                    }
                __syncthreads();
                if (tid == 0) n_cand = 0;
            }
            __syncthreads();
        }
    }
    if (w != 0) return;
    if constexpr (SPLIT) {
        const int64_t at_part = n * a.parts + part;
        if (lane == 0) a.part[at_part] = make_float4(r.m, r.s, r.t, 0.f);
        if (TOP && lane < a.top) a.part_keys[at_part * a.top + lane] = list;
    } else {
        finish_row<T>(a, n, r, list, lane);
    }
}

// The parts of a row (at most 64: one per lane).  16 waves merge the parts' lists
// in turn, then each other's.
constexpr int kJoinWaves = 16;
template <typename T> __global__ __launch_bounds__(64 * kJoinWaves) void lp_join(LogprobsArgs a) {
    __shared__ uint64_t lists[kJoinWaves][64];
    const int64_t n = blockIdx.x;
    const int lane = threadIdx.x & 63, w = wave_id();
    if (a.tokens[n] == a.ignore) {
        if (w == 0) skip_row(a, n, lane);
        return;
    }
    uint64_t list = 0;
    if (a.top > 0) {
        const uint64_t* keys = a.part_keys + n * a.parts * a.top;
        for (int i = w; i < a.parts; i += kJoinWaves)
            list = i == w ? (lane < a.top ? keys[i * a.top + lane] : 0) : merge_list(list, keys + i * a.top, a.top, lane);
        lists[w][lane] = list;
#pragma unroll
        for (int half = kJoinWaves / 2; half > 0; half /= 2) {
            __syncthreads();
            if (w < half) lists[w][lane] = list = merge_list(list, lists[w + half], 64, lane);
        }
    }
    if (w != 0) return;
    Sums r;
    if (lane < a.parts) {
        const float4 p = a.part[n * a.parts + lane];
        r.m = p.x, r.s = p.y, r.t = p.z;
    }
    r = join_wave(r, lane);
    finish_row<T>(a, n, r, list, lane);
}

// One workgroup to `per_part` elements of a row.
template <typename T> __global__ __launch_bounds__(kLpThreads) void lp_bwd(LogprobsArgs a) {
    constexpr int V = kVec<T>, NT = kLpThreads;
    const int64_t n = blockIdx.x / (unsigned)a.parts, lo = blockIdx.x % (unsigned)a.parts * a.per_part;
    const int len = (int)(min(lo + a.per_part, a.V) - lo);
    const T* z = (const T*)a.z + n * a.ld + lo;
    T* g = (T*)a.grad + n * a.ldg + lo;
    const int head = min(to_boundary(g), len), nvec = (len - head) / V, rest = len - nvec * V;
    const int y = a.tokens[n];
    const bool on = y != a.ignore && y >= 0 && y < a.V;
    float gl = 0.f, ge = 0.f, entropy = 0.f;
    float2 s = make_float2(0.f, 0.f);
    if (on) {
        if (a.grad_logprob) gl = a.grad_logprob[n];
        if (a.grad_entropy) ge = a.grad_entropy[n], entropy = a.entropy_in[n];
        s = a.stats_in[n];
    }
    const int64_t yl = on ? y - lo : -1;
    auto grad = [&](float x, int i) {
        const float q = (x - s.x) - s.y, p = __expf(q);
        const float v = p == 0.f ? 0.f : -p * fmaf(ge, q + entropy, gl);  // no 0 * inf, and a NaN stays
        return i == yl ? v + gl : v;
    };
    for (int j = threadIdx.x; j < nvec; j += NT) {
        float x[V] = {};
        const int i = head + j * V;
        if (on) {
            AnyVec<T, V>::load(z + i, x);
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = grad(x[e], i + e);
        }
        AnyVec<T, V>::store(g + i, x);
    }
    if ((int)threadIdx.x < rest) {
        const int i = (int)threadIdx.x < head ? (int)threadIdx.x : nvec * V + (int)threadIdx.x;
        g[i] = (T)(on ? grad((float)z[i], i) : 0.f);
    }
}

// Parts of a row: until four workgroups a CU run, none under kMinPart elements.
constexpr int64_t kMinPart = 4096, kMaxParts = 64;
void cut(int64_t N, int64_t V, int* parts, int64_t* per_part) {
    const int64_t want = std::min<int64_t>({kMaxParts, 4 * device_cus() / std::max<int64_t>(N, 1), V / kMinPart});
    int64_t p = std::max<int64_t>(1, want);
    *per_part = ((V + p - 1) / p + 63) / 64 * 64;
    *parts = (int)((V + *per_part - 1) / *per_part);
}

template <typename T> hipError_t fwd(const LogprobsArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.N * a.parts)), block(kLpThreads);
    if (a.parts > 1) {
        if (a.top) hipLaunchKernelGGL((lp_fwd<T, true, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((lp_fwd<T, false, true>), grid, block, 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((lp_join<T>), dim3((unsigned)a.N), dim3(64 * kJoinWaves), 0, st, a);
    } else if (a.top) {
        hipLaunchKernelGGL((lp_fwd<T, true, false>), grid, block, 0, st, a);
    } else {
        hipLaunchKernelGGL((lp_fwd<T, false, false>), grid, block, 0, st, a);
    }
    return hipGetLastError();
}

size_t up(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

size_t logprobs_workspace(int64_t N, int64_t V, int top) {
    int parts;
    int64_t per;
    cut(N, V, &parts, &per);
    return parts > 1 ? up((size_t)N * parts * sizeof(float4)) + (size_t)N * parts * top * 8 : 0;
}

hipError_t launch_logprobs_fwd(LogprobsArgs a, bool is_bf16, void* workspace, hipStream_t st) {
    if (a.N == 0) return hipSuccess;
    cut(a.N, a.V, &a.parts, &a.per_part);
    a.part = static_cast<float4*>(workspace);
    a.part_keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) +
                                              up((size_t)a.N * a.parts * sizeof(float4)));
    return is_bf16 ? fwd<bf16>(a, st) : fwd<float>(a, st);
}

hipError_t launch_logprobs_bwd(const LogprobsArgs& args, bool is_bf16, hipStream_t st) {
    if (args.N == 0) return hipSuccess;
    LogprobsArgs a = args;
    a.per_part = (int64_t)kLpThreads * kBwdVecs * (is_bf16 ? kVec<bf16> : kVec<float>);
    // a launch takes fewer than 2^32 threads
    while (a.N * ((a.V + a.per_part - 1) / a.per_part) >= (int64_t(1) << 32) / kLpThreads) a.per_part *= 2;
    a.parts = (int)((a.V + a.per_part - 1) / a.per_part);
    const dim3 grid((unsigned)(a.N * a.parts));
    if (is_bf16) hipLaunchKernelGGL((lp_bwd<bf16>), grid, dim3(kLpThreads), 0, st, a);
    else hipLaunchKernelGGL((lp_bwd<float>), grid, dim3(kLpThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace mft
