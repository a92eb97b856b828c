// One AdamW step over many tensors (C ABI in include/mft/adamw.h).
//
// Bound by memory: in fp32 28 bytes a value (the gradient and three values read,
// three written), with 8-bit states and a bf16 parameter 16.  A block's 27 M values in
// fp32 127 us (6.0 TB/s, part of it from the last-level cache) and 36 for the sums of
// squares; a bf16 table of 168 M with 8-bit states 493 us (5.5 TB/s).
//
// The tensors are cut into chunks of whole groups of 256 values, a workgroup to a
// chunk.  A launch's tensors lie in its arguments, which the host fills and a
// captured graph keeps: no table is copied to the device.  Each wave finds its
// chunk's tensor by comparing the chunk's number with the tensors' first chunks, a
// lane each.
//
// Three kinds of launches: the sums of the gradients' squares (with clipping
// only), each workgroup's to a place of its own; one workgroup that adds them in
// their order, counts the step and leaves the step's factors; the step itself.
#include "adamw_kernels.h"

#include <algorithm>
#include <cmath>

#include "attn_geometry.h"
#include "attn_kernels.h"
#include "e4m3.h"
#include "row_util.h"

namespace mft {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kGroup = MFT_ADAMW_GROUP;
static_assert(kGroup == 64 * 4, "a wave holds a group, four values a lane");

// A launch's tensors: as many as a wave has lanes, in less than 4 KiB of arguments.
template <int BITS> struct Entry {
    int64_t n;
    float* p;
    bf16* p16;  // or null
    const void* g;
    void* m;
    void* v;
    float decay;
    int first;  // chunk
};
template <> struct Entry<8> {
    int64_t n;
    float* p;
    bf16* p16;
    const void* g;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    float decay;
    int first;
};
template <int BITS> constexpr int kEntries = BITS == 32 ? 64 : 48;
struct Factors {
    float lr, step_size;  // lr / (1 - beta1^t)
    float root;           // 1 / sqrt(1 - beta2^t)
    float clip;
};
template <int BITS> struct Args {
    Entry<BITS> t[kEntries<BITS>];
    const Factors* f;
    float beta1, rest1, beta2, rest2, eps;
    int count;
    int64_t chunk;  // values, whole groups
};
// The same of the sums of squares.
struct Gradient {
    int64_t n;
    const void* g;
    const void* p16;  // or null: fp32
    int first;
};
constexpr int kGradients = 120;
struct SquaresArgs {
    Gradient t[kGradients];
    double* sums;  // a workgroup each
    int count;
    int64_t chunk;
};
static_assert(sizeof(Args<32>) <= 4000 && sizeof(Args<8>) <= 4000 && sizeof(SquaresArgs) <= 4000, "a launch's arguments");

// This workgroup's tensor, and its values from *from on up to *to.
template <typename A> __device__ __forceinline__ int place(const A& a, int64_t* from, int64_t* to) {
    constexpr int most = (int)(sizeof(a.t) / sizeof(a.t[0]));
    const int lane = threadIdx.x & 63, b = (int)blockIdx.x;
    int before = 0;
#pragma unroll
    for (int i = lane; i < (most + 63) / 64 * 64; i += 64)
        before += __popcll(__ballot(i < a.count && a.t[i < a.count ? i : 0].first <= b));
    const int i = __builtin_amdgcn_readfirstlane(before - 1);
    *from = (int64_t)(b - a.t[i].first) * a.chunk;
    *to = min(*from + a.chunk, a.t[i].n);
    return i;
}

// Four consecutive gradients as floats; zeros past `n`.
template <typename E> __device__ __forceinline__ void load4(const E& t, int64_t i, float* g) {
    if (t.p16) load_part<bf16, 4>((const bf16*)t.g, i, t.n, g);
    else load_part<float, 4>((const float*)t.g, i, t.n, g);
}

__global__ __launch_bounds__(kThreads) void adamw_squares(SquaresArgs a) {
    __shared__ double s[kThreads];
    int64_t from, to;
    const int k = place(a, &from, &to);
    double sum = 0.0;
#pragma unroll 4
    for (int64_t i = from + threadIdx.x * 4; i < to; i += kThreads * 4) {
        float g[4];
        load4(a.t[k], i, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fma((double)g[e], (double)g[e], sum);
    }
    s[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int o = kThreads / 2; o > 0; o /= 2) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.sums[blockIdx.x] = s[0];
}

struct StepArgs {
    int64_t* step;
    const float* lr_device;
    double lr, log_beta1, log_beta2, max_norm;  // 0: not clipped
    const double* sums;
    int count;
    float* norm;
    Factors* f;
};
constexpr int kStepThreads = 512;
__global__ __launch_bounds__(kStepThreads) void adamw_factors(StepArgs a) {
    __shared__ double s[kStepThreads];
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.count; i += kStepThreads) sum += a.sums[i];
    s[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int o = kStepThreads / 2; o > 0; o /= 2) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const int64_t t = *a.step + 1;
    *a.step = t;
    const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
    Factors f;
    f.lr = (float)lr;
    f.step_size = (float)(lr / -expm1((double)t * a.log_beta1));  // 1 - beta^t
    f.root = (float)(1.0 / sqrt(-expm1((double)t * a.log_beta2)));
    f.clip = 1.f;
    if (a.max_norm > 0.0) {
        const double norm = sqrt(s[0]), c = a.max_norm / (norm + 1e-6);
        f.clip = (float)(c > 1.0 ? 1.0 : c);  // a NaN stays
        if (a.norm) *a.norm = (float)norm;
    }
    *a.f = f;
}

// One value's step.  The averages are rounded as by torch's multi-tensor operations (the state times beta, then the
// gradient's share with one rounding): with the gradient's product rounded first 400 of 168 M 8-bit numbers of a step
// came out one off, where a quotient is halfway between two, and now and then a scale of the next step by percents.
template <int BITS>
__device__ __forceinline__ void update(const Args<BITS>& a, const Factors& f, float keep, float g, float& p, float& m,
                                       float& v, float& root) {
    g *= f.clip;
    m = fmaf(a.rest1, g, a.beta1 * m);
    v = fmaf(a.rest2 * g, g, a.beta2 * v);
    root = sqrtf(v);
    p = fmaf(p, keep, -f.step_size * (m / fmaf(root, f.root, a.eps)));
}

__global__ __launch_bounds__(kThreads) void adamw_step32(Args<32> a) {
    int64_t from, to;
    const Entry<32>& t = a.t[place(a, &from, &to)];
    const Factors f = *a.f;
    const float keep = 1.f - f.lr * t.decay;
    float *m = (float*)t.m, *v = (float*)t.v;
#pragma unroll 2
    for (int64_t i = from + threadIdx.x * 4; i < to; i += kThreads * 4) {
        float g[4], p[4], x[4], y[4];
        load4(t, i, g);
        load_part<float, 4>(t.p, i, t.n, p);
        load_part<float, 4>(m, i, t.n, x);
        load_part<float, 4>(v, i, t.n, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float root;
            update(a, f, keep, g[e], p[e], x[e], y[e], root);
        }
        store_part<float, 4>(t.p, i, t.n, p);
        store_part<float, 4>(m, i, t.n, x);
        store_part<float, 4>(v, i, t.n, y);
        if (t.p16) store_part<bf16, 4>(t.p16, i, t.n, p);
    }
}

// Four e4m3 numbers (or what is left before `n`) times a scale.
__device__ __forceinline__ void load_e4m3(const uint8_t* q, int64_t i, int64_t n, float scale, float* x) {
    typedef uint32_t any32 __attribute__((aligned(1)));
    uint32_t r = 0;
    if (i + 4 <= n) {
        r = *reinterpret_cast<const any32*>(q + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) r |= (uint32_t)q[i + e] << (8 * e);
    }
    e4m3_unpack4(r, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= scale;
}

// A wave's group of an 8-bit state; past the end m, v and g are zero and change nothing.
__global__ __launch_bounds__(kThreads) void adamw_step8(Args<8> a) {
    int64_t from, to;
    const Entry<8>& t = a.t[place(a, &from, &to)];
    const Factors f = *a.f;
    const float keep = 1.f - f.lr * t.decay;
    const int lane = threadIdx.x & 63;
    uint8_t *mq = (uint8_t*)t.m, *vq = (uint8_t*)t.v;
#pragma unroll 2
    for (int64_t i0 = from + wave_id() * kGroup; i0 < to; i0 += kWaves * kGroup) {
        const int64_t i = i0 + lane * 4, group = i0 / kGroup;
        float g[4] = {}, p[4] = {}, x[4] = {}, y[4] = {}, r[4];
        if (i < t.n) {
            load4(t, i, g);
            load_part<float, 4>(t.p, i, t.n, p);
            load_e4m3(mq, i, t.n, t.m_scale[group], x);
            load_e4m3(vq, i, t.n, t.v_scale[group], y);
        }
        uint32_t most_m = 0, most_r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] *= y[e];
            update(a, f, keep, g[e], p[e], x[e], y[e], r[e]);
            most_m = max(most_m, __float_as_uint(x[e]) & 0x7fffffffu);
            most_r = max(most_r, __float_as_uint(r[e]) & 0x7fffffffu);
        }
        const float ms = e4m3_scale(wave_max_u(most_m, lane)), rs = e4m3_scale(wave_max_u(most_r, lane));
        if (lane == 0) t.m_scale[group] = ms, t.v_scale[group] = rs;
        if (i >= t.n) continue;
        bool some[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) some[e] = r[e] > 0.f;
        E4m3Divisor(ms).divide<4>(x);
        E4m3Divisor(rs).divide<4>(r);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = some[e] && r[e] < kE4m3Min ? kE4m3Min : r[e];
        e4m3_store<4>(mq + i, t.n - i, x);
        e4m3_store<4>(vq + i, t.n - i, r);
        store_part<float, 4>(t.p, i, t.n, p);
        if (t.p16) store_part<bf16, 4>(t.p16, i, t.n, p);
    }
}

void fill(Entry<32>& e, const mft_adamw_tensor& t) {
    e.n = t.n, e.p = t.param, e.p16 = (bf16*)t.param_bf16, e.g = t.grad, e.m = t.exp_avg, e.v = t.exp_avg_sq;
    e.decay = (float)t.weight_decay;
}
void fill(Entry<8>& e, const mft_adamw_tensor& t) {
    e.n = t.n, e.p = t.param, e.p16 = (bf16*)t.param_bf16, e.g = t.grad, e.m = t.exp_avg, e.v = t.exp_avg_sq;
    e.m_scale = t.exp_avg_scale, e.v_scale = t.exp_avg_sq_scale;
    e.decay = (float)t.weight_decay;
}
void fill(Gradient& e, const mft_adamw_tensor& t) { e.n = t.n, e.g = t.grad, e.p16 = t.param_bf16; }
bool steps(const mft_adamw_tensor& t) { return t.n > 0 && t.grad; }

constexpr int64_t kSquares = 2048;  // workgroups of the sums of squares, but for one more a tensor

// Launches over all tensors in chunks of `chunk` values: launch(args, workgroups).
template <typename A, typename F>
void over(A& a, int32_t n, const mft_adamw_tensor* tensors, int64_t chunk, F launch) {
    a.chunk = chunk;
    a.count = 0;
    int64_t blocks = 0;
    auto flush = [&] {
        if (a.count) launch(a, (unsigned)blocks);
        a.count = 0, blocks = 0;
    };
    for (int32_t i = 0; i < n; ++i) {
        if (!steps(tensors[i])) continue;
        fill(a.t[a.count], tensors[i]);
        a.t[a.count].first = (int)blocks;
        blocks += (tensors[i].n + chunk - 1) / chunk;
        if (++a.count == (int)(sizeof(a.t) / sizeof(a.t[0]))) flush();
    }
    flush();
}

int64_t whole(int64_t values, int64_t least) {
    return std::max(least, (values + kGroup * kWaves - 1) / (kGroup * kWaves) * (kGroup * kWaves));
}

template <int BITS>
hipError_t run(const mft_adamw_desc& d, int32_t n, const mft_adamw_tensor* tensors, int64_t* step, float* norm,
               void* workspace, hipStream_t st) {
    int64_t total = 0;
    for (int32_t i = 0; i < n; ++i) total += steps(tensors[i]) ? tensors[i].n : 0;
    if (total == 0) return hipSuccess;
    Args<BITS> a{};
    a.f = static_cast<Factors*>(workspace);
    a.beta1 = (float)d.beta1, a.rest1 = (float)(1.0 - d.beta1);
    a.beta2 = (float)d.beta2, a.rest2 = (float)(1.0 - d.beta2);
    a.eps = (float)d.eps;
    double* sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
    int64_t count = 0;
    if (d.max_norm > 0.0) {
        SquaresArgs squares{};
        over(squares, n, tensors, whole((total + kSquares - 1) / kSquares, 4096), [&](SquaresArgs& q, unsigned blocks) {
            q.sums = sums + count;
            count += blocks;
            hipLaunchKernelGGL(adamw_squares, dim3(blocks), dim3(kThreads), 0, st, q);
        });
    }
    StepArgs s{step, d.lr_device, d.lr, std::log(d.beta1), std::log(d.beta2), d.max_norm, sums, (int)count, norm,
               static_cast<Factors*>(workspace)};
    hipLaunchKernelGGL(adamw_factors, dim3(1), dim3(kStepThreads), 0, st, s);
    // 2^22 workgroups at most: a launch takes fewer than 2^32 threads
    over(a, n, tensors, whole((total >> 21) + 1, 2048), [&](Args<BITS>& q, unsigned blocks) {
        if constexpr (BITS == 32) hipLaunchKernelGGL(adamw_step32, dim3(blocks), dim3(kThreads), 0, st, q);
        else hipLaunchKernelGGL(adamw_step8, dim3(blocks), dim3(kThreads), 0, st, q);
    });
    return hipGetLastError();
}

}  // namespace

size_t adamw_workspace(int32_t n) { return 256 + (size_t)(kSquares + n) * sizeof(double); }

hipError_t launch_adamw(const mft_adamw_desc& d, int32_t n, const mft_adamw_tensor* tensors, int64_t* step, float* norm,
                        void* workspace, hipStream_t st) {
    return d.state_bits == 32 ? run<32>(d, n, tensors, step, norm, workspace, st)
                              : run<8>(d, n, tensors, step, norm, workspace, st);
}

}  // namespace mft
