// Which kernels the products of the gated linear layer and the rows of the RMS norm take, on the host: one line
// of entries for each line of sizes on stdin.  The planners are those of the source itself, which is included whole (OF:
// GATED, E4M3, F32 or RMS says which); without a GPU they assume 256 CUs.  Linked against libmft_attn.so and
// run by tests/test_block_plans.py.
#include <cstdio>

#if defined(OF_GATED)
#include "gated_gemm.hip"
#elif defined(OF_E4M3)
#include "gated_e4m3.hip"
#elif defined(OF_F32)
#include "gemm_f32.hip"
#elif defined(OF_RMS)
#include "rms_norm.hip"
#endif

using namespace mft;

int main() {
#if defined(OF_RMS)
    // D: a row's waves and chunks of a thread (0: by memory), and whether its vectors are whole
    long long D;
    while (std::scanf("%lld", &D) == 1) {
        for (int vec : {4, 8}) {
            const Shape f = fwd_shape(D, vec), b = bwd_shape(D, vec);
            std::printf("fwd.%s.%dx%d bwd.%s.%dx%d.%s ", vec == 4 ? "f32" : "bf16", f.wpr, f.ch, vec == 4 ? "f32" : "bf16", b.wpr,
                        b.ch, D % vec == 0 ? "even" : "odd");
        }
        std::printf("\n");
    }
#else
    // N in ff: tile, layout of the weights, whole or cut along k
    long long N, in, ff;
    while (std::scanf("%lld %lld %lld", &N, &in, &ff) == 3) {
#if defined(OF_F32)
        // the forward's products of any layout; dx (along both halves, or twice with the second added) and both dW
        for (int w_t : {0, 1}) {
            auto say = [&](const char* what, int64_t M, int64_t n, int64_t K, int ta, int tb) {
                GemmF32 g{};
                g.M = M, g.N = g.ldc = n;
                g.terms[0] = {nullptr, nullptr, K, K, K, ta, tb, 1.f};
                const Plan p = plan(g);
                std::printf("%s.%s.%s.%s ", what, w_t ? "ff_in" : "in_ff", p.small ? "64" : "128", p.a.whole ? "whole" : "cut");
            };
            const bool joins = in * ff <= 1 << 21;
            if (N > 2) say("fwd", N, ff, in, 0, w_t);
            say(joins ? "dx" : "dx_added", N, in, joins ? 2 * ff : ff, 0, !w_t);
            if (w_t) say("dW_both", 2 * ff, in, N, 1, 0);
            else say("dW", in, ff, N, 1, 0);
        }
#else
        for (int w_t : {0, 1}) {
            LinearProduct g{};
            g.M = N, g.N = ff, g.K = in, g.p_kc = 1, g.q_kc = w_t;
            if (N <= 2) continue;  // kernels of their own
#if defined(OF_E4M3)
            if (!w_t) continue;
            const Shape& t = kShapes[shape_of(g)];
            std::printf("e4m3.%dx%d.%s.%s ", t.bn, t.bm, N % t.bm || 2 * ff % t.bn ? "ragged" : "full", off_rows(g) ? "copied" : "in_place");
#else
            const Plan p = plan(g, true);
            std::printf("gated.%s.%dx%d%s.%s ", w_t ? "ff_in" : "in_ff", kGated[p.shape].bn, kGated[p.shape].bm,
                        kGated[p.shape].deep ? "deep" : "", p.a.whole ? "whole" : "cut");
            if (ff % kSlab == 0 && (w_t == 0 || in % 8 == 0)) {  // else the linear layer's product of copies
                LinearProduct x{};
                x.M = N, x.N = in, x.K = x.ldp = 2 * ff, x.joint = ff;
                x.p_kc = 1, x.q_kc = w_t == 0;
                const Plan q = plan(x, false);
                std::printf("joined.%s.%dx%d%s.%s ", w_t ? "ff_in" : "in_ff", kJoined[q.shape].bn, kJoined[q.shape].bm,
                            kJoined[q.shape].deep ? "deep" : "", q.a.whole ? "whole" : "cut");
            }
#endif
        }
#endif
        std::printf("\n");
    }
#endif
    return 0;
}
