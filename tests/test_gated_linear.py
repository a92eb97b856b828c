"""The gated linear layer (mft_gated_linear_* through the torch helpers) against its
formulas in 64 bits, and refusals.

Bounds, per element, with u = 2^-24 and h half a step of the type (2^-8 for bf16).
gate and up are products of K terms in fp32: off by 2 (K + 8) u of the sum of the
magnitudes (the products of bf16 numbers are exact; twice over in case the matrix
unit truncates), and stored by h of themselves more.  In 8 bits the matrix unit first
adds eight products, each cut to a multiple of 2^-13 of 2^(a + b), with a and b the
exponents of the largest one's factors: seven cuts of at most 2^-13 of the
largest, so 7 2^-13 of the sum of the magnitudes.  Where all factors lie in [1, 16)
the products are multiples of 2^-6 and the largest's exponents give at most 2^6: nothing
is cut, and the bound is the first.  The activations'
slopes stay under 1.13, and their own evaluation under u (24 + 8 |z|) of max(|y|,
|z|).  The backward is given gate and up: act'(z) is off by u (32 + 16 |z|^2 + 16 |z|);
dgate and dup, rounded to bf16, by h of themselves more; dx and the weights' gradients
carry that through their sums.
"""
import ctypes as C
import math

import pytest
import torch
import torch.nn.functional as F

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = {"relu": F.relu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}


def half(t):
    return torch.finfo(t).eps / 2 if t == torch.bfloat16 else U


def make(N, n_in, n_ff, dtype, seed, w_t=False):
    g = torch.Generator().manual_seed(seed)
    t = DT[dtype]
    x = torch.randn(N, n_in, generator=g).to(t)
    Wg, Wu = ((torch.randn(n_in, n_ff, generator=g) / math.sqrt(n_in)).to(t) for _ in range(2))
    gate, up = ((1.5 * torch.randn(N, n_ff, generator=g)).to(t) for _ in range(2))
    dh = (0.1 * torch.randn(N, n_ff, generator=g)).to(t)
    return dict(x=x, W_gate=Wg.t().contiguous() if w_t else Wg, W_up=Wu.t().contiguous() if w_t else Wu, gate=gate, up=up,
                dh=dh)


def of_act(z, act):
    """act(z), and how far the kernels' may be off it."""
    y = ACTS[act](z)
    return y, U * (24 + 8 * z.abs()) * torch.maximum(y.abs(), z.abs()) if act != "relu" else torch.zeros_like(y)


def ref_forward(x, Wg, Wu, act, t, scale=(1.0, 1.0, 1.0), cut=0.0):
    """(gate, its bound, up, its bound, h, its bound), W [in, ff] in 64 bits, times the rows' scales; cut: what the
    products may lose of the sum of their magnitudes."""
    K = x.shape[1]
    xs, gs, us = scale
    out = []
    for W, s in ((Wg, gs), (Wu, us)):
        z = (x @ W) * xs * s
        out.append((z, (2 * (K + 8) * U + cut) * (x.abs() @ W.abs()) * xs * s + 4 * U * z.abs()))
    (g, eg), (u, eu) = out
    a, ea = of_act(g, act)
    h = a * u
    eh = u.abs() * (1.13 * eg + ea) + a.abs() * eu + (1.13 * eg + ea) * eu + (half(t) + 2 * U) * h.abs() + 1e-30
    return g, eg + half(t) * g.abs() + 1e-30, u, eu + half(t) * u.abs() + 1e-30, h, eh


def ref_backward(x, Wg, Wu, gate, up, dh, act, t):
    z = gate.clone().requires_grad_(True)
    slope, = torch.autograd.grad(ACTS[act](z).sum(), z)
    a, ea = of_act(gate, act)
    dg, du = dh * up * slope, dh * a
    h = half(t) if t == torch.bfloat16 else 0
    es = 0 if act == "relu" else U * (32 + 16 * gate * gate + 16 * gate.abs())
    eg = (dh * up).abs() * es + (4 * U + h) * dg.abs()
    eu = dh.abs() * ea + (2 * U + h) * du.abs()
    N, ff = dg.shape
    dx = dg @ Wg.t() + du @ Wu.t()
    mags = dg.abs() @ Wg.abs().t() + du.abs() @ Wu.abs().t()
    ex = eg @ Wg.abs().t() + eu @ Wu.abs().t() + 2 * (2 * ff + 16) * U * mags + half(t) * dx.abs() + 1e-30
    out = [dx, ex]
    for d, e in ((dg, eg), (du, eu)):
        dW = x.t() @ d
        out += [dW, x.abs().t() @ e + 2 * (N + 8) * U * (x.abs().t() @ d.abs()) + half(t) * dW.abs() + 1e-30]
    return out


def within(got, ref, tol, what=""):
    assert got.shape == ref.shape
    off = (got.detach().double() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def check(dev, N, n_in, n_ff, dtype, act, w_t, seed):
    from mobilefinetuner_amd import gated_linear as L
    print(f"[case] {N} x {n_in} -> {n_ff} {dtype} {act} {'[ff, in]' if w_t else '[in, ff]'}", flush=True)
    d = {k: v.to(dev) for k, v in make(N, n_in, n_ff, dtype, seed, w_t).items()}
    up = {k: v.double() for k, v in d.items()}
    Wg, Wu = (up[k].t() if w_t else up[k] for k in ("W_gate", "W_up"))
    t = DT[dtype]
    h, gate, rise = L.gated_linear(d["x"], d["W_gate"], d["W_up"], act, w_t, want_preact=True)
    rg, tg, ru, tu, rh, th = ref_forward(up["x"], Wg, Wu, act, t)
    assert h.dtype == gate.dtype == rise.dtype == t
    within(gate, rg, tg, "gate")
    within(rise, ru, tu, "up")
    within(h, rh, th, "h")
    only = L.gated_linear(d["x"], d["W_gate"], d["W_up"], act, w_t)
    assert torch.equal(only[0], h) and only[1] is None and only[2] is None
    dx, dWg, dWu = L.gated_linear_backward(d["x"], d["W_gate"], d["W_up"], d["gate"], d["up"], d["dh"], act, w_t)
    rx, tx, rwg, twg, rwu, twu = ref_backward(up["x"], Wg, Wu, up["gate"], up["up"], up["dh"], act, t)
    if w_t:
        rwg, twg, rwu, twu = rwg.t(), twg.t(), rwu.t(), twu.t()
    assert dx.dtype == dWg.dtype == dWu.dtype == t
    within(dx, rx, tx, "dx")
    within(dWg, rwg, twg, "dW_gate")
    within(dWu, rwu, twu, "dW_up")


# N, in, ff: one token and few, each tile with whole and ragged edges, odd sizes, K below a stage and
# with a partial last stage, sizes of one
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 768, 1024), (1, 33, 4100), (2, 1024, 512), (2, 100, 9), (3, 33, 17), (5, 640, 2048),
          (8, 896, 896), (17, 65, 130), (33, 128, 64), (64, 64, 64), (100, 200, 300), (129, 257, 511), (128, 128, 256),
          (300, 1152, 640), (333, 72, 1000), (1000, 8, 8), (1024, 512, 256), (513, 1000, 104)]


@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_ff", "ff_in"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(dev, shape, dtype, w_t):
    check(dev, *shape, dtype, "gelu_tanh", w_t, sum(shape))


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 200, 72), (3, 200, 136), (150, 96, 264)], ids=lambda s: "x".join(map(str, s)))
def test_activations(dev, shape, dtype, act):
    for w_t in (False, True):
        check(dev, *shape, dtype, act, w_t, 7)


# products that fill the GPU with the largest tiles, with the middle ones, and that are cut along K; off 16
# bytes with and without copies
@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_ff", "ff_in"])
@pytest.mark.parametrize("shape", [(4096, 256, 2048), (4100, 264, 2056), (2048, 320, 1024), (96, 4096, 128),
                                   (2000, 2048, 72), (512, 1024, 8192), (700, 1153, 2001), (2000, 601, 1999),
                                   (256, 2048, 1024), (64, 8192, 64)], ids=lambda s: "x".join(map(str, s)))
def test_large_products(dev, shape, w_t):
    check(dev, *shape, "bf16", "silu", w_t, 3)


CUT = 7 * 2.0 ** -13


def eight_bits(N, n_in, n_ff, seed, near=False):
    """e4m3 numbers of all sizes (near: 0 and those from 1 up to 16) with their scales: x [N, in], W_gate and W_up
    [ff, in]."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for rows in (N, n_ff, n_ff):
        if near:
            q = torch.randint(-1, 2, (rows, n_in), generator=g) * (1 + torch.randint(0, 8, (rows, n_in), generator=g) / 8) * \
                2.0 ** torch.randint(0, 4, (rows, n_in), generator=g)
        else:
            q = torch.randn(rows, n_in, generator=g) * 2.0 ** torch.randint(-8, 7, (rows, n_in), generator=g)
        out += [q.clamp(-448, 448).to(torch.float8_e4m3fn), 2.0 ** torch.randint(-9, -5, (rows,), generator=g) *
                (1 + torch.rand(rows, generator=g)) / math.sqrt(n_in)]
    return out


def check_e4m3(dev, N, n_in, n_ff, act, seed, shift=0, near=False):
    from mobilefinetuner_amd import gated_linear as L
    print(f"[case] {N} x {n_in} -> {n_ff} e4m3 {act} off {shift} {'near' if near else ''}", flush=True)
    args = [t.to(dev) for t in eight_bits(N, n_in, n_ff, seed, near)]
    if shift:
        for i in (0, 2, 4):
            flat = torch.zeros(args[i].numel() + shift, dtype=torch.uint8, device=dev)[shift:].view(args[i].shape)
            flat.copy_(args[i].view(torch.uint8))
            args[i] = flat.view(torch.float8_e4m3fn)
    h = L.gated_linear_e4m3(*args, act)
    x, Wg, Wu = (args[i].float().double() for i in (0, 2, 4))
    scale = [args[1].double()[:, None], args[3].double(), args[5].double()]
    rh, th = ref_forward(x, Wg.t(), Wu.t(), act, torch.bfloat16, scale, 0.0 if near else CUT)[4:]
    assert h.dtype == torch.bfloat16
    within(h, rh, th, "h")


# the shapes above, and every tile: of 256 x 256, 128 x 192, 128 x 128 and 128 x 64, whole and ragged
@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES + [(3, 128, 64), (65, 144, 100), (2048, 256, 8192), (2100, 272, 8200),
                                            (512, 640, 8192), (500, 208, 8190), (256, 128, 8192), (250, 272, 8100),
                                            (33, 4096, 128), (2000, 601, 1999), (1024, 4096, 8192),
                                            (1000, 4112, 8200), (8192, 1152, 2048), (8190, 1168, 2046),
                                            (2048, 2048, 1024), (2000, 2064, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_eight_bits(dev, shape):
    check_e4m3(dev, *shape, "gelu_tanh", sum(shape))
    check_e4m3(dev, *shape, "gelu_tanh", sum(shape), near=True)


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("shape", [(1, 200, 72), (2, 128, 70), (150, 96, 264), (300, 384, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_eight_bits_off_16_bytes(dev, shape, act):
    for shift in (0, 1, 8):
        check_e4m3(dev, *shape, act, 7, shift, near=shift == 1)


@pytest.mark.gpu
def test_eight_bits_of_a_norm(dev):
    """rms_norm_e4m3 and quantize_rows into gated_linear_e4m3, in batches of rows, against their numbers in 64 bits;
    a NaN stays in its row; no rows; replays follow their inputs."""
    from mobilefinetuner_amd import gated_linear as L
    from mobilefinetuner_amd import rms_norm as R
    d = {k: v.to(dev) for k, v in make(60, 256, 384, "bf16", 12, True).items()}
    w = torch.randn(256, device=dev) * 0.2
    (gq, gs), (uq, us) = R.quantize_rows(d["W_gate"]), R.quantize_rows(d["W_up"])

    def step():
        q, scale, _ = R.rms_norm_e4m3(d["x"].view(3, 20, 256), w)
        return q, scale, L.gated_linear_e4m3(q, scale, gq, gs, uq, us, "silu")

    def right(q, scale, h):
        scales = [scale.double().view(60, 1), gs.double(), us.double()]
        rh, th = ref_forward(q.float().double().view(60, 256), gq.float().double().t(), uq.float().double().t(), "silu",
                             torch.bfloat16, scales, CUT)[4:]
        assert h.shape == (3, 20, 384)
        within(h.view(60, 384), rh, th)

    right(*step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (13, 14, 15):
        d["x"].copy_(make(60, 256, 384, "bf16", seed, True)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(held, step()))
        right(*held)
    clean = step()[2].view(60, 384)
    d["x"][33, 5] = math.nan
    h = step()[2].view(60, 384)
    keep = torch.arange(60, device=dev) != 33
    assert torch.isnan(h[33]).all() and torch.equal(h[keep], clean[keep])
    none = d["x"][:0].to(torch.float8_e4m3fn)
    assert L.gated_linear_e4m3(none, torch.zeros(0, device=dev), gq, gs, uq, us).shape == (0, 384)
    one = L.gated_linear_e4m3(held[0][0, :1], held[1][0, :1], gq, gs, uq, us, "silu")  # a kernel of its own
    scales = [held[1][0, :1, None].double(), gs.double(), us.double()]
    within(one, *ref_forward(held[0][0, :1].float().double(), gq.float().double().t(), uq.float().double().t(), "silu",
                             torch.bfloat16, scales)[4:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_leading_dimensions_and_other_layouts(dev, dtype):
    """Batches of rows, operands that are not contiguous and weights off 16 bytes: the results of copies."""
    from mobilefinetuner_amd import gated_linear as L
    d = {k: v.to(dev) for k, v in make(24, 96, 136, dtype, 5).items()}
    call = lambda x, a, b: L.gated_linear(x, a, b, "silu", False, True)  # noqa: E731
    ref = call(d["x"], d["W_gate"], d["W_up"])
    got = call(d["x"].view(2, 3, 4, 96), d["W_gate"], d["W_up"])
    assert got[0].shape == (2, 3, 4, 136) and all(torch.equal(p.view(24, 136), q) for p, q in zip(got, ref))

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:]
        return flat.view(t.shape).copy_(t)

    wide = torch.zeros(24, 200, dtype=DT[dtype], device=dev)
    wide[:, 7:103] = d["x"]
    for x, a, b in ((wide[:, 7:103], d["W_gate"].t().contiguous().t(), d["W_up"]),
                    (shifted(d["x"]), d["W_gate"], shifted(d["W_up"])), (d["x"], shifted(d["W_gate"]), d["W_up"])):
        for p, q in zip(call(x, a, b), ref):
            assert torch.equal(p, q) or float((p - q).abs().max()) <= 2 * half(DT[dtype]) * float(q.abs().max())
    back = L.gated_linear_backward(d["x"], d["W_gate"], d["W_up"], d["gate"], d["up"], d["dh"], "silu")
    other = L.gated_linear_backward(d["x"].view(4, 6, 96), shifted(d["W_gate"]), shifted(d["W_up"]),
                                    d["gate"].view(4, 6, 136), d["up"].view(4, 6, 136), d["dh"].view(4, 6, 136), "silu")
    for p, q in zip(other, back):
        assert float((p.view(q.shape) - q).abs().max()) <= 2 * half(DT[dtype]) * float(q.abs().max())


@pytest.mark.gpu
def test_one_row_strided_numbers_and_one_weight_for_both(dev):
    """x without leading dimensions, e4m3 numbers that are not contiguous, and gate and up by one trained weight,
    whose gradient is the sum of both."""
    from mobilefinetuner_amd import gated_linear as L
    d = {k: v.to(dev) for k, v in make(3, 96, 40, "f32", 17).items()}
    row = L.gated_linear(d["x"][0], d["W_gate"], d["W_up"])[0]
    assert row.shape == (40,) and torch.equal(row, L.gated_linear(d["x"][:1], d["W_gate"], d["W_up"])[0][0])
    q, qs, g, gs, u, us = (t.to(dev) for t in eight_bits(10, 96, 64, 18))
    wide = torch.zeros(10, 192, dtype=torch.uint8, device=dev)
    wide[:, ::2] = q.view(torch.uint8)
    got = L.gated_linear_e4m3(wide.view(torch.float8_e4m3fn)[:, ::2], qs, g.t().contiguous().t(), gs, u, us)
    assert torch.equal(got, L.gated_linear_e4m3(q, qs, g, gs, u, us))
    W = d["W_gate"].clone().requires_grad_(True)
    L.GatedLinear.apply(d["x"], W, W, "silu").backward(d["dh"])
    _, gate, up = L.gated_linear(d["x"], W.detach(), W.detach(), "silu", False, True)
    _, a, b = L.gated_linear_backward(d["x"], W.detach(), W.detach(), gate, up, d["dh"], "silu")
    assert torch.equal(W.grad, a + b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows_and_parts_of_the_gradient(dev, dtype):
    from mobilefinetuner_amd import gated_linear as L
    for N in (0, 40):
        d = {k: v.to(dev) for k, v in make(N, 72, 48, dtype, 6).items()}
        args = [d[k] for k in ("x", "W_gate", "W_up", "gate", "up", "dh")]
        assert L.gated_linear(*args[:3])[0].shape == (N, 48)
        whole = L.gated_linear_backward(*args)
        if N == 0:
            assert whole[0].shape == (0, 72) and (whole[1] == 0).all() and (whole[2] == 0).all()
        for want in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
            only = L.gated_linear_backward(*args, want_x=want[0], want_gate=want[1], want_up=want[2])
            for o, w, on in zip(only, whole, want):
                assert torch.equal(o, w) if on else o is None


@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True])
def test_values_that_are_not_numbers(dev, w_t):
    """A NaN of x stays in its row, one of a weight in its column."""
    from mobilefinetuner_amd import gated_linear as L
    for dtype in ("f32", "bf16"):
        for N in (1, 70):
            d = {k: v.to(dev) for k, v in make(N, 136, 200, dtype, 9, w_t).items()}
            clean = L.gated_linear(d["x"], d["W_gate"], d["W_up"], "silu", w_t)[0]
            x, W = d["x"].clone(), d["W_up"].clone()
            x[N // 2, 5] = math.nan
            h = L.gated_linear(x, d["W_gate"], d["W_up"], "silu", w_t)[0]
            rows = torch.arange(N, device=dev) != N // 2
            assert torch.isnan(h[N // 2]).all() and torch.equal(h[rows], clean[rows])
            W[(33, 7) if w_t else (7, 33)] = math.nan
            h = L.gated_linear(d["x"], d["W_gate"], W, "silu", w_t)[0]
            cols = torch.arange(200, device=dev) != 33
            assert torch.isnan(h[:, 33]).all() and torch.equal(h[:, cols], clean[:, cols])


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """More than 2^31 values of h: the last rows are those of a call of their own, to the rounding of h."""
    from mobilefinetuner_amd import gated_linear as L
    N, n_in, n_ff = (1 << 18) + 40, 64, 8320
    d = {k: v.to(dev) for k, v in make(40, n_in, n_ff, "bf16", 11).items()}
    x = torch.zeros(N, n_in, dtype=torch.bfloat16, device=dev)
    x[-40:] = d["x"]
    h, gate, up = L.gated_linear(x, d["W_gate"], d["W_up"], "silu", False, True)
    ref = L.gated_linear(d["x"], d["W_gate"], d["W_up"], "silu", False, True)
    for p, q in zip((h, gate, up), ref):
        assert float((p[-40:] - q).abs().max()) <= 2 * half(torch.bfloat16) * float(q.abs().max())
        assert (p[:100] == 0).all()
    gate[-40:], up[-40:] = d["gate"], d["up"]
    h[-40:] = d["dh"]
    dx, dWg, dWu = L.gated_linear_backward(x, d["W_gate"], d["W_up"], gate, up, h, "silu")
    back = L.gated_linear_backward(d["x"], d["W_gate"], d["W_up"], d["gate"], d["up"], d["dh"], "silu")
    assert (dx[:100] == 0).all()
    for p, q in zip((dx[-40:], dWg, dWu), back):
        assert float((p - q).abs().max()) <= 2 * half(torch.bfloat16) * float(q.abs().max())
    del h, gate, up
    args = [t.to(dev) for t in eight_bits(40, n_in, n_ff, 11, near=True)]
    x8 = torch.zeros(N, n_in, dtype=torch.uint8, device=dev)
    x8[-40:] = args[0].view(torch.uint8)
    scale = torch.ones(N, device=dev)
    scale[-40:] = args[1]
    h = L.gated_linear_e4m3(x8.view(torch.float8_e4m3fn), scale, *args[2:])
    assert torch.equal(h[-40:], L.gated_linear_e4m3(*args)) and (h[:100] == 0).all()  # sums that nothing rounds
    del h, x8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_autograd_gradients_against_differences(dev, dtype, act):
    """The node's gradients are the helpers', and (fp32) those of differences: the loss sum(h c) moves by the
    gradient along a direction v, to the second order of the step and the loss's rounding over it.  ReLU has
    no second order where gate's sign stays: its gates are kept from zero."""
    from mobilefinetuner_amd import gated_linear as L
    s = {k: v.to(dev) for k, v in make(7, 40, 24, dtype, 8).items()}
    leaves = [s[k].clone().requires_grad_(True) for k in ("x", "W_gate", "W_up")]
    h = L.GatedLinear.apply(*leaves, act, False)
    h.backward(s["dh"])
    at = [v.detach() for v in leaves]
    _, gate, up = L.gated_linear(*at, act, False, True)
    for g, r in zip((v.grad for v in leaves), L.gated_linear_backward(*at, gate, up, s["dh"], act)):
        assert torch.equal(g, r)
    if dtype == "bf16" or act == "relu":
        return
    g = torch.Generator().manual_seed(1)
    t = 2.0 ** -7
    for i, p in enumerate(at):
        v = torch.randn(p.shape, generator=g).to(dev) * (1.0 if i == 0 else 40 ** -0.5)
        loss = []
        for k in (t, -t):
            q = [u + k * v if j == i else u for j, u in enumerate(at)]
            loss.append(float((L.gated_linear(*q, act)[0].double() * s["dh"].double()).sum()))
        slope = (loss[0] - loss[1]) / (2 * t)
        scale = float(s["dh"].double().norm() * v.double().norm()) * math.sqrt(24) * 4
        assert abs(slope - float((leaves[i].grad.double() * v.double()).sum())) <= scale * (4 * t * t + 256 * U / t)


@pytest.mark.gpu
def test_repeated_calls_and_streams(dev):
    """The same bits from every call, also from two streams at once, each with its own workspace."""
    from mobilefinetuner_amd import gated_linear as L
    for shape in ((600, 512, 384), (96, 4096, 128)):
        d = {k: v.to(dev) for k, v in make(*shape, "bf16", 9).items()}
        args = [d[k] for k in ("x", "W_gate", "W_up", "gate", "up", "dh")]
        ref = L.gated_linear(*args[:3])[:1] + L.gated_linear_backward(*args)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                got.append(L.gated_linear(*args[:3])[:1] + L.gated_linear_backward(*args))
        torch.cuda.synchronize()
        for r in got:
            assert all(torch.equal(p, q) for p, q in zip(r, ref))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_graph_follows_its_inputs(dev, dtype):
    from mobilefinetuner_amd import gated_linear as L
    names = ("x", "W_gate", "W_up", "gate", "up", "dh")
    d = {k: v.to(dev) for k, v in make(96, 1024, 136, dtype, 10).items()}

    def step():
        return L.gated_linear(*(d[k] for k in names[:3]))[:1] + L.gated_linear_backward(*(d[k] for k in names))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (11, 12, 13):
        for k, v in make(96, 1024, 136, dtype, seed).items():
            d[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


@pytest.mark.parametrize("change,message", [
    (dict(N=-1), "N >= 0"), (dict(in_dim=0), "positive"), (dict(ff_dim=0), "positive"), (dict(N=1 << 31), "below"),
    (dict(in_dim=(1 << 24) + 1), "at most"), (dict(ff_dim=(1 << 24) + 1), "at most"), (dict(dtype=1), "dtype"),
    (dict(activation=0), "activation"), (dict(activation=4), "activation"),
    (dict(N=1 << 24, ff_dim=1 << 20), "too large together"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.gated_linear_desc(**{**dict(N=4, in_dim=64, ff_dim=32, dtype=capi.MFT_BF16, w_transposed=True), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.gated_linear_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.gated_linear_fwd(d, 16, 32, 48, 64, None, None, 80, None)
    with pytest.raises(capi.MftError, match=message):
        capi.gated_linear_bwd(d, 16, 32, 48, 64, 80, 96, 112, 128, 144, 160, None)
    with pytest.raises(capi.MftError, match=message):
        capi.gated_linear_e4m3_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.gated_linear_e4m3_fwd(d, 16, 32, 48, 64, 80, 96, 112, 128, None)


def test_operands_refused(capi):
    d = capi.gated_linear_desc(4, 64, 32)
    fwd, bwd = [16, 32, 48, 64, 80, 96, 112], [16, 32, 48, 64, 80, 96, 112, 128, 144, 160]
    but = lambda a, **c: [c.get(f"_{i}", v) for i, v in enumerate(a)]  # noqa: E731
    for i in (0, 1, 2, 3, 6):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.gated_linear_fwd(d, *but(fwd, **{f"_{i}": None}), None)
    for i in (4, 5):
        with pytest.raises(capi.MftError, match="together"):
            capi.gated_linear_fwd(d, *but(fwd, **{f"_{i}": None}), None)
    for i, j in ((3, 0), (3, 1), (3, 2), (3, 4), (3, 5), (4, 0), (4, 5), (5, 2)):
        with pytest.raises(capi.MftError, match="may not be"):
            capi.gated_linear_fwd(d, *but(fwd, **{f"_{i}": fwd[j]}), None)
    for i in (0, 1, 2, 3, 4, 5, 9):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.gated_linear_bwd(d, *but(bwd, **{f"_{i}": None}), None)
    for i, j in ((6, 5), (6, 0), (7, 1), (8, 3), (6, 7), (6, 8), (7, 8)):
        with pytest.raises(capi.MftError, match="may not be"):
            capi.gated_linear_bwd(d, *but(bwd, **{f"_{i}": bwd[j]}), None)
    e = capi.gated_linear_desc(4, 65, 32, capi.MFT_BF16, True)
    eight = [16, 32, 48, 64, 80, 96, 112, 128]
    for i in range(8):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.gated_linear_e4m3_fwd(e, *but(eight, **{f"_{i}": None}), None)
    for i in range(6):
        with pytest.raises(capi.MftError, match="may not be"):
            capi.gated_linear_e4m3_fwd(e, *but(eight, _6=eight[i]), None)
    for change, message in ((dict(dtype=capi.MFT_F32), "dtype"), (dict(w_transposed=False), "stored")):
        f = capi.gated_linear_desc(4, 64, 32, **{**dict(dtype=capi.MFT_BF16, w_transposed=True), **change})
        with pytest.raises(capi.MftError, match=message):
            capi.gated_linear_e4m3_fwd(f, *eight, None)
    assert capi.lib().mft_gated_linear_e4m3_fwd(C.byref(capi.gated_linear_desc(0, 64, 32, capi.MFT_BF16, True)),
                                                *[None] * 9) == capi.MFT_OK
    assert capi.lib().mft_gated_linear_fwd(None, *fwd, None) == capi.MFT_ERR_INVALID_ARG
    empty = C.byref(capi.gated_linear_desc(0, 64, 32))
    assert capi.lib().mft_gated_linear_fwd(empty, *[None] * 8) == capi.MFT_OK
    assert capi.lib().mft_gated_linear_bwd(empty, *[None] * 11) == capi.MFT_OK


def test_no_cpu_path():
    from mobilefinetuner_amd import gated_linear as L
    with pytest.raises(ValueError, match="no CPU path"):
        L.gated_linear(torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4, 3))


@pytest.mark.gpu
def test_operands_that_do_not_fit_refused(dev):
    from mobilefinetuner_amd import gated_linear as L
    x, W, g = torch.zeros(2, 8, device=dev), torch.zeros(8, 6, device=dev), torch.zeros(2, 6, device=dev)
    for bad in (lambda: L.gated_linear(x, W, W[:, :5]), lambda: L.gated_linear(x, W, W.bfloat16()),
                lambda: L.gated_linear(x, W.cpu(), W), lambda: L.gated_linear(x[:, :7], W, W),
                lambda: L.gated_linear(x, W, W, "none"), lambda: L.gated_linear(x, W, W, w_transposed=True),
                lambda: L.gated_linear(x, W[None], W[None]), lambda: L.gated_linear(x.half(), W.half(), W.half()),
                lambda: L.gated_linear_backward(x, W, W, g, g, g[:1]), lambda: L.gated_linear_backward(x, W, W, None, g, g),
                lambda: L.gated_linear_backward(x, W, W, g, g.bfloat16(), g)):
        with pytest.raises(ValueError):
            bad()
    q, s, w, ws = x.to(torch.float8_e4m3fn), g[:, 0].contiguous(), W.t().contiguous().to(torch.float8_e4m3fn), x[0, :6]
    L.gated_linear_e4m3(q, s, w, ws, w, ws)
    for bad in (lambda: L.gated_linear_e4m3(x, s, w, ws, w, ws), lambda: L.gated_linear_e4m3(q, s, W, ws, W, ws),
                lambda: L.gated_linear_e4m3(q, s[:1], w, ws, w, ws), lambda: L.gated_linear_e4m3(q, s, w, s, w, ws),
                lambda: L.gated_linear_e4m3(q, s, w, ws, w, ws.bfloat16()), lambda: L.gated_linear(q, w, w)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 72, 48), (33, 65, 51), (509, 640, 2048)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_have_memory_of_their_own(dev, shape):
    """Each weight's gradient alone in its storage, and the same bits wherever the caller's buffers lie: one behind
    the other, apart, in the other order, off 16 bytes."""
    from mobilefinetuner_amd import capi
    from mobilefinetuner_amd import gated_linear as L
    print(f"[case] {shape}", flush=True)
    N, n_in, n_ff = shape
    n = n_ff * n_in
    d = {k: v.to(dev) for k, v in make(*shape, "f32", 19, True).items()}
    args = [d[k] for k in ("x", "W_gate", "W_up", "gate", "up", "dh")]
    _, a, b = L.gated_linear_backward(*args, w_transposed=True)
    held = [(g.untyped_storage().nbytes(), g.storage_offset()) for g in (a, b)]
    assert held == [(4 * n, 0)] * 2
    desc = capi.gated_linear_desc(N, n_in, n_ff, w_transposed=True)
    ws = torch.empty(capi.gated_linear_workspace_size(desc)[1], dtype=torch.uint8, device=dev)
    for at, too in ((0, n), (0, n + 64), (n + 64, 0), (0, n + 1), (3, n + 8)):
        out = torch.full((2 * n + 128,), math.nan, device=dev)
        capi.gated_linear_bwd(desc, *(t.data_ptr() for t in args), None, out.data_ptr() + 4 * at, out.data_ptr() + 4 * too,
                              ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[at : at + n], a.view(-1)) and torch.equal(out[too : too + n], b.view(-1))
        assert int(out.isnan().sum()) == 128  # nothing else is written
