"""The linear layer with a fused epilogue (mft_linear_* through the torch helpers)
against its formulas in 64 bits, and refusals.

Bounds, per element, with u = 2^-24 and h half a step of the type (2^-8 for
bf16).  A product of K terms in fp32 is off by (K + 8) u of the sum of the
magnitudes; with bf16 that holds as its products are exact, twice over in case
the matrix unit truncates.  z adds the bias's rounding and, stored, h of itself.
The activations' slopes stay under 1.13, and their own evaluation (exponential
and reciprocal, of an argument x that is off by 4 u |x|) under u (24 + 8 |z|) of
max(|y|, |z|).  The backward is given z: act'(z) is off by u (32 + 16 |z|^2 + 16 |z|)
(the exponent's error, at most that, times |z|; slopes under 1.13), dz, rounded
to bf16, by h of itself more; dx and dW carry dz's error through their sums.
"""
import ctypes as C
import math

import pytest
import torch
import torch.nn.functional as F

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = {"none": lambda z: z, "relu": F.relu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}


def half(t):
    return torch.finfo(t).eps / 2 if t == torch.bfloat16 else U


def make(N, n_in, n_out, dtype, seed, w_t=False, act="none"):
    g = torch.Generator().manual_seed(seed)
    t = DT[dtype]
    x = torch.randn(N, n_in, generator=g).to(t)
    W = (torch.randn(n_in, n_out, generator=g) / math.sqrt(n_in)).to(t)
    bias, res = 0.3 * torch.randn(n_out, generator=g), torch.randn(N, n_out, generator=g).to(t)
    z = (x.double() @ W.double() + bias).to(t)
    dy = (0.1 * torch.randn(N, n_out, generator=g)).to(t)
    return dict(x=x, W=W.t().contiguous() if w_t else W, bias=bias, residual=res, z=z, dy=dy)


def ref_forward(s, act, w_t, bias=True, residual=True):
    x, W = s["x"].double(), s["W"].double()
    W = W.t() if w_t else W
    K, t = x.shape[1], s["x"].dtype
    z = x @ W + (s["bias"].double() if bias else 0)
    ez = 2 * (K + 8) * U * (x.abs() @ W.abs()) + 2 * U * z.abs() + (U * s["bias"].double().abs() if bias else 0)
    y = ACTS[act](z) + (s["residual"].double() if residual else 0)
    ea = 0 if act == "none" else U * (24 + 8 * z.abs()) * torch.maximum(ACTS[act](z).abs(), z.abs())
    return z, ez + half(t) * z.abs() + 1e-30, y, 1.13 * ez + ea + (half(t) + 2 * U) * y.abs() + U + 1e-30


def ref_backward(s, act, w_t):
    x, W, dy = s["x"].double(), s["W"].double(), s["dy"].double()
    W = W.t() if w_t else W
    t = s["x"].dtype
    dz, edz = dy, torch.zeros_like(dy)
    if act != "none":
        z = s["z"].double().requires_grad_(True)
        dz, = torch.autograd.grad(ACTS[act](z), z, dy)
        z = z.detach()
        if act != "relu":
            edz = dy.abs() * U * (32 + 16 * z * z + 16 * z.abs())
        edz = edz + 2 * U * dz.abs()
    db, edb = dz.sum(0), edz.sum(0) + U * (len(x) + 64) * dz.abs().sum(0) + 1e-30
    if act != "none" and t == torch.bfloat16:
        edz = edz + half(t) * dz.abs()
    N, out = dz.shape
    dx, dW = dz @ W.t(), x.t() @ dz
    ex = edz @ W.abs().t() + 2 * (out + 8) * U * (dz.abs() @ W.abs().t()) + half(t) * dx.abs() + 1e-30
    eW = x.abs().t() @ edz + 2 * (N + 8) * U * (x.abs().t() @ dz.abs()) + half(t) * dW.abs() + 1e-30
    if w_t:
        dW, eW = dW.t(), eW.t()
    return dx, ex, dW, eW, db, edb


def within(got, ref, tol, what=""):
    off = (got.detach().cpu().double() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def check(dev, N, n_in, n_out, dtype, act, w_t, seed):
    from mobilefinetuner_amd import linear as L
    print(f"[case] {N} x {n_in} -> {n_out} {dtype} {act} {'[out, in]' if w_t else '[in, out]'}", flush=True)
    s = make(N, n_in, n_out, dtype, seed, w_t, act)
    d = {k: v.to(dev) for k, v in s.items()}
    y, z = L.linear(d["x"], d["W"], d["bias"], act, d["residual"], w_t, want_preact=act != "none")
    rz, tz, ry, ty = ref_forward(s, act, w_t)
    within(y, ry, ty, "y")
    if act != "none":
        within(z, rz, tz, "z")
    dx, dW, db = L.linear_backward(d["x"], d["W"], d["z"], d["dy"], act, w_t)
    rx, tx, rw, tw, rb, tb = ref_backward(s, act, w_t)
    assert dx.dtype == dW.dtype == s["x"].dtype and db.dtype == torch.float32
    within(dx, rx, tx, "dx")
    within(dW, rw, tw, "dW")
    within(db, rb, tb, "db")


# N, in, out: one token and few, each tile with whole and ragged edges, odd sizes, K below a stage
# and with a partial last stage, sizes of one
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 768, 1024), (2, 1024, 512), (3, 33, 17), (5, 640, 2048), (8, 896, 896), (17, 65, 130),
          (33, 128, 64), (64, 64, 64), (100, 200, 300), (129, 257, 511), (128, 128, 256), (300, 1152, 640), (333, 72, 1000),
          (1000, 8, 8), (1024, 512, 256), (513, 1000, 104)]


@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(dev, shape, dtype, w_t):
    check(dev, *shape, dtype, "gelu_tanh", w_t, sum(shape))


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 200, 136), (150, 96, 264)], ids=lambda s: "x".join(map(str, s)))
def test_activations(dev, shape, dtype, act):
    for w_t in (False, True):
        check(dev, *shape, dtype, act, w_t, 7)


# products that fill the GPU with the largest tiles, with the middle ones, and that are cut along K
@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_out", "out_in"])
@pytest.mark.parametrize("shape", [(4096, 256, 2048), (4100, 264, 2056), (2048, 320, 1024), (96, 4096, 128),
                                   (2000, 2048, 72)], ids=lambda s: "x".join(map(str, s)))
def test_large_products(dev, shape, w_t):
    """Against float64 products on the GPU (the bounds above)."""
    from mobilefinetuner_amd import linear as L
    N, n_in, n_out = shape
    print(f"[case] {shape} {w_t}", flush=True)
    s = {k: v.to(dev) for k, v in make(N, n_in, n_out, "bf16", 3, w_t).items()}
    for act in ("none", "silu"):
        y, z = L.linear(s["x"], s["W"], s["bias"], act, s["residual"], w_t, want_preact=act != "none")
        rz, tz, ry, ty = ref_forward(s, act, w_t)
        within(y, ry.cpu(), ty.cpu(), "y")
        dx, dW, db = L.linear_backward(s["x"], s["W"], s["z"], s["dy"], act, w_t)
        rx, tx, rw, tw, rb, tb = (r.cpu() for r in ref_backward(s, act, w_t))
        within(dx, rx, tx, "dx")
        within(dW, rw, tw, "dW")
        within(db, rb, tb, "db")


def within_gpu(got, ref, tol, what):
    worst = float(((got.double() - ref).abs() / tol).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


# Every tile that a product may run in (256 x 128 and 128 x 128 for two workgroups to a CU, 64 x 64,
# 256 x 256, and 128, 192 and 256 x 128 for a CU of their own), whole and cut along K, with ragged
# edges; rows on 16 bytes (multiples of 8) and off them (copied to whole rows first, or read as they
# are).  W both ways makes each product run with k contiguous in one operand, in both and in none.
TILES = [(8727, 70, 1178), (518, 5516, 6648), (8554, 196, 864), (5442, 330, 4975), (561, 5634, 5067), (8584, 3457, 616),
         (8662, 614, 3514), (93, 1856, 2144), (3328, 6573, 67), (64, 1400, 5039), (5693, 144, 5753), (65, 5135, 4161),
         (1761, 64, 3761), (1020, 66, 5471), (143, 4982, 5773), (6377, 132, 4750), (700, 601, 1203), (1300, 1201, 1501),
         (8728, 72, 1176), (520, 5512, 6648), (8552, 200, 864), (5440, 328, 4968), (568, 5632, 5064), (8584, 3456, 616),
         (96, 1864, 2152), (5696, 144, 5752), (64, 5136, 4168), (1768, 72, 3768), (1032, 72, 5480), (144, 4984, 5776)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", TILES, ids=lambda s: "x".join(map(str, s)))
def test_every_tile(dev, shape):
    from mobilefinetuner_amd import linear as L
    N, n_in, n_out = shape
    g = torch.Generator(device=dev).manual_seed(N)

    def randn(*size):
        return torch.randn(*size, device=dev, generator=g)

    t = torch.bfloat16
    x, W = randn(N, n_in).to(t), (randn(n_in, n_out) / math.sqrt(n_in)).to(t)
    s = dict(x=x, W=W, bias=0.3 * randn(n_out), residual=randn(N, n_out).to(t), dy=(0.1 * randn(N, n_out)).to(t))
    s["z"] = (x.double() @ W.double() + s["bias"]).to(t)
    rz, tz, ry, ty = ref_forward(s, "silu", False)
    rx, tx, rw, tw, rb, tb = ref_backward(s, "silu", False)
    plain = ref_backward(s, "none", False)
    for w_t in (False, True):
        print(f"[case] {shape} {'[out, in]' if w_t else '[in, out]'}", flush=True)
        w = W.t().contiguous() if w_t else W
        y, z = L.linear(x, w, s["bias"], "silu", s["residual"], w_t, want_preact=True)
        within_gpu(y, ry, ty, "y")
        within_gpu(z, rz, tz, "z")
        dx, dW, db = L.linear_backward(x, w, s["z"], s["dy"], "silu", w_t)
        within_gpu(dx, rx, tx, "dx")
        within_gpu(dW.t() if w_t else dW, rw, tw, "dW")
        within_gpu(db, rb, tb, "db")
        dx, dW, db = L.linear_backward(x, w, None, s["dy"], "none", w_t)
        within_gpu(dx, plain[0], plain[1], "dx")
        within_gpu(dW.t() if w_t else dW, plain[2], plain[3], "dW")
        within_gpu(db, plain[4], plain[5], "db")


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """y with more than 2^31 elements: its first and last rows are those of a call of their own
    (a row's terms are added in the same order in every tile but the groups' of a CU's own, whose
    two sums are added last: 2 (K + 8) u of the magnitudes, and the rounding of each)."""
    from mobilefinetuner_amd import linear as L
    N, n_in, n_out = (1 << 19) + 40, 64, 4160
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(N, n_in, device=dev, generator=g).bfloat16()
    W = (torch.randn(n_in, n_out, device=dev, generator=g) / 8).bfloat16()
    y = L.linear(x, W)[0]
    for rows in (slice(0, 300), slice(N - 300, N)):
        s = dict(x=x[rows], W=W, bias=None)
        _, _, ry, ty = ref_forward(s, "none", False, False, False)
        within_gpu(y[rows], ry, ty, "y")
    del y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 40])
def test_parts_of_the_epilogue_and_of_the_gradient(dev, dtype, N):
    from mobilefinetuner_amd import linear as L
    s = make(N, 96, 80, dtype, 4)
    d = {k: v.to(dev) for k, v in s.items()}
    for act in ("none", "gelu_tanh"):
        for bias in (False, True):
            for res in (False, True):
                y, z = L.linear(d["x"], d["W"], d["bias"] if bias else None, act, d["residual"] if res else None)
                assert z is None
                _, _, ry, ty = ref_forward(s, act, False, bias, res)
                within(y, ry, ty, "y")
        whole = L.linear_backward(d["x"], d["W"], d["z"], d["dy"], act)
        for want in range(8):
            got = L.linear_backward(d["x"], d["W"], d["z"], d["dy"], act, False, *(bool(want >> i & 1) for i in range(3)))
            for i in range(3):
                assert got[i] is None if not want >> i & 1 else torch.equal(got[i], whole[i])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 96, 80), (40, 96, 80), (64, 4096, 72), (300, 65, 131)],
                         ids=lambda s: "x".join(map(str, s)))
def test_residual_in_place(dev, dtype, shape):
    """y given the residual's own memory, through the C ABI: one row, a tile, K cut into slices, odd sizes."""
    from mobilefinetuner_amd import capi, linear as L
    N, n_in, n_out = shape
    d = {k: v.to(dev) for k, v in make(*shape, dtype, 11).items()}
    for act in ("none", "silu"):
        ref = L.linear(d["x"], d["W"], d["bias"], act, d["residual"])[0]
        y = d["residual"].clone()
        desc = capi.linear_desc(N, n_in, n_out, capi.MFT_BF16 if dtype == "bf16" else capi.MFT_F32, False,
                                L.ACTIVATIONS[act])
        ws = torch.empty(max(1, capi.linear_workspace_size(desc)[0]), dtype=torch.uint8, device=dev)
        capi.linear_fwd(desc, d["x"].data_ptr(), d["W"].data_ptr(), d["bias"].data_ptr(), y.data_ptr(), y.data_ptr(),
                        None, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert torch.equal(y, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows_and_leading_dimensions(dev, dtype):
    from mobilefinetuner_amd import linear as L
    d = {k: v.to(dev) for k, v in make(6, 40, 24, dtype, 5).items()}
    y, z = L.linear(d["x"][:0], d["W"], d["bias"], "silu", want_preact=True)
    assert y.shape == z.shape == (0, 24)
    dx, dW, db = L.linear_backward(d["x"][:0], d["W"], z, y, "silu")
    assert dx.shape == (0, 40) and (dW == 0).all() and (db == 0).all()
    ref = L.linear(d["x"], d["W"], d["bias"], "none", d["residual"])[0]
    got = L.linear(d["x"].view(2, 3, 40), d["W"], d["bias"], "none", d["residual"].view(2, 3, 24))[0]
    assert got.shape == (2, 3, 24) and torch.equal(got.view(6, 24), ref)
    got = L.linear(d["x"][0], d["W"], d["bias"], "none", d["residual"][0])[0]
    assert got.shape == (24,)
    # operands that are not contiguous
    wide = torch.cat([d["x"], d["x"]], 1)
    assert torch.equal(L.linear(wide[:, 40:], d["W"].t().contiguous().t(), d["bias"], "none", d["residual"])[0], ref)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1, 4])
@pytest.mark.parametrize("N", [2, 70])
def test_operands_off_16_bytes(dev, N, offset):
    """Bases that no direct load takes: the same results (a product's terms in the same order)."""
    from mobilefinetuner_amd import linear as L
    d = {k: v.to(dev) for k, v in make(N, 128, 192, "bf16", 6).items()}

    def moved(t):
        u = torch.empty(t.numel() + offset, dtype=t.dtype, device=dev)[offset:].view(t.shape)
        return u.copy_(t)

    ref = L.linear(d["x"], d["W"], d["bias"], "silu", d["residual"], want_preact=True)
    got = L.linear(moved(d["x"]), moved(d["W"]), moved(d["bias"]), "silu", moved(d["residual"]), want_preact=True)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    ref = L.linear_backward(d["x"], d["W"], d["z"], d["dy"], "silu")
    got = L.linear_backward(moved(d["x"]), moved(d["W"]), moved(d["z"]), moved(d["dy"]), "silu")
    assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_that_are_not_numbers_stay_in_their_row(dev, dtype):
    from mobilefinetuner_amd import linear as L
    for N in (3, 150):
        d = {k: v.to(dev) for k, v in make(N, 100, 72, dtype, 8).items()}
        clean = L.linear(d["x"], d["W"], d["bias"], "gelu_tanh", d["residual"])[0]
        x = d["x"].clone()
        x[1, 99] = math.nan
        y = L.linear(x, d["W"], d["bias"], "gelu_tanh", d["residual"])[0]
        assert torch.isnan(y[1]).all()
        keep = [i for i in range(N) if i != 1]
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 40])
def test_relu_of_infinities(dev, N, dtype):
    from mobilefinetuner_amd import linear as L
    x, W = torch.zeros(N, 8, dtype=DT[dtype], device=dev), torch.ones(8, 3, dtype=DT[dtype], device=dev)
    y, z = L.linear(x, W, torch.tensor([-math.inf, math.inf, math.nan], device=dev), "relu", want_preact=True)
    assert (y[:, 0] == 0).all() and (y[:, 1] == math.inf).all() and torch.isnan(y[:, 2]).all()
    assert (z[:, 0] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_most_rows(dev, dtype):
    """2^29 rows, as many tiles as a launch takes: sums of two small whole numbers, exact in both types."""
    from mobilefinetuner_amd import linear as L
    N = 1 << 29
    x = torch.zeros(N, 2, dtype=DT[dtype], device=dev)
    x[-70:], x[:70] = 2, 1
    W, b = torch.tensor([[1.0], [3.0]], device=dev).to(DT[dtype]), torch.ones(1, device=dev)
    y = L.linear(x, W, b)[0]
    assert (y[-70:] == 9).all() and (y[:70] == 5).all() and (y[70:-70] == 1).all()
    dx, dW, db = L.linear_backward(x, W, None, y)
    assert torch.equal(dx[-1], (9 * W[:, 0])) and torch.equal(dx[0], 5 * W[:, 0]) and torch.equal(dx[100], W[:, 0])
    ref = 70 * (2 * 9 + 5)
    assert (dW.float() - ref).abs().max() <= torch.finfo(DT[dtype]).eps / 2 * ref


@pytest.mark.gpu
def test_far_pre_activations(dev):
    """Activations and derivatives far from zero: no NaN, their limits."""
    from mobilefinetuner_amd import linear as L
    for dtype in DT.values():
        z = torch.tensor([[-3e38, -1e20, -1e4, -90.0, -30.0, 30.0, 90.0, 1e4, 1e20, 3e38]], device=dev).to(dtype)
        one = torch.ones(1, 1, device=dev, dtype=dtype)
        for act in ("relu", "gelu_tanh", "silu"):
            y = L.linear(one, z, None, act)[0]
            assert torch.equal(y[0, 5:], z[0, 5:]) and (y[0, :4].abs() <= 1e-30).all()
            db = L.linear_backward(one, z, z, torch.ones_like(z), act)[2]
            assert torch.equal(db[5:], torch.ones(5, device=dev)) and (db[:4].abs() <= 1e-25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd_gradients_against_differences(dev, dtype):
    from mobilefinetuner_amd import linear as L
    d = {k: v.to(dev) for k, v in make(7, 48, 40, dtype, 9).items()}
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "W", "bias", "residual")}
    y = L.Linear.apply(*leaves.values(), "gelu_tanh", False)
    y.backward(d["dy"])
    z = L.linear(d["x"], d["W"], d["bias"], "gelu_tanh", want_preact=True)[1]
    ref = (*L.linear_backward(d["x"], d["W"], z, d["dy"], "gelu_tanh"), d["dy"])
    assert all(torch.equal(t.grad, r) for t, r in zip(leaves.values(), ref))
    if dtype == "bf16":
        return
    g, step = torch.Generator().manual_seed(1), 2.0 ** -7
    for name in leaves:
        v = torch.randn(d[name].shape, generator=g).to(dev)
        loss = []
        for s in (step, -step):
            q = {**d, name: d[name] + s * v}
            loss.append(float((L.linear(q["x"], q["W"], q["bias"], "gelu_tanh", q["residual"])[0].double()
                               * d["dy"].double()).sum()))
        slope, along = (loss[0] - loss[1]) / (2 * step), float((leaves[name].grad.double() * v.double()).sum())
        # the third derivative along v, at most a few times sum |dy| |dz|^3, and the loss's rounding
        dz = (v.double() @ d["W"].double() if name == "x" else d["x"].double() @ v.double() if name == "W"
              else v.double().expand(7, 40))
        scale = float((d["dy"].double().abs() * (1 + dz.abs() ** 3)).sum())
        assert abs(slope - along) <= scale * (step * step + 64 * U / step)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 512, 256), (200, 512, 256), (96, 4096, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_graph_and_streams(dev, shape, dtype):
    from mobilefinetuner_amd import linear as L
    d = {k: v.to(dev) for k, v in make(*shape, dtype, 10).items()}

    def step():
        y, z = L.linear(d["x"], d["W"], d["bias"], "silu", d["residual"], want_preact=True)
        return (y, z, *L.linear_backward(d["x"], d["W"], z, d["dy"], "silu"))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        for k, v in make(*shape, dtype, seed).items():
            d[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
    ref = [t.clone() for t in step()]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(p, q) for p, q in zip(r, ref))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_block_with_its_norm_and_scored_tokens(dev, dtype):
    """The operators as a model runs them: h + W2 gelu(W1 LN(h) + b1) + b2, a last norm, the head,
    the given tokens' log probabilities; gradients of every parameter against the same graph of
    torch's own operators in 64 bits."""
    from mobilefinetuner_amd import layer_norm as LN, linear as L, logprobs as P
    g = torch.Generator().manual_seed(20)
    t, N, D, V = DT[dtype], 24, 64, 500
    p = dict(h=torch.randn(N, D, generator=g).to(t), w1=(torch.randn(D, 4 * D, generator=g) / 8).to(t),
             w2=(torch.randn(4 * D, D, generator=g) / 16).to(t), head=(torch.randn(V, D, generator=g) / 8).to(t),
             g1=1 + 0.1 * torch.randn(D, generator=g), c1=0.1 * torch.randn(D, generator=g),
             g2=1 + 0.1 * torch.randn(D, generator=g), c2=0.1 * torch.randn(D, generator=g),
             b1=0.1 * torch.randn(4 * D, generator=g), b2=0.1 * torch.randn(D, generator=g))
    tok = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    tok[5] = -100
    a, b = torch.randn(N, generator=g), 0.1 * torch.randn(N, generator=g)

    q = {k: v.to(dev).requires_grad_(True) for k, v in p.items()}
    u = L.Linear.apply(LN.LayerNorm.apply(q["h"], q["g1"], q["c1"], 1e-5), q["w1"], q["b1"], None, "gelu_tanh", False)
    r = L.Linear.apply(u, q["w2"], q["b2"], q["h"], "none", False)
    logits = L.Linear.apply(LN.LayerNorm.apply(r, q["g2"], q["c2"], 1e-5), q["head"], None, None, "none", True)
    lp, ent = P.TokenLogprobs.apply(logits, tok.to(dev))
    ((lp * a.to(dev)).sum() + (ent * b.to(dev)).sum()).backward()

    e = {k: v.double().requires_grad_(True) for k, v in p.items()}
    u = F.gelu(F.layer_norm(e["h"], (D,), e["g1"], e["c1"], 1e-5) @ e["w1"] + e["b1"], approximate="tanh")
    r = e["h"] + u @ e["w2"] + e["b2"]
    lsm = torch.log_softmax(F.layer_norm(r, (D,), e["g2"], e["c2"], 1e-5) @ e["head"].t(), -1)
    on = (tok >= 0).double()
    rlp = lsm.gather(1, tok.long().clamp(min=0)[:, None])[:, 0] * on
    rent = -(lsm.exp() * lsm).sum(-1) * on
    ((rlp * a).sum() + (rent * b).sum()).backward()

    # Seven tensors are rounded on the way forward and as many gradients on the way back: each by
    # half a step, 2^-9 of its norm at the most (uniform within the step: 2^-8 / sqrt(3) a value at
    # the foot of a binade, less elsewhere), amplified at most by the norms' and the softmax's
    # slopes (under 4 here): 14 * 4 * 2^-9 = 0.11 of a gradient's norm, if all of them added up; as
    # independent errors their root, 0.03.  fp32: the same of 2^-25, times sums of 500 terms.
    bound = 0.11 if dtype == "bf16" else 14 * 4 * 2.0 ** -25 * 500
    assert float((lp.detach().cpu().double() - rlp.detach()).norm() / rlp.detach().norm()) <= bound
    for k in p:
        assert q[k].grad.dtype == p[k].dtype
        rel = float((q[k].grad.cpu().double() - e[k].grad).norm() / e[k].grad.norm())
        assert rel <= bound, (k, rel)


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


@pytest.mark.parametrize("change,message", [
    (dict(N=-1), "N >= 0"), (dict(in_dim=0), "positive"), (dict(out_dim=-4), "positive"), (dict(dtype=1), "dtype"),
    (dict(activation=4), "activation"), (dict(activation=-1), "activation"), (dict(in_dim=1 << 25), "2\\^24"),
    (dict(N=1 << 31), "2\\^31"), (dict(N=1 << 24, in_dim=1 << 16), "too large"),
    (dict(N=(1 << 29) + 1), "too large"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.linear_desc(**{**dict(N=4, in_dim=64, out_dim=32), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.linear_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.linear_fwd(d, 16, 32, None, None, 48, None, 64, None)
    with pytest.raises(capi.MftError, match=message):
        capi.linear_bwd(d, 16, 32, None, 48, 64, 80, None, 96, None)


@pytest.mark.parametrize("dtype", [0, 2])
def test_null_and_aliased_operands_refused(capi, dtype):
    act = capi.linear_desc(4, 64, 32, dtype, False, capi.MFT_ACT_SILU)
    plain = capi.linear_desc(4, 64, 32, dtype)
    good = [16, 32, None, None, 48, None, 64]
    for i in (0, 1, 4):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.linear_fwd(plain, *[None if j == i else a for j, a in enumerate(good)], None)
    with pytest.raises(capi.MftError, match="activation only"):
        capi.linear_fwd(plain, 16, 32, None, None, 48, 80, 64, None)
    for y, z, res in ((16, None, None), (32, None, None), (48, 48, None), (48, 16, None), (48, 80, 80)):
        with pytest.raises(capi.MftError, match="may not be"):
            capi.linear_fwd(act, 16, 32, None, res, y, z, 64, None)
    cut = capi.linear_desc(1, 1 << 14, 8, dtype)
    if capi.linear_workspace_size(cut)[0]:
        with pytest.raises(capi.MftError, match="workspace"):
            capi.linear_fwd(cut, 16, 32, None, None, 48, None, None, None)
    good = [16, 32, 48, 64, 80, 96, 112, 128]
    for i in (0, 1, 2, 3, 7):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.linear_bwd(act, *[None if j == i else a for j, a in enumerate(good)], None)
    for dx, dW in ((64, None), (16, None), (32, None), (48, None), (None, 32), (None, 16), (None, 64), (None, 48)):
        with pytest.raises(capi.MftError, match="may not be"):
            capi.linear_bwd(act, 16, 32, 48, 64, dx, dW, None, 128, None)
    empty = capi.linear_desc(0, 64, 32, dtype)
    assert capi.lib().mft_linear_fwd(C.byref(empty), *[None] * 8) == capi.MFT_OK
    assert capi.lib().mft_linear_bwd(C.byref(act), 16, 32, 48, 64, None, None, None, 128, None) == capi.MFT_OK


@pytest.mark.parametrize("dtype", [0, 2])
def test_outputs_over_weights_or_each_other_refused(capi, dtype):
    d = capi.linear_desc(4, 64, 32, dtype, False, capi.MFT_ACT_SILU)
    with pytest.raises(capi.MftError, match="may not be"):
        capi.linear_fwd(d, 16, 32, None, None, 48, 32, 64, None)
    with pytest.raises(capi.MftError, match="may not be one"):
        capi.linear_bwd(d, 16, 32, 48, 64, 80, 80, None, 128, None)


def test_no_cpu_path():
    from mobilefinetuner_amd import linear as L
    with pytest.raises(ValueError, match="no CPU path"):
        L.linear(torch.zeros(2, 4), torch.zeros(4, 4))


@pytest.mark.gpu
def test_operands_that_do_not_fit_refused(dev):
    from mobilefinetuner_amd import linear as L
    x, W, b = torch.zeros(2, 8, device=dev), torch.zeros(8, 6, device=dev), torch.zeros(6, device=dev)
    y = torch.zeros(2, 6, device=dev)
    for bad in (lambda: L.linear(x, W[:7]), lambda: L.linear(x, W, w_transposed=True), lambda: L.linear(x, W.bfloat16()),
                lambda: L.linear(x, W, b[:5]), lambda: L.linear(x, W, b, "gelu"), lambda: L.linear(x, W.cpu()),
                lambda: L.linear(x, W, b, residual=x), lambda: L.linear(x, W, b, want_preact=True),
                lambda: L.linear(x.bfloat16(), W.bfloat16(), b.bfloat16()),
                lambda: L.linear_backward(x, W, None, y, "silu"), lambda: L.linear_backward(x, W, None, y[:1])):
        with pytest.raises(ValueError):
            bad()
