"""Layer norm (mft_layer_norm_* through the torch helpers) against its formula in
64 bits, and its refusals.

Bounds, per element, with u = 2^-24 and K = 80 (the longest chain of fp32
additions of a row's sum: 64 values of a thread, then the tree over threads).
A mean above the deviation is corrected by the sum about it, so its error is K u
of the mean deviation, which rstd scales to at most 1; one below has K u of the
mean magnitude, at most sqrt(2) deviations.  rstd's relative error is half of its
sum's and a few roundings.  So h = (x - mean) rstd is off by
u ((K / 2 + 8) |h| + 2 K), and y by |w| times that, the roundings of the
product and the sum, and half a step of its type.  The backward takes the
statistics as given: h is off by 3 u |h|, the two row sums by (K + 4) u of the
sums of magnitudes, and a sum over N rows by (N + 64) u of its magnitudes.
"""
import ctypes as C
import math

import pytest
import torch

U = 2.0 ** -24
K = 80
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


def make(N, D, dtype, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, D, generator=g) * (0.5 + torch.rand(N, 1, generator=g)) + offset).to(DT[dtype])
    w, b = 1 + 0.2 * torch.randn(D, generator=g), 0.1 * torch.randn(D, generator=g)
    dy = (0.1 * torch.randn(N, D, generator=g)).to(DT[dtype])
    return x, w, b, dy


def ref_stats(x, eps):
    xd = x.double()
    mean = xd.mean(-1)
    return mean, 1 / torch.sqrt(((xd - mean[..., None]) ** 2).mean(-1) + eps)


def ref_forward(x, w, b, eps):
    mean, rstd = ref_stats(x, eps)
    h = (x.double() - mean[..., None]) * rstd[..., None]
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    y = h * wd + (0 if b is None else b.double())
    bound = wd.abs() * U * ((K / 2 + 8) * h.abs() + 2 * K) + 3 * U * (y.abs() + (h * wd).abs())
    return y, bound + half_step(x.dtype) * y.abs(), mean, rstd


def ref_backward(x, w, mean, rstd, dy):
    xd, dyd, r = x.double(), dy.double(), rstd.double()[:, None]
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    h = (xd - mean.double()[:, None]) * r
    g = dyd * wd
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - c1 - h * c2)
    a1, a2 = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    tol = U * r * (4 * g.abs() + (K + 6) * a1 + (K + 12) * h.abs() * a2) + half_step(x.dtype) * dx.abs()
    n = x.shape[0]
    tol_w = U * (n + 68) * (dyd * h).abs().sum(0)
    tol_b = U * (n + 64) * dyd.abs().sum(0)
    return dx, (dyd * h).sum(0), dyd.sum(0), tol + 1e-300, tol_w + 1e-300, tol_b + 1e-300


def within(got, ref, tol):
    off = (got.detach().cpu().double() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


# one element, below a vector, off the vectors, each count of waves and chunks, beyond registers
WIDTHS = [1, 2, 7, 64, 65, 255, 256, 513, 768, 1153, 2047, 4100, 8193, 20000, 40001, 70000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_forward_and_backward(dev, D, dtype):
    from mobilefinetuner_amd import layer_norm as L
    N = 5 if D > 8000 else 37
    print(f"[case] D {D} {dtype}", flush=True)
    x, w, b, dy = make(N, D, dtype, D)
    y, mean, rstd = L.layer_norm(x.to(dev), w.to(dev), b.to(dev), 1e-5)
    ry, tol, rmean, rrstd = ref_forward(x, w, b, 1e-5)
    within(y, ry, tol)
    within(rstd, rrstd, U * (K / 2 + 8) * rrstd)
    within(mean, rmean, U * (2 * rmean.abs() + 2 * K / rrstd) + 1e-300)
    dx, dw, db = L.layer_norm_backward(x.to(dev), w.to(dev), mean, rstd, dy.to(dev))
    rdx, rdw, rdb, t, tw, tb = ref_backward(x, w, mean.cpu(), rstd.cpu(), dy)
    assert dx.dtype == x.dtype and dw.dtype == db.dtype == torch.float32
    within(dx, rdx, t)
    within(dw, rdw, tw)
    within(db, rdb, tb)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [0, 1, 3, 1000, 5000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_row_counts(dev, N, dtype):
    """No row, one, fewer than a workgroup takes, more than all workgroups take at once."""
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, dy = make(N, 200, dtype, N)
    y, mean, rstd = L.layer_norm(x.to(dev), w.to(dev), b.to(dev))
    dx, dw, db = L.layer_norm_backward(x.to(dev), w.to(dev), mean, rstd, dy.to(dev))
    assert y.shape == x.shape and mean.shape == rstd.shape == (N,) and dx.shape == x.shape
    ry, tol, _, _ = ref_forward(x, w, b, 1e-5)
    within(y, ry, tol)
    rdx, rdw, rdb, t, tw, tb = ref_backward(x, w, mean.cpu(), rstd.cpu(), dy)
    within(dx, rdx, t)
    within(dw, rdw, tw)
    within(db, rdb, tb)


@pytest.mark.gpu
def test_a_mean_far_above_the_deviation(dev):
    """x = 4096 + normal values: the corrected mean keeps the digits that the fp32 input has."""
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, _ = make(9, 1500, "f32", 4, offset=4096.0)
    y, _, _ = L.layer_norm(x.to(dev), w.to(dev), b.to(dev))
    ry, tol, _, _ = ref_forward(x, w, b, 1e-5)
    within(y, ry, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_parameters_and_parts_of_the_gradient(dev, dtype):
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, dy = (t.to(dev) for t in make(33, 300, dtype, 5))
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, mean, rstd = L.layer_norm(x, ww, bb)
        ry, tol, _, _ = ref_forward(x.cpu(), None if ww is None else w.cpu(), None if bb is None else b.cpu(), 1e-5)
        within(y, ry, tol)
        whole = L.layer_norm_backward(x, ww, mean, rstd, dy)
        rdx, rdw, rdb, t, tw, tb = ref_backward(x.cpu(), None if ww is None else w.cpu(), mean.cpu(), rstd.cpu(),
                                                dy.cpu())
        within(whole[0], rdx, t)
        within(whole[1], rdw, tw)
        within(whole[2], rdb, tb)
        only = L.layer_norm_backward(x, ww, mean, rstd, dy, want_params=False)
        assert torch.equal(only[0], whole[0]) and only[1] is None and only[2] is None
        only = L.layer_norm_backward(x, ww, mean, rstd, dy, want_x=False)
        assert only[0] is None and torch.equal(only[1], whole[1]) and torch.equal(only[2], whole[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows(dev, dtype):
    """Columns of a wider tensor (rows off every vector boundary), a transposed batch, rows given
    several times, and a last dimension that is not contiguous: the results of a copy."""
    from mobilefinetuner_amd import layer_norm as L
    wide = make(24, 701, dtype, 6)[0].to(dev)
    w, b = (t.to(dev) for t in make(1, 300, dtype, 6)[1:3])
    views = [wide[:, 3:303], wide[:, 100:400].reshape(4, 6, 300).transpose(0, 1), wide[:1, 5:305].expand(7, 300),
             wide[:, :600:2], wide[::2, 401:701]]
    for v in views:
        c = v.contiguous()
        y, mean, rstd = L.layer_norm(v, w, b)
        yc, mc, rc = L.layer_norm(c, w, b)
        assert torch.equal(y, yc) and torch.equal(mean, mc) and torch.equal(rstd, rc)
        got = L.layer_norm_backward(v, w, mean, rstd, v)
        ref = L.layer_norm_backward(c, w, mean, rstd, c)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the last rows' results are those of a call of their own."""
    from mobilefinetuner_amd import layer_norm as L
    N, D = (1 << 20) + 300, 2056
    x = torch.zeros(N, D, dtype=torch.bfloat16, device=dev)
    last, w, b, dy = (t.to(dev) for t in make(5, D, "bf16", 14))
    x[-5:] = last
    y, mean, rstd = L.layer_norm(x, w, b)
    ref = L.layer_norm(last, w, b)
    assert torch.equal(y[-5:], ref[0]) and torch.equal(mean[-5:], ref[1]) and torch.equal(rstd[-5:], ref[2])
    assert torch.equal(y[0], b.bfloat16())
    y.zero_()  # as dy, but for the last rows
    y[-5:] = dy
    dx, dw, _ = L.layer_norm_backward(x, w, mean, rstd, y)
    assert torch.equal(dx[-5:], L.layer_norm_backward(last, w, *ref[1:], dy)[0]) and (dx[:5] == 0).all()
    del x, y, dx


@pytest.mark.gpu
@pytest.mark.parametrize("N,D", [((1 << 25) + 70, 8), ((1 << 21) + 3, 16400)])
def test_more_rows_than_a_launch_takes(dev, N, D):
    """Rows held by a wave, by sixteen, and their last ones as in a call of their own."""
    from mobilefinetuner_amd import layer_norm as L
    x = torch.zeros(N, D, dtype=torch.bfloat16, device=dev)
    last, w, b, dy = (t.to(dev) for t in make(5, D, "bf16", 15))
    x[-5:] = last
    y, mean, rstd = L.layer_norm(x, w, b)
    ref = L.layer_norm(last, w, b)
    assert all(torch.equal(p[-5:], q) for p, q in zip((y, mean, rstd), ref))
    assert torch.equal(y[0], b.bfloat16()) and torch.equal(y[N - 6], y[0]) and (rstd[:-5] == rstd[0]).all()
    if D > 16384:  # beyond the backward's registers
        y.zero_()
        y[-5:] = dy
        dx = L.layer_norm_backward(x, w, mean, rstd, y, want_params=False)[0]
        assert torch.equal(dx[-5:], L.layer_norm_backward(last, w, *ref[1:], dy, want_params=False)[0])
        del dx
    del x, y


@pytest.mark.gpu
@pytest.mark.parametrize("D", [(1 << 25) + 33, 1 << 26, (1 << 26) + 4099])
def test_wider_rows_than_a_launch_takes(dev, D):
    """The parameters' gradients on either side of a launch's columns.  Multiples of 1/2 whose sums stay below
    2^23 (a thread's share of a row is some 2^16 products of at most 50, of mean zero): all sums are exact, and
    dx has the roundings of its last few operations."""
    from mobilefinetuner_amd import layer_norm as L
    print(f"[case] D {D}", flush=True)
    j = torch.arange(D, device=dev)
    x = torch.stack([j % 13 - 6, j % 7 - 3]).bfloat16()
    dy = torch.stack([j % 5 - 2, j % 11 - 5]).bfloat16()
    mean, rstd = torch.tensor([1.0, -2.0], device=dev), torch.tensor([0.5, 2.0], device=dev)
    dx, dw, db = L.layer_norm_backward(x, None, mean, rstd, dy)
    h = (x.float() - mean[:, None]) * rstd[:, None]
    assert torch.equal(db, dy.float().sum(0)) and torch.equal(dw, (dy.float() * h).sum(0))
    c1, c2 = (dy.double().mean(1, keepdim=True), (dy.double() * h.double()).mean(1, keepdim=True))
    ref = rstd.double()[:, None] * (dy.double() - c1 - h.double() * c2)
    tol = 8 * U * rstd.double()[:, None] * (dy.abs() + c1.abs() + (h * c2).abs()) + half_step(x.dtype) * ref.abs()
    assert bool(((dx.double() - ref).abs() <= tol).all())
    del x, dy, dx, h, ref, tol


@pytest.mark.gpu
def test_values_that_are_not_numbers_stay_in_their_row(dev):
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, dy = (t.to(dev) for t in make(8, 257, "f32", 7))
    clean = L.layer_norm(x, w, b)[0]
    x2 = x.clone()
    x2[2, 100], x2[5, 256], x2[6, 0] = math.nan, math.inf, -math.inf
    y = L.layer_norm(x2, w, b)[0]
    assert torch.isnan(y[[2, 5, 6]]).all()
    keep = [0, 1, 3, 4, 7]
    assert torch.equal(y[keep], clean[keep])
    zero = torch.full((2, 257), 3.5, device=dev)  # no deviation: eps alone
    y, mean, rstd = L.layer_norm(zero, w, b, 1e-5)
    assert torch.equal(mean, zero[:, 0]) and torch.allclose(y, b.expand(2, 257), rtol=0, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd_gradients_against_differences(dev, dtype):
    """The autograd node's gradients are the helpers', and (fp32) those of differences: the loss
    sum(y c) moves by the gradient along a direction v, to the second order of the step
    (t^2 times a third derivative of order one) and the loss's rounding over the step."""
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, c = (t.to(dev) for t in make(6, 130, dtype, 8))
    x, w, b = (t.clone().requires_grad_(True) for t in (x, w, b))
    y = L.LayerNorm.apply(x, w, b, 1e-5)
    y.backward(c)
    _, mean, rstd = L.layer_norm(x.detach(), w.detach(), b.detach())
    for g, r in zip((x.grad, w.grad, b.grad), L.layer_norm_backward(x.detach(), w.detach(), mean, rstd, c)):
        assert torch.equal(g, r)
    if dtype == "bf16":
        return
    g = torch.Generator().manual_seed(1)
    t = 2.0 ** -7
    for p in (x, w, b):
        v = torch.randn(p.shape, generator=g).to(dev)
        loss = []
        with torch.no_grad():
            for s in (t, -t):
                q = [u + s * v if u is p else u for u in (x, w, b)]
                loss.append((L.layer_norm(*q)[0].double() * c.double()).sum().item())
        slope = (loss[0] - loss[1]) / (2 * t)
        scale = float(c.double().norm() * v.double().norm())
        assert abs(slope - float((p.grad.double() * v.double()).sum())) <= scale * (4 * t * t + 256 * U / t)


@pytest.mark.gpu
def test_repeated_calls_and_streams(dev):
    """The same bits from every call, also from two streams at once, each with its own workspace."""
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, dy = (t.to(dev) for t in make(3000, 768, "bf16", 9))
    y, mean, rstd = L.layer_norm(x, w, b)
    ref = L.layer_norm_backward(x, w, mean, rstd, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(L.layer_norm_backward(x, w, mean, rstd, dy))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(p, q) for p, q in zip(r, ref))


@pytest.mark.gpu
def test_captured_graph_follows_its_inputs(dev):
    from mobilefinetuner_amd import layer_norm as L
    x, w, b, dy = (t.to(dev) for t in make(500, 640, "bf16", 10))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, mean, rstd = L.layer_norm(x, w, b)
        L.layer_norm_backward(x, w, mean, rstd, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = L.layer_norm(x, w, b)
        grads = L.layer_norm_backward(x, w, mean, rstd, dy)
    for seed in (11, 12, 13):
        nx, _, _, ndy = make(500, 640, "bf16", seed)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        ry, rm, rr = L.layer_norm(x, w, b)
        assert torch.equal(y, ry) and torch.equal(mean, rm) and torch.equal(rstd, rr)
        assert all(torch.equal(p, q) for p, q in zip(grads, L.layer_norm_backward(x, w, rm, rr, dy)))


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


@pytest.mark.parametrize("change,message", [
    (dict(N=-1), "N >= 0"), (dict(D=0), "D > 0"), (dict(D=(1 << 30) + 1), "at most"), (dict(dtype=1), "dtype"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(x_stride=63), "stride"),
    (dict(dy_stride=-64), "stride"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.layer_norm_desc(**{**dict(N=4, D=64), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.layer_norm_fwd(d, 16, None, None, 32, None, None, None)
    with pytest.raises(capi.MftError, match=message):
        capi.layer_norm_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.layer_norm_bwd(d, 16, None, 16, 16, 16, 32, None, None, 64, None)


def test_null_and_aliased_operands_refused(capi):
    d = capi.layer_norm_desc(4, 64)
    for args in ((None, None, None, 32, None, None), (16, None, None, None, None, None)):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.layer_norm_fwd(d, *args, None)
    good = [16, None, 32, 48, 64, 80, None, None, 96]
    for i in (0, 2, 3, 4, 8):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.layer_norm_bwd(d, *[None if j == i else a for j, a in enumerate(good)], None)
    with pytest.raises(capi.MftError, match="may not be x"):
        capi.layer_norm_bwd(d, 16, None, 32, 48, 64, 16, None, None, 96, None)
    assert capi.lib().mft_layer_norm_fwd(None, 16, None, None, 32, None, None, None) == capi.MFT_ERR_INVALID_ARG
    assert capi.lib().mft_layer_norm_fwd(C.byref(capi.layer_norm_desc(0, 64)), None, None, None, None, None, None,
                                         None) == capi.MFT_OK


def test_in_place_with_other_strides_refused(capi):
    """Rows would be overwritten before they are read."""
    with pytest.raises(capi.MftError, match="in place"):
        capi.layer_norm_fwd(capi.layer_norm_desc(4, 64, x_stride=80), 16, None, None, 16, None, None, None)
    with pytest.raises(capi.MftError, match="in place"):
        capi.layer_norm_bwd(capi.layer_norm_desc(4, 64, dx_stride=80), 16, None, 32, 48, 64, 64, None, None, 96, None)


def test_no_cpu_path():
    from mobilefinetuner_amd import layer_norm as L
    with pytest.raises(ValueError, match="no CPU path"):
        L.layer_norm(torch.zeros(2, 4))


@pytest.mark.gpu
def test_operands_that_do_not_fit_refused(dev):
    from mobilefinetuner_amd import layer_norm as L
    x, w = torch.zeros(2, 8, device=dev), torch.ones(8, device=dev)
    s = torch.zeros(2, device=dev)
    for bad in (lambda: L.layer_norm(x, w[:7]), lambda: L.layer_norm(x, w.bfloat16()), lambda: L.layer_norm(x, w.cpu()),
                lambda: L.layer_norm(x.half()), lambda: L.layer_norm(x[:, :0]),
                lambda: L.layer_norm_backward(x, w, s[:1], s, x), lambda: L.layer_norm_backward(x, w, s, s, x.bfloat16()),
                lambda: L.layer_norm_backward(x, w, s, s, x[:1])):
        with pytest.raises(ValueError):
            bad()
