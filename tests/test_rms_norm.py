"""The root-mean-square norm (mft_rms_norm_* through the torch helpers) against its
formula in 64 bits, and its refusals.

Bounds, per element, with u = 2^-24 and K = 80 (the longest chain of fp32
additions of a row's sum: 64 values of a thread, then the tree over threads).
The sum of squares is off by K u of itself, rstd by (K / 2 + 4) u of itself, and
y = s rstd f by that, the roundings of f and of two products, and half a step
of its type.  s itself is the sum in fp32 rounded to the rows' type, to the bit.
In 8 bits y / scale is rounded by at most 2^-4 of itself, or half the smallest
number (2^-10) below the normal ones, and the scale is off as y is.  The backward
takes rstd as given: h is off by u |h|, the row's sum by (K + 4) u of its
magnitudes, and a sum over N rows by (N + 64) u of its magnitudes.
"""
import ctypes as C
import math

import pytest
import torch

U = 2.0 ** -24
K = 80
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
NORMS = ["gemma", "affine"]


def half_step(t):
    return torch.finfo(t).eps / 2


def make(N, D, dtype, seed):
    """x, residual, weight, dy, dtotal."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, D, generator=g) * (0.5 + torch.rand(N, 1, generator=g))).to(DT[dtype])
    r = torch.randn(N, D, generator=g).to(DT[dtype])
    w = 0.3 * torch.randn(D, generator=g)
    dy, dt = ((0.1 * torch.randn(N, D, generator=g)).to(DT[dtype]) for _ in range(2))
    return x, r, w, dy, dt


def factor(w, norm, D):
    if w is None:
        return torch.ones(D, dtype=torch.float64)
    return w.double() + (1 if norm == "gemma" else 0)


def total_of(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def ref_forward(s, w, norm, eps):
    """(y, its bound before the last rounding, rstd) from the stream s."""
    sd = s.double()
    rstd = 1 / torch.sqrt((sd * sd).mean(-1) + eps)
    y = sd * rstd[..., None] * factor(w, norm, s.shape[-1])
    return y, U * (K / 2 + 12) * y.abs() + 1e-300, rstd


def ref_backward(s, w, norm, rstd, dy, dt):
    sd, dyd, r = s.double(), dy.double(), rstd.double()[:, None]
    h = sd * r
    g = dyd * factor(w, norm, s.shape[-1])
    c2, a2 = (g * h).mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    dx = r * (g - h * c2)
    tol = U * (r * (5 * g.abs() + (K + 12) * h.abs() * a2) + dx.abs())
    if dt is not None:
        dx = dx + dt.double()
    tol = tol + (U + half_step(s.dtype)) * dx.abs() + 1e-300
    return dx, (dyd * h).sum(0), tol, U * (s.shape[0] + 68) * (dyd * h).abs().sum(0) + 1e-300


def within(got, ref, tol):
    off = (got.detach().cpu().double() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def e4m3_within(q, scale, y, tol):
    """q * scale against y, which is known to tol before its rounding."""
    top = y.abs().amax(-1)
    rs = (top / 448).clamp(min=2.0 ** -126)
    slack = (U * (K / 2 + 16)) * rs
    within(scale, rs, slack)
    got = q.float().cpu().double() * scale.cpu().double()[..., None]
    within(got, y, (2.0 ** -4 + 4 * U) * y.abs() + 1.1 * tol + (2.0 ** -10 * (1 + 2.0 ** -10)) * rs[..., None])
    assert bool((q.float().abs().amax(-1).cpu() == 448).all()) or bool((top < 448 * 2.0 ** -120).any())


# one element, below a vector, off the vectors, each count of waves and chunks, beyond registers
WIDTHS = [1, 2, 7, 64, 65, 255, 256, 513, 768, 1152, 1153, 1800, 2047, 4100, 8193, 20000, 40001, 70000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_forward_and_backward(dev, D, dtype):
    from mobilefinetuner_amd import rms_norm as L
    N = 5 if D > 8000 else 37
    print(f"[case] D {D} {dtype}", flush=True)
    x, r, w, dy, dt = make(N, D, dtype, D)
    for norm, res, dtot in (("gemma", r, dt), ("affine", None, None)):
        on = [None if t is None else t.to(dev) for t in (x, r if res is not None else None, w, dy, dtot)]
        s = total_of(x, res)
        y, total, rstd = L.rms_norm(on[0], on[2], on[1], norm, 1e-6)
        assert total is None if res is None else torch.equal(total.cpu(), s)
        ry, tol, rr = ref_forward(s, w, norm, 1e-6)
        assert y.dtype == x.dtype
        within(y, ry, tol + half_step(x.dtype) * ry.abs())
        within(rstd, rr, U * (K / 2 + 4) * rr)
        sd = on[0] if total is None else total
        dx, dw = L.rms_norm_backward(sd, on[2], rstd, on[3], on[4], norm)
        rdx, rdw, t, tw = ref_backward(s, w, norm, rstd.cpu(), dy, dtot)
        assert dx.dtype == x.dtype and dw.dtype == torch.float32
        within(dx, rdx, t)
        within(dw, rdw, tw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_eight_bits(dev, D, dtype):
    from mobilefinetuner_amd import rms_norm as L
    N = 5 if D > 8000 else 37
    print(f"[case] D {D} {dtype}", flush=True)
    x, r, w, _, _ = make(N, D, dtype, D)
    for norm, res in (("gemma", r), ("affine", None)):
        s = total_of(x, res)
        q, scale, total = L.rms_norm_e4m3(x.to(dev), w.to(dev), None if res is None else res.to(dev), norm, 1e-6)
        assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (N,)
        assert total is None if res is None else torch.equal(total.cpu(), s)
        ry, tol, _ = ref_forward(s, w, norm, 1e-6)
        e4m3_within(q, scale, ry, tol)
    q, scale = L.quantize_rows(x.to(dev))
    e4m3_within(q, scale, x.double(), torch.full((), 1e-300))


@pytest.mark.gpu
def test_rows_that_e4m3_holds_exactly(dev):
    """Rows of e4m3 numbers times a power of two with a 448 among them come back to the bit, zeros and
    the smallest scale among them."""
    from mobilefinetuner_amd import rms_norm as L
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[~torch.isnan(codes)]
    x = torch.stack([codes * 2.0 ** e for e in (0, -30, 40, -126)])
    q, scale = L.quantize_rows(x.to(dev))
    assert torch.equal(scale.cpu(), torch.tensor([1.0, 2.0 ** -30, 2.0 ** 40, 2.0 ** -126]))
    assert torch.equal(q.float().cpu(), codes.expand(4, -1))
    q, scale = L.quantize_rows(torch.zeros(3, 77, device=dev))
    assert (q.float() == 0).all() and (scale == 2.0 ** -126).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [0, 1, 3, 1000, 5000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_row_counts(dev, N, dtype):
    """No row, one, fewer than a workgroup takes, more than all workgroups take at once."""
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = make(N, 200, dtype, N)
    y, total, rstd = L.rms_norm(x.to(dev), w.to(dev), r.to(dev))
    dx, dw = L.rms_norm_backward(total, w.to(dev), rstd, dy.to(dev), dt.to(dev))
    assert y.shape == total.shape == dx.shape == x.shape and rstd.shape == (N,)
    s = total_of(x, r)
    ry, tol, _ = ref_forward(s, w, "gemma", 1e-6)
    within(y, ry, tol + half_step(x.dtype) * ry.abs())
    rdx, rdw, t, tw = ref_backward(s, w, "gemma", rstd.cpu(), dy, dt)
    within(dx, rdx, t)
    within(dw, rdw, tw)
    q, scale, _ = L.rms_norm_e4m3(x.to(dev), w.to(dev), r.to(dev))
    assert q.shape == x.shape and scale.shape == (N,)
    e4m3_within(q, scale, ry, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_a_weight_and_parts_of_the_gradient(dev, dtype):
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = (t.to(dev) for t in make(33, 300, dtype, 5))
    for ww, norm in ((None, "gemma"), (w, "gemma"), (None, "affine"), (w, "affine")):
        y, _, rstd = L.rms_norm(x, ww, None, norm)
        wc = None if ww is None else w.cpu()
        ry, tol, _ = ref_forward(x.cpu(), wc, norm, 1e-6)
        within(y, ry, tol + half_step(x.dtype) * ry.abs())
        for d in (None, dt):
            whole = L.rms_norm_backward(x, ww, rstd, dy, d, norm)
            rdx, rdw, t, tw = ref_backward(x.cpu(), wc, norm, rstd.cpu(), dy.cpu(), None if d is None else dt.cpu())
            within(whole[0], rdx, t)
            within(whole[1], rdw, tw)
            only = L.rms_norm_backward(x, ww, rstd, dy, d, norm, want_weight=False)
            assert torch.equal(only[0], whole[0]) and only[1] is None
            only = L.rms_norm_backward(x, ww, rstd, dy, d, norm, want_x=False)
            assert only[0] is None and torch.equal(only[1], whole[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows(dev, dtype):
    """Columns of a wider tensor (rows off every vector boundary), a transposed batch, rows given
    several times, and a last dimension that is not contiguous: the results of a copy."""
    from mobilefinetuner_amd import rms_norm as L
    wide, other = (t.to(dev) for t in make(24, 701, dtype, 6)[:2])
    w = make(1, 300, dtype, 6)[2].to(dev)
    cuts = [lambda t: t[:, 3:303], lambda t: t[:, 100:400].reshape(4, 6, 300).transpose(0, 1),
            lambda t: t[:1, 5:305].expand(7, 300), lambda t: t[:, :600:2], lambda t: t[::2, 401:701]]
    for cut in cuts:
        v, r = cut(wide), cut(other)
        c, rc = v.contiguous(), r.contiguous()
        got, ref = L.rms_norm(v, w, r), L.rms_norm(c, w, rc)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
        got8, ref8 = L.rms_norm_e4m3(v, w, r), L.rms_norm_e4m3(c, w, rc)
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(got8, ref8))
        rstd = ref[2]
        got, ref = L.rms_norm_backward(v, w, rstd, r, v), L.rms_norm_backward(c, w, rstd, rc, c)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [300, 1152, 40001])
def test_outputs_in_place(dev, D):
    """The C ABI's in-place forms: total over the residual, y over x, dx over dy or dtotal."""
    from mobilefinetuner_amd import capi
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = (t.to(dev) for t in make(9, D, "bf16", 3))
    y, total, rstd = L.rms_norm(x, w, r)
    dx, dw = L.rms_norm_backward(total, w, rstd, dy, dt)
    st = torch.cuda.current_stream().cuda_stream
    d = capi.rms_norm_desc(9, D, capi.MFT_BF16)
    for swap in (False, True):
        x2, r2, rs = x.clone(), r.clone(), torch.empty_like(rstd)
        to = (x2, r2) if swap else (r2, x2)  # total's place, y's place
        capi.rms_norm_fwd(d, x2.data_ptr(), r2.data_ptr(), w.data_ptr(), to[0].data_ptr(), to[1].data_ptr(),
                          rs.data_ptr(), st)
        assert torch.equal(to[0], total) and torch.equal(to[1], y) and torch.equal(rs, rstd)
    ws = torch.empty(capi.rms_norm_workspace_size(d), dtype=torch.uint8, device=dev)
    for which in (0, 1):
        g = [dy.clone(), dt.clone()]
        w2 = torch.empty_like(w)
        capi.rms_norm_bwd(d, total.data_ptr(), w.data_ptr(), rstd.data_ptr(), g[0].data_ptr(), g[1].data_ptr(),
                          g[which].data_ptr(), w2.data_ptr(), ws.data_ptr(), st)
        assert torch.equal(g[which], dx) and torch.equal(w2, dw)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the last rows' results are those of a call of their own."""
    from mobilefinetuner_amd import rms_norm as L
    N, D = (1 << 20) + 300, 2056
    x = torch.zeros(N, D, dtype=torch.bfloat16, device=dev)
    last, _, w, dy, _ = (t.to(dev) for t in make(5, D, "bf16", 14))
    x[-5:] = last
    y, total, rstd = L.rms_norm(x, w, x)
    ref = L.rms_norm(last, w, last)
    assert all(torch.equal(p[-5:], q) for p, q in zip((y, total, rstd), ref)) and (y[:5] == 0).all()
    del y
    q, scale, _ = L.rms_norm_e4m3(x, w)
    q2, scale2, _ = L.rms_norm_e4m3(last, w)
    assert torch.equal(q[-5:].float(), q2.float()) and torch.equal(scale[-5:], scale2)
    del q
    x.zero_()  # as dy, but for the last rows
    x[-5:] = dy
    dx, dw = L.rms_norm_backward(total, w, rstd, x, x)
    assert torch.equal(dx[-5:], L.rms_norm_backward(ref[1], w, ref[2], dy, dy)[0]) and (dx[:5] == 0).all()
    del x, dx, total


@pytest.mark.gpu
@pytest.mark.parametrize("N,D", [((1 << 25) + 70, 8), ((1 << 21) + 3, 16400)])
def test_more_rows_than_a_launch_takes(dev, N, D):
    """Rows held by a wave, by sixteen, and their last ones as in a call of their own."""
    from mobilefinetuner_amd import rms_norm as L
    x = torch.zeros(N, D, dtype=torch.bfloat16, device=dev)
    last, _, w, dy, _ = (t.to(dev) for t in make(5, D, "bf16", 15))
    x[-5:] = last
    q, scale, _ = L.rms_norm_e4m3(x, w)
    assert all(torch.equal(p[-5:].float(), r.float()) for p, r in zip((q, scale), L.rms_norm_e4m3(last, w)))
    assert (scale[:-5] == 2.0 ** -126).all()
    del q
    y, _, rstd = L.rms_norm(x, w)
    ref = L.rms_norm(last, w)
    assert torch.equal(y[-5:], ref[0]) and torch.equal(rstd[-5:], ref[2]) and (rstd[:-5] == rstd[0]).all()
    if D > 16384:  # beyond the backward's registers
        y.zero_()
        y[-5:] = dy
        dx = L.rms_norm_backward(x, w, rstd, y, want_weight=False)[0]
        assert torch.equal(dx[-5:], L.rms_norm_backward(last, w, ref[2], dy, want_weight=False)[0])
        del dx
    del x, y


@pytest.mark.gpu
@pytest.mark.parametrize("D", [(1 << 26) - 8, (1 << 26) + 4099])
def test_wider_rows_than_a_launch_takes(dev, D):
    """The weight's gradient on either side of a launch's columns.  Multiples of 1/2 whose products with
    rstd of 1/2 and 2 are exact, and so are the sums of two rows."""
    from mobilefinetuner_amd import rms_norm as L
    print(f"[case] D {D}", flush=True)
    j = torch.arange(D, device=dev)
    x = torch.stack([j % 13 - 6, j % 7 - 3]).bfloat16()
    dy = torch.stack([j % 5 - 2, j % 11 - 5]).bfloat16()
    rstd = torch.tensor([0.5, 2.0], device=dev)
    _, dw = L.rms_norm_backward(x, None, rstd, dy, want_x=False)
    assert torch.equal(dw, (dy.float() * (x.float() * rstd[:, None])).sum(0))
    del x, dy, dw, j


@pytest.mark.gpu
@pytest.mark.parametrize("D", [257, 4097, 70000])
def test_values_that_are_not_numbers_stay_in_their_row(dev, D):
    """A NaN makes its row NaN; an infinity makes rstd 0, so itself NaN and the rest of its row 0.  In 8 bits
    both have no numbers, and neither has a row whose sum of squares overflows (0)."""
    from mobilefinetuner_amd import rms_norm as L
    x, _, w, _, _ = (t.to(dev) for t in make(8, D, "f32", 7))
    clean, clean8 = L.rms_norm(x, w)[0], L.rms_norm_e4m3(x, w)
    x2 = x.clone()
    x2[2, 100], x2[5, 256], x2[6, 0] = math.nan, math.inf, -math.inf
    keep = [0, 1, 3, 4, 7]
    y, _, rstd = L.rms_norm(x2, w)
    assert torch.isnan(y[2]).all() and (rstd[[5, 6]] == 0).all() and torch.isnan(y[5, 256]) and torch.isnan(y[6, 0])
    assert (y[5, :256] == 0).all() and (y[6, 1:] == 0).all() and torch.equal(y[keep], clean[keep])
    q, scale, _ = L.rms_norm_e4m3(x2, w)
    assert torch.isnan(scale[[2, 5, 6]]).all() and torch.isnan(q.float()[[2, 5, 6]]).all()
    assert torch.equal(q.float()[keep], clean8[0].float()[keep]) and torch.equal(scale[keep], clean8[1][keep])
    q, scale = L.quantize_rows(x2)
    assert torch.isnan(scale[2]) and torch.isinf(scale[[5, 6]]).all() and torch.isnan(q.float()[2]).all()
    assert torch.isnan(q.float()[5, 256]) and (q.float()[5, :256] == 0).all()
    zero, _, rstd = L.rms_norm(torch.zeros(2, D, device=dev), w, eps=0.25)
    assert (zero == 0).all() and (rstd == 2.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norm", NORMS)
def test_autograd_gradients_against_differences(dev, dtype, norm):
    """The nodes' gradients are the helpers', and (fp32) those of differences: the loss sum(y c) + sum(total e)
    moves by the gradient along a direction v, to the second order of the step (t^2 times a third
    derivative of order one) and the loss's rounding over the step."""
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, c, e = (t.to(dev) for t in make(6, 130, dtype, 8))
    x, r, w = (t.clone().requires_grad_(True) for t in (x, r, w))
    y, total = L.AddRMSNorm.apply(x, r, w, norm, 1e-6)
    torch.autograd.backward([y, total], [c, e])
    _, s, rstd = L.rms_norm(x.detach(), w.detach(), r.detach(), norm)
    dx, dw = L.rms_norm_backward(s, w.detach(), rstd, c, e, norm)
    assert torch.equal(total, s) and torch.equal(x.grad, dx) and torch.equal(r.grad, dx) and torch.equal(w.grad, dw)
    assert x.grad.data_ptr() != r.grad.data_ptr()
    x3 = x.detach().clone().requires_grad_(True)
    L.RMSNorm.apply(x3, w.detach(), norm, 1e-6).backward(c)
    _, _, rs = L.rms_norm(x3.detach(), w.detach(), None, norm)
    assert torch.equal(x3.grad, L.rms_norm_backward(x3.detach(), w.detach(), rs, c, None, norm)[0])
    only = x.detach().clone().requires_grad_(True)  # the norm's output is not used
    L.AddRMSNorm.apply(only, r.detach(), w, norm, 1e-6)[1].backward(e)
    assert torch.equal(only.grad, e)
    if dtype == "bf16":
        return
    g = torch.Generator().manual_seed(1)
    t = 2.0 ** -7
    for p in (x, r, w):
        v = torch.randn(p.shape, generator=g).to(dev)
        loss = []
        with torch.no_grad():
            for k in (t, -t):
                q = [u + k * v if u is p else u for u in (x, r, w)]
                yy, tt, _ = L.rms_norm(q[0], q[2], q[1], norm)
                loss.append(float((yy.double() * c.double()).sum() + (tt.double() * e.double()).sum()))
        slope = (loss[0] - loss[1]) / (2 * t)
        scale = float((c.double().norm() + e.double().norm()) * v.double().norm())
        assert abs(slope - float((p.grad.double() * v.double()).sum())) <= scale * (4 * t * t + 256 * U / t)


@pytest.mark.gpu
def test_repeated_calls_and_streams(dev):
    """The same bits from every call, also from two streams at once, each with its own workspace."""
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = (t.to(dev) for t in make(3000, 768, "bf16", 9))
    _, total, rstd = L.rms_norm(x, w, r)
    ref = L.rms_norm_backward(total, w, rstd, dy, dt)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(L.rms_norm_backward(total, w, rstd, dy, dt))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, ref))


@pytest.mark.gpu
def test_captured_graph_follows_its_inputs(dev):
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = (t.to(dev) for t in make(500, 640, "bf16", 10))

    def step():
        y, total, rstd = L.rms_norm(x, w, r)
        q, scale, _ = L.rms_norm_e4m3(x, w, r)
        return [y, total, rstd, q, scale, *L.rms_norm_backward(total, w, rstd, dy, dt)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (11, 12, 13):
        for t, n in zip((x, r, dy, dt), [v for i, v in enumerate(make(500, 640, "bf16", seed)) if i != 2]):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(held, step()))


@pytest.mark.gpu
def test_one_row_broadcast_rows_and_a_stream_added_to_itself(dev):
    """x without leading dimensions, gradients of broadcast x, and x as its own residual: as by rows, by a
    product of a copy, and twice one gradient."""
    from mobilefinetuner_amd import rms_norm as L
    x, r, w, dy, dt = (t.to(dev) for t in make(5, 96, "f32", 16))
    rows, one = L.rms_norm(x, w, r), L.rms_norm(x[3], w, r[3])
    assert one[2].shape == () and all(torch.equal(p[3], q) for p, q in zip(rows, one))
    q, scale = L.quantize_rows(x[3])
    assert q.shape == (96,) and scale.shape == () and torch.equal(q.float(), L.quantize_rows(x)[0][3].float())
    dx, _ = L.rms_norm_backward(one[1], w, one[2], dy[3], dt[3])
    assert torch.equal(dx, L.rms_norm_backward(rows[1], w, rows[2], dy, dt, want_weight=False)[0][3])
    b = x[:1].clone().requires_grad_(True)
    y, total = L.AddRMSNorm.apply(b.expand(5, 96), r, w)
    torch.autograd.backward([y, total], [dy, dt])
    c = x[:1].expand(5, 96).clone().requires_grad_(True)
    y, total = L.AddRMSNorm.apply(c, r, w)
    torch.autograd.backward([y, total], [dy, dt])
    assert torch.equal(b.grad, c.grad.sum(0, keepdim=True))
    s = x.clone().requires_grad_(True)
    y, total = L.AddRMSNorm.apply(s, s, w)
    torch.autograd.backward([y, total], [dy, dt])
    _, total, rstd = L.rms_norm(x, w, x)
    assert torch.equal(s.grad, 2 * L.rms_norm_backward(total, w, rstd, dy, dt)[0])


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


@pytest.mark.parametrize("change,message", [
    (dict(N=-1), "N >= 0"), (dict(N=1 << 31), "below"), (dict(D=0), "D > 0"), (dict(D=(1 << 30) + 1), "at most"),
    (dict(dtype=1), "dtype"), (dict(norm=3), "norm"), (dict(norm=-1), "norm"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(x_stride=63), "stride"),
    (dict(residual_stride=1), "stride"), (dict(dy_stride=-64), "stride"), (dict(dtotal_stride=63), "stride"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.rms_norm_desc(**{**dict(N=4, D=64), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.rms_norm_fwd(d, 16, None, None, None, 32, None, None)
    with pytest.raises(capi.MftError, match=message):
        capi.rms_norm_e4m3_fwd(d, 16, None, None, None, 32, 48, None)
    with pytest.raises(capi.MftError, match=message):
        capi.rms_norm_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.rms_norm_bwd(d, 16, None, 16, 16, None, 32, None, 64, None)


def test_operands_refused(capi):
    d, none = capi.rms_norm_desc(4, 64), capi.rms_norm_desc(4, 64, norm=capi.MFT_NORM_NONE)
    for call, message in (
            (lambda: capi.rms_norm_fwd(d, None, None, None, None, 32, None, None), "non-NULL"),
            (lambda: capi.rms_norm_fwd(d, 16, None, None, None, None, None, None), "non-NULL"),
            (lambda: capi.rms_norm_fwd(d, 16, 32, None, None, 48, None, None), "together"),
            (lambda: capi.rms_norm_fwd(d, 16, None, None, 32, 48, None, None), "together"),
            (lambda: capi.rms_norm_fwd(d, 16, 32, None, 48, 48, None, None), "may not be total"),
            (lambda: capi.rms_norm_fwd(none, 16, None, None, None, 48, None, None), "norm must be"),
            (lambda: capi.rms_norm_e4m3_fwd(d, 16, None, None, None, 48, None, None), "scale"),
            (lambda: capi.rms_norm_e4m3_fwd(d, 16, None, None, None, 16, 64, None), "may not be x"),
            (lambda: capi.rms_norm_e4m3_fwd(d, 16, 48, None, 80, 48, 64, None), "may not be x or residual"),
            (lambda: capi.rms_norm_e4m3_fwd(none, 16, None, 80, None, 48, 64, None), "no weight"),
            (lambda: capi.rms_norm_bwd(d, 16, None, 32, 48, None, 16, None, 64, None), "may not be x")):
        with pytest.raises(capi.MftError, match=message):
            call()
    good = [16, None, 32, 48, None, 80, None, 96]
    for i in (0, 2, 3, 7):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.rms_norm_bwd(d, *[None if j == i else a for j, a in enumerate(good)], None)
    assert capi.lib().mft_rms_norm_fwd(None, 16, None, None, None, 32, None, None) == capi.MFT_ERR_INVALID_ARG
    empty = C.byref(capi.rms_norm_desc(0, 64))
    assert capi.lib().mft_rms_norm_fwd(empty, None, None, None, None, None, None, None) == capi.MFT_OK
    assert capi.lib().mft_rms_norm_e4m3_fwd(empty, None, None, None, None, None, None, None) == capi.MFT_OK


def test_in_place_with_other_strides_refused(capi):
    """Rows would be overwritten before they are read."""
    for d, args in ((capi.rms_norm_desc(4, 64, x_stride=80), (16, None, None, None, 16)),
                    (capi.rms_norm_desc(4, 64, residual_stride=80), (16, 32, None, 48, 32)),
                    (capi.rms_norm_desc(4, 64, total_stride=80), (16, 32, None, 32, 48)),
                    (capi.rms_norm_desc(4, 64, total_stride=80), (16, 32, None, 16, 48))):
        with pytest.raises(capi.MftError, match="in place"):
            capi.rms_norm_fwd(d, *args, None, None)
    for g, t, dx in ((48, None, 48), (48, 64, 64)):
        with pytest.raises(capi.MftError, match="in place"):
            capi.rms_norm_bwd(capi.rms_norm_desc(4, 64, dx_stride=80), 16, None, 32, g, t, dx, None, 96, None)


def test_no_cpu_path():
    from mobilefinetuner_amd import rms_norm as L
    for f in (L.rms_norm, L.rms_norm_e4m3, L.quantize_rows):
        with pytest.raises(ValueError, match="no CPU path"):
            f(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="norm must be"):
        L.rms_norm(torch.zeros(2, 4), norm="layer")


@pytest.mark.gpu
def test_operands_that_do_not_fit_refused(dev):
    from mobilefinetuner_amd import rms_norm as L
    x, w = torch.zeros(2, 8, device=dev), torch.ones(8, device=dev)
    s = torch.zeros(2, device=dev)
    for bad in (lambda: L.rms_norm(x, w[:7]), lambda: L.rms_norm(x, w.bfloat16()), lambda: L.rms_norm(x, w.cpu()),
                lambda: L.rms_norm(x.half()), lambda: L.rms_norm(x[:, :0]), lambda: L.rms_norm(x, w, x[:1]),
                lambda: L.rms_norm(x, w, x.bfloat16()), lambda: L.rms_norm(x, w, norm="none"),
                lambda: L.quantize_rows(x.half()), lambda: L.rms_norm_backward(x, w, s[:1], x),
                lambda: L.rms_norm_backward(x, w, s, x.bfloat16()), lambda: L.rms_norm_backward(x, w, s, x[:1]),
                lambda: L.rms_norm_backward(x, w, s, x, x[:1])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 1152, 1153, 4100, 20000, 70000])
def test_eight_bits_are_those_of_the_quotient(dev, D, dtype):
    """To the bit, scale = max (1 / 448) and q = e4m3(x / scale), all in fp32: the quotients of bf16 rows often lie
    halfway between two numbers, where one by a reciprocal comes out on the other side.  From the smallest
    scales to the largest; a kernel for each count of waves, and one by memory.  torch's own operations on the GPU
    give the same."""
    from mobilefinetuner_amd import rms_norm as L
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(max(7, 400000 // D), D, generator=g) * 2.0 ** -7).to(DT[dtype])
    for i, e in enumerate((-118, -100, 60, 126)):
        x[i] = (x[i].float().clamp(-0.03, 0.03) * 2.0 ** e).to(DT[dtype])
    print(f"[case] {list(x.shape)} {dtype}", flush=True)
    q, scale = L.quantize_rows(x.to(dev))
    up = x.float()
    want = (up.abs().amax(1) * (torch.tensor(1.0) / 448)).clamp(min=2.0 ** -126)
    assert torch.equal(scale.cpu(), want)
    assert torch.equal(q.float().cpu(), (up / want[:, None]).to(torch.float8_e4m3fn).float())
    own = (up.to(dev).abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
    assert torch.equal(own, scale) and torch.equal((up.to(dev) / own[:, None]).to(torch.float8_e4m3fn).float(), q.float())
