"""Token log probabilities, entropy, alternatives and the gradient (mft_logprobs_*
through the torch helpers) against their formulas in 64 bits, and refusals.

Bounds, with u = 2^-24, d = z - max and K = V / 256 + 80, the longest chain of
fp32 additions of a row's sums (a thread's share, its unaligned ends, the tree).
d is off by u |d|, exp(d) by (3 |d| + 4) u of itself (the rounded argument of the
power of two, the instruction), so S by (K + 4 + 3 E|d|) u of itself, where E is
the mean over p; log S by that much and its own rounding; T = S E[d] by
u S ((K + 6) E|d| + 3 E d^2).  A part's sums, moved to the row's maximum, add a
rounding each (in K).  The gradient takes the statistics as given:
q = (z - max) - log S is off by u (|z - max| + |q|), p by u (3 |q| + |z - max| + 6)
of itself.  Alternatives are compared exactly.
"""
import ctypes as C
import math

import pytest
import torch

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100


def make(N, V, dtype, seed, sigma=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (sigma * torch.randn(N, V, generator=g)).to(DT[dtype])
    return z, torch.randint(0, V, (N,), generator=g, dtype=torch.int32), torch.randn(N, generator=g), \
        torch.randn(N, generator=g)


def ref_forward(z, t, top):
    zd = z.double()
    V = z.shape[-1]
    m = zd.max(-1, keepdim=True).values
    d = zd - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    p = e / s
    dd = torch.where(p > 0, d, torch.zeros_like(d))
    e1, e2 = (p * -dd).sum(-1), (p * dd * dd).sum(-1)
    log_s = torch.log(s)[..., 0]
    k = V / 256 + 80
    s_err = U * (k + 4 + 3 * e1 + 2 * log_s.abs())
    dt = d.gather(-1, t.long().clamp(0, V - 1)[:, None])[:, 0]
    out = {"logprob": (dt - log_s, s_err + U * (dt.abs() + 2 * (dt - log_s).abs())),
           "entropy": (log_s + e1, s_err * (1 + e1) + U * ((k + 8) * e1 + 3 * e2 + 2 * (log_s + e1).abs()) + 1e-300)}
    if top:
        ids = torch.sort(zd, dim=-1, descending=True, stable=True).indices[:, :top]
        best = d.gather(-1, ids) - log_s[:, None]
        out["top"] = (best, s_err[:, None] + U * (d.gather(-1, ids).abs() + 2 * best.abs()))
        out["ids"] = ids.int()
    return out


def ref_backward(z, t, stats, entropy, gl, ge):
    zd, st = z.double(), stats.double()
    d = zd - st[:, :1]
    q = d - st[:, 1:]
    p = torch.exp(q)
    live = p > 0
    q0, d0 = torch.where(live, q, torch.zeros_like(q)), torch.where(live, d, torch.zeros_like(d))
    glc, gec, h = gl.double()[:, None], ge.double()[:, None], entropy.double()[:, None]
    g = -p * (glc + gec * (q0 + h))
    size = p * (glc.abs() + gec.abs() * (q0.abs() + h))
    g.scatter_add_(1, t.long()[:, None], glc)
    tol = U * size * (3 * q0.abs() + d0.abs() + 10)
    tol.scatter_add_(1, t.long()[:, None], U * glc.abs())
    # probabilities under the smallest normal number may be flushed
    return g, tol + torch.finfo(z.dtype).eps / 2 * g.abs() + 1e-36


def within(got, ref, tol):
    off = (got.detach().cpu().double() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def check_forward(z, t, top, dev):
    from mobilefinetuner_amd import logprobs as L
    lp, ent, stats, best, ids = L.token_logprobs(z.to(dev), t.to(dev), top)
    ref = ref_forward(z, t, top)
    within(lp, *ref["logprob"])
    within(ent, *ref["entropy"])
    if top:
        assert torch.equal(ids.cpu(), ref["ids"])
        within(best, *ref["top"])
    return stats, ent


# below a vector, off the vectors, one part and several, more parts than fill the last
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 64), (7, 255), (4, 1000), (3, 4097), (2, 8200), (1, 50257), (2, 131073),
          (1, 262144), (1, 300001), (1100, 333), (1030, 8193)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_forward_and_backward(dev, N, V, dtype):
    from mobilefinetuner_amd import logprobs as L
    print(f"[case] {N} x {V} {dtype}", flush=True)
    z, t, gl, ge = make(N, V, dtype, N + V)
    for top in sorted({0, min(5, V), min(20, V), min(64, V)}):
        stats, ent = check_forward(z, t, top, dev)
    g = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev))
    assert g.dtype == z.dtype
    within(g, *ref_backward(z, t, stats.cpu(), ent.cpu(), gl, ge))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 2048, 20000, 140000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few values", "one thread's", "clusters", "zeros"])
def test_alternatives_of_hard_rows(dev, V, kind):
    """Ties by the hundred thousand, orders in which every element is a new maximum, and rows whose
    largest elements all fall to one thread of the workgroup."""
    g = torch.Generator().manual_seed(V)
    j = torch.arange(V)
    z = {"equal": torch.zeros(V), "rising": j.float() / V, "falling": -j.float() / V,
         "few values": torch.randint(0, 3, (V,), generator=g).float(),
         "one thread's": torch.where(j % 1024 < 4, 5.0 + (j % 97) / 97.0, -j.float() / V),
         "clusters": torch.randn(V, generator=g) + 6.0 * ((j // 40) % 50 == 7),
         "zeros": torch.where(j % 2 == 0, torch.tensor(0.0), torch.tensor(-0.0))}[kind]
    print(f"[case] {kind} {V}", flush=True)
    for dtype in DT:
        zz = z.to(DT[dtype])[None].repeat(2, 1)
        t = torch.tensor([0, V - 1], dtype=torch.int32)
        for top in (1, 20, min(64, V)):
            check_forward(zz, t, top, dev)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 5000, 70000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_excluded_logits(dev, V, dtype):
    """Rows with few entries above -inf: those come first, then -inf ones by index; gradients of
    excluded entries are exactly 0."""
    from mobilefinetuner_amd import logprobs as L
    z, t, gl, ge = make(3, V, dtype, V)
    z[0, 10:], z[1, ::2], z[2, 1:] = -math.inf, -math.inf, -math.inf
    t = torch.tensor([3, 1, 0], dtype=torch.int32)
    stats, ent = check_forward(z, t, 0, dev)
    lp, _, _, best, ids = L.token_logprobs(z.to(dev), t.to(dev), 20)
    order = torch.sort(z.double(), dim=-1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(ids.cpu(), order.int())
    assert torch.equal(best.cpu() == -math.inf, z.gather(1, order) == -math.inf)
    assert lp[2].item() == 0.0 and ent[2].item() == 0.0
    g = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev)).cpu()
    assert (g[z == -math.inf] == 0).all()
    within(g, *ref_backward(z, t, stats.cpu(), ent.cpu(), gl, ge))
    # a given token that is excluded
    lp = L.token_logprobs(z.to(dev), torch.tensor([50, 0, 1], dtype=torch.int32, device=dev))[0]
    assert (lp == -math.inf).all()


# one workgroup to a row below 8192, or with more rows than half the workgroups; parts of one else
@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(6, 300), (6, 5000), (6, 70001), (1030, 9000), (6, 262144)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lowest", ["finfo.min", -1e38, -1e35, -1e30])
def test_logits_excluded_by_a_finite_value(dev, lowest, dtype, N, V):
    """Their probability is 0, and they add nothing to the entropy or the gradient, whoever meets them first
    or alone: a thread, a wave, a part."""
    from mobilefinetuner_amd import logprobs as L
    print(f"[case] {N} x {V} {dtype} {lowest}", flush=True)
    low = torch.finfo(DT[dtype]).min if lowest == "finfo.min" else lowest
    z, t, gl, ge = make(N, V, dtype, V)
    live = torch.zeros(6, V, dtype=torch.bool)
    live[0, V // 2] = True                            # one value, of one thread
    live[1, :10] = True                               # the first ones
    live[2, -(V // 3):] = True                        # behind what is masked
    live[3, ::7] = True                               # in every vector
    live[4] = torch.arange(V) // 8 % 256 >= 128       # of every other wave or two; none of 300
    live[5] = torch.arange(V) // 1024 % 2 == 1        # rounds of vectors
    live[5, -1] = True
    live = live.repeat(N // 6 + 1, 1)[:N]
    z[~live] = low
    t = torch.where(torch.arange(N) % 2 == 0, live.int().argmax(1), t.long()).int()
    stats, ent = check_forward(z, t, min(20, V), dev)
    assert torch.isfinite(ent).all() and (ent[0::6] == 0).all()
    g = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev)).cpu()
    within(g, *ref_backward(z, t, stats.cpu(), ent.cpu(), gl, ge))
    some = live.any(1)  # row 4 of 300 has nothing else: the uniform distribution
    masked = ~live & some[:, None]
    masked.scatter_(1, t.long()[:, None], False)
    assert (g[masked] == 0).all()
    # the sums are those of a row with -inf in their place
    z[~live] = -math.inf
    _, e2, s2, _, _ = L.token_logprobs(z.to(dev), t.to(dev))
    assert torch.equal(s2[some], stats[some]) and torch.equal(e2[some], ent[some])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 70001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("large", [1e9, 1e20, 1e30])
def test_large_entropy_gradients_of_excluded_logits(dev, large, dtype, V):
    """A probability of 0 adds nothing however large the entropy's gradient is; one that is lost below
    2^-126 is a logit at most 104 under the largest."""
    from mobilefinetuner_amd import logprobs as L
    print(f"[case] {large} {dtype} {V}", flush=True)
    z, t, gl, ge = make(4, V, dtype, V)
    ge = large * torch.tensor([1.0, -1.0, 0.5, -0.3])
    z[0, ::3], z[1, ::3], z[2, 5:] = -math.inf, torch.finfo(DT[dtype]).min, -200.0
    t = torch.tensor([1, 0, 7, V - 1], dtype=torch.int32)  # row 1's and 2's are excluded ones
    _, ent, stats, _, _ = L.token_logprobs(z.to(dev), t.to(dev))
    g = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev)).cpu()
    ref, tol = ref_backward(z, t, stats.cpu(), ent.cpu(), gl, ge)
    lost = 2.0 ** -126 * (gl.abs() + ge.abs() * (104 + ent.cpu()))
    within(g, ref, tol + lost.double()[:, None])
    assert g[1, 0] == gl[1].to(z.dtype) and g[2, 7] == gl[2].to(z.dtype)
    assert (g[0, ::3] == 0).all() and (g[1, 3::3] == 0).all() and (g[2, 8:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000, 60000])
def test_rows_without_a_distribution(dev, V):
    """Nothing but -inf, a NaN, +inf: NaN in that row alone; alternatives are its numbers."""
    from mobilefinetuner_amd import logprobs as L
    z, t, _, _ = make(6, V, "f32", V)
    clean = [x.clone() for x in L.token_logprobs(z.to(dev), t.to(dev), 4)]
    z[1], z[3, V // 2], z[4, 7], z[5, 3:] = -math.inf, math.nan, math.inf, math.nan
    lp, ent, _, best, ids = L.token_logprobs(z.to(dev), t.to(dev), 4)
    bad = [1, 3, 4, 5]
    assert torch.isnan(lp[[1, 3]]).all() and torch.isnan(ent[bad]).all() and torch.isnan(best[[1, 3, 5]]).all()
    for row in (0, 2):
        assert lp[row] == clean[0][row] and ent[row] == clean[1][row] and torch.equal(ids[row], clean[4][row])
    assert ids[1].tolist() == [0, 1, 2, 3]
    numbers = torch.where(torch.isnan(z), torch.tensor(-math.inf), z)
    assert ids[3].tolist() == torch.sort(numbers[3], descending=True, stable=True).indices[:4].tolist()
    assert ids[4, 0].item() == 7
    first = torch.sort(z[5, :3], descending=True, stable=True).indices.tolist()
    assert ids[5].tolist() == first + [-1]


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(9, 700), (3, 20000), (2000, 100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ignored_rows_are_not_read_and_tokens_out_of_range(dev, N, V, dtype):
    from mobilefinetuner_amd import logprobs as L
    z, t, gl, ge = make(N, V, dtype, N)
    t[1] = IGNORE
    z[1] = math.nan
    lp, ent, stats, best, ids = L.token_logprobs(z.to(dev), t.to(dev), 3)
    assert lp[1] == 0 and ent[1] == 0 and (stats[1] == 0).all() and (best[1] == -math.inf).all() and (ids[1] == -1).all()
    g = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev))
    assert (g[1] == 0).all() and torch.isfinite(g).all()
    for wrong in (V, -1, 2 ** 31 - 1):
        t[0] = wrong
        with pytest.raises(ValueError, match="out of range"):
            L.token_logprobs(z.to(dev), t.to(dev), 3)
        lp2, ent2, _, best2, ids2 = L.token_logprobs(z.to(dev), t.to(dev), 3, check_tokens=False)
        assert torch.isnan(lp2[0]) and ent2[0] == ent[0] and torch.equal(ids2, ids) and torch.equal(best2, best)
        assert torch.equal(lp2[2:], lp[2:])
        g2 = L.token_logprobs_backward(z.to(dev), t.to(dev), stats, ent, gl.to(dev), ge.to(dev))
        assert (g2[0] == 0).all() and torch.equal(g2[2:], g[2:])
    # another index to ignore; -100 is then out of range
    t[0], t[1] = 7, 7
    lp3 = L.token_logprobs(z.to(dev), t.to(dev), ignore_index=7)[0]
    assert lp3[0] == 0 and lp3[1] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shapes_and_strides(dev, dtype):
    """[B, S, V], a single row, a vocabulary padded to a wider row, a transposed batch, no row."""
    from mobilefinetuner_amd import logprobs as L
    z, t, gl, ge = (x.to(dev) for x in make(12, 1003, dtype, 1))
    views = [(z[:, :1001], t % 1001), (z.view(3, 4, 1003), t.view(3, 4)), (z[0], t[0]), (z[:, 1:1000], t % 999),
             (z.view(3, 4, 1003).transpose(0, 1), t.view(3, 4).t()), (z[:, ::2], t % 502), (z[:0], t[:0]),
             (z[3:4, :900].expand(5, 900), t[:5] % 900)]
    for v, tt in views:
        c, tc = v.contiguous(), tt.contiguous()
        got, ref = L.token_logprobs(v, tt, 5), L.token_logprobs(c, tc, 5)
        assert got[0].shape == tt.shape and got[2].shape == (*tt.shape, 2) and got[3].shape == (*tt.shape, 5)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
        a = torch.ones(tt.shape, device=dev)
        g = L.token_logprobs_backward(v, tt, got[2], got[1], a, a)
        assert g.shape == v.shape and torch.equal(g, L.token_logprobs_backward(c, tc, got[2], got[1], a, a))
        g = L.token_logprobs_backward(v, tt, got[2], None, a)
        assert torch.equal(g, L.token_logprobs_backward(v, tt, got[2], got[1], a, torch.zeros_like(a)))


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A row that starts past 2^32 bytes and 2^31 elements: its results are those of a copy."""
    from mobilefinetuner_amd import logprobs as L
    V, N = 262144, 8200
    z = torch.empty(N, V, dtype=torch.bfloat16, device=dev)  # 4.3 GB
    t = torch.full((N,), IGNORE, dtype=torch.int32, device=dev)
    z[-2:] = make(2, V, "bf16", 3)[0].to(dev)
    t[-2:] = torch.tensor([5, V - 1], dtype=torch.int32, device=dev)
    got, ref = L.token_logprobs(z, t, 8), L.token_logprobs(z[-2:].clone(), t[-2:], 8)
    assert torch.equal(got[4][-2:], ref[4])
    # the two were cut into other parts: their sums differ in the order of additions
    for p, q in zip(got[:2], ref[:2]):
        assert torch.allclose(p[-2:], q, rtol=0, atol=1e-5)
    assert (got[0][:-2] == 0).all()
    del z


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd_gradients_against_differences(dev, dtype):
    from mobilefinetuner_amd import logprobs as L
    z, t, gl, ge = (x.to(dev) for x in make(5, 200, dtype, 2, 1.0))
    t[2] = IGNORE
    z.requires_grad_(True)
    lp, ent = L.TokenLogprobs.apply(z, t)
    ((lp * gl).sum() + (ent * ge).sum()).backward()
    _, e, stats, _, _ = L.token_logprobs(z.detach(), t)
    assert torch.equal(z.grad, L.token_logprobs_backward(z.detach(), t, stats, e, gl, ge))
    only = torch.autograd.grad(L.TokenLogprobs.apply(z, t)[0].sum(), z)[0]
    assert torch.equal(only, L.token_logprobs_backward(z.detach(), t, stats, e, torch.ones_like(gl)))
    only = torch.autograd.grad(L.TokenLogprobs.apply(z, t)[1].sum(), z)[0]
    assert torch.equal(only, L.token_logprobs_backward(z.detach(), t, stats, e, None, torch.ones_like(gl)))
    if dtype == "bf16":
        return
    # along a direction: second order of the step, and the losses' rounding over it
    v = torch.randn(z.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    step, loss = 2.0 ** -6, []
    for s in (step, -step):
        a, b, _, _, _ = L.token_logprobs(z.detach() + s * v, t)
        loss.append(float((a.double() * gl).sum() + (b.double() * ge).sum()))
    slope, along = (loss[0] - loss[1]) / (2 * step), float((z.grad.double() * v).sum())
    scale = float((gl.abs() + ge.abs()).sum())
    assert abs(slope - along) <= scale * (20 * step * step + 400 * U / step)


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(3, 50257), (40, 3001)])
def test_captured_graph_and_streams(dev, N, V):
    from mobilefinetuner_amd import logprobs as L
    z, t, gl, ge = (x.to(dev) for x in make(N, V, "bf16", 5))

    def step():
        lp, ent, stats, best, ids = L.token_logprobs(z, t, 10, check_tokens=False)
        return lp, ent, best, ids, L.token_logprobs_backward(z, t, stats, ent, gl, ge)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (6, 7, 8):
        nz, nt, _, _ = make(N, V, "bf16", seed)
        z.copy_(nz)
        t.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
    ref = [x.clone() for x in step()]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(p, q) for p, q in zip(r, ref))


@pytest.mark.gpu
def test_the_most_rows(dev):
    """2^24 - 1 rows: the last ones as in a call of their own."""
    from mobilefinetuner_amd import logprobs as L
    N = (1 << 24) - 1
    z = torch.zeros(N, 3, dtype=torch.bfloat16, device=dev)
    z[-5:] = torch.randn(5, 3, generator=torch.Generator().manual_seed(5)).to(dev)
    t = torch.ones(N, dtype=torch.int32, device=dev)
    got, ref = L.token_logprobs(z, t, 2), L.token_logprobs(z[-5:], t[-5:], 2)
    assert all(torch.equal(p[-5:], q) for p, q in zip(got, ref))
    one = torch.ones(N, device=dev)
    g = L.token_logprobs_backward(z, t, got[2], got[1], one)
    assert torch.equal(g[-5:], L.token_logprobs_backward(z[-5:], t[-5:], ref[2], ref[1], one[-5:]))


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


@pytest.mark.parametrize("change,message", [
    (dict(N=-1), "N >= 0"), (dict(V=0), "V > 0"), (dict(N=(1 << 24) + 1), "2\\^24"), (dict(N=1 << 24), "2\\^24"), (dict(V=(1 << 30) + 1), "2\\^30"),
    (dict(dtype=1), "dtype"), (dict(top=-1), "top"), (dict(top=65), "top"), (dict(V=10, top=11), "top"),
    (dict(ld=99), "stride"), (dict(grad_ld=-100), "stride"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.logprobs_desc(**{**dict(N=4, V=100), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.logprobs_workspace_size(d)
    with pytest.raises(capi.MftError, match=message):
        capi.logprobs_fwd(d, 16, 32, 48, None, None, 64, 80, None, 96, None)
    with pytest.raises(capi.MftError, match=message):
        capi.logprobs_bwd(d, 16, 32, 48, None, 64, None, 80, None)


def test_null_operands_refused(capi):
    d = capi.logprobs_desc(4, 100, top=2)
    good = [16, 32, 48, None, None, 64, 80, None, 96]
    for i in (0, 1, 2, 5, 6):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.logprobs_fwd(d, *[None if j == i else a for j, a in enumerate(good)], None)
    cut = capi.logprobs_desc(1, 100000)
    assert capi.logprobs_workspace_size(cut) > 0
    with pytest.raises(capi.MftError, match="workspace"):
        capi.logprobs_fwd(cut, 16, 32, 48, None, None, None, None, None, None, None)
    good = [16, 32, 48, None, 64, None, 80]
    for i in (0, 1, 2, 6):
        with pytest.raises(capi.MftError, match="non-NULL"):
            capi.logprobs_bwd(d, *[None if j == i else a for j, a in enumerate(good)], None)
    with pytest.raises(capi.MftError, match="entropy"):
        capi.logprobs_bwd(d, 16, 32, 48, None, 64, 80, 96, None)
    with pytest.raises(capi.MftError, match="in place"):
        capi.logprobs_bwd(capi.logprobs_desc(4, 100, ld=104), 16, 32, 48, None, 64, None, 16, None)
    empty = capi.logprobs_desc(0, 100)
    assert capi.lib().mft_logprobs_fwd(C.byref(empty), *[None] * 10) == capi.MFT_OK


@pytest.mark.parametrize("wrong", [2 ** 32 - 100, 2 ** 31, -2 ** 31 - 1])
def test_an_ignore_index_beyond_the_tokens_type_refused(capi, wrong):
    """Its low 32 bits are another token's."""
    with pytest.raises(ValueError, match="int32"):
        capi.logprobs_desc(4, 100, ignore_index=wrong)
    for most in (2 ** 31 - 1, -2 ** 31):
        assert capi.logprobs_desc(4, 100, ignore_index=most).ignore_index == most


def test_no_cpu_path():
    from mobilefinetuner_amd import logprobs as L
    with pytest.raises(ValueError, match="no CPU path"):
        L.token_logprobs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int32))


@pytest.mark.gpu
def test_operands_that_do_not_fit_refused(dev):
    from mobilefinetuner_amd import logprobs as L
    z, t = torch.zeros(2, 8, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    s, e = torch.zeros(2, 2, device=dev), torch.zeros(2, device=dev)
    for bad in (lambda: L.token_logprobs(z, t.long()), lambda: L.token_logprobs(z, t[:1]),
                lambda: L.token_logprobs(z.half(), t), lambda: L.token_logprobs(z[:, :0], t),
                lambda: L.token_logprobs(z, t.cpu()), lambda: L.token_logprobs_backward(z, t, e, e, e),
                lambda: L.token_logprobs_backward(z, t, s, e, e.bfloat16())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="top"):
        L.token_logprobs(z, t, 9)
