"""The AdamW step (mft_adamw_* through AdamW) against its formula in 64 bits, and its refusals.

Bounds, per value, with u = 2^-24, from the state before the step as it is held:
m is a sum of two products of rounded factors (the clipped gradient has two
roundings of its own): 6 u of their magnitudes; v has the gradient's twice: 10 u.
The change step_size m / (root + eps) has m's error, and 16 u of itself from v, its
root, the factors and the division; p has 4 u of itself on top, and half a step of
its type.  In 8 bits x / scale is rounded by at most 2^-4 of itself, or half the
smallest number (2^-10), and a positive root by up to that number; before that the
state is as above, with one rounding more from its scale.
"""
import ctypes as C
import math

import pytest
import torch

U = 2.0 ** -24
BF16 = torch.finfo(torch.bfloat16).eps / 2
LR, BETAS, EPS = 3e-3, (0.9, 0.999), 1e-8


def make(sizes, kinds, seed, offset=0):
    """Parameters of the given sizes with gradients: "f32" or "bf16" each, `offset` values into their memory."""
    g = torch.Generator().manual_seed(seed)
    params = []
    for n, kind in zip(sizes, kinds):
        t = torch.float32 if kind == "f32" else torch.bfloat16
        data = torch.empty(n + offset, dtype=t, device="cuda")[offset:]
        data.copy_(torch.randn(n, generator=g) * 0.05)
        p = data.requires_grad_(True)
        grad = torch.empty(n + offset, dtype=t, device="cuda")[offset:]
        p.grad = grad.copy_(torch.randn(n, generator=g) * 10.0 ** torch.randint(-4, 1, (1,), generator=g).item())
        params.append(p)
    return params


def held(opt, name, i):
    """State `name` of parameter i in 64 bits: e4m3 numbers times their scales."""
    x = opt.views(name)[i].detach().cpu().double().reshape(-1)
    if opt.state_bits == 8:
        s = opt.views(name + "_scale")[i].cpu().double().repeat_interleave(256)[: x.numel()]
        return x * s
    return x


def snapshot(opt):
    out = []
    masters = opt.views("master") if "master" in opt.state else [None] * len(opt.params)
    for i, (p, w) in enumerate(zip(opt.params, masters)):
        v = held(opt, "exp_avg_sq", i)
        out.append(dict(p=(p if w is None else w).detach().cpu().double().reshape(-1), m=held(opt, "exp_avg", i),
                        v=v * v if opt.state_bits == 8 else v, g=None if p.grad is None else p.grad.cpu().double().reshape(-1)))
    return out


def within(got, ref, tol):
    off = (got - ref).abs()
    assert bool((off <= tol).all()), f"{float((off / tol).max()):.3g} times the bound"


def check(opt, before, t, max_norm, norm, lr=LR):
    """opt's state after step t against the formula from `before`."""
    on = [b["g"] for b in before if b["g"] is not None]
    clip = 1.0
    if max_norm is not None:
        ref = math.sqrt(sum(float((g * g).sum()) for g in on))
        assert abs(float(norm) - ref) <= (U + 1e-12) * ref
        clip = min(1.0, max_norm / (ref + 1e-6))
    b1, b2 = opt.betas
    after = snapshot(opt)
    for i, (old, new) in enumerate(zip(before, after)):
        if old["g"] is None:
            assert all(torch.equal(old[k], new[k]) for k in "pmv")
            continue
        g = clip * old["g"]
        m, v = b1 * old["m"] + (1 - b1) * g, b2 * old["v"] + (1 - b2) * g * g
        tm, tv = 7 * U * (b1 * old["m"].abs() + (1 - b1) * g.abs()) + 2.0 ** -148, 12 * U * v + 2.0 ** -148
        root = v.sqrt()
        under = root / math.sqrt(-math.expm1(t * math.log(b2))) + opt.eps
        size = lr / -math.expm1(t * math.log(b1)) if b1 > 0 else lr
        p = old["p"] * (1 - lr * opt.weight_decay[i]) - size * m / under
        within(new["p"], p, 4 * U * (old["p"].abs() + p.abs()) + size / under * (tm + 16 * U * m.abs()))
        if opt.params[i].dtype == torch.bfloat16:
            assert torch.equal(opt.params[i].detach().reshape(-1), opt.views("master")[i].reshape(-1).bfloat16())
        if opt.state_bits == 32:
            within(new["m"], m, tm)
            within(new["v"], v, tv)
            continue
        tr = 8 * U * root + 2.0 ** -74
        for name, x, tx, least in (("exp_avg", m, tm, 2.0 ** -10), ("exp_avg_sq", root, tr, 2.0 ** -9)):
            groups, off = (torch.nn.functional.pad(q, (0, -len(x) % 256)).view(-1, 256).abs().amax(1) for q in (x, tx))
            scale = (groups / 448).clamp(min=2.0 ** -126)
            # a group's largest value is off by its largest error at most: m may be a small difference
            within(opt.views(name + "_scale")[i].cpu().double(), scale, off / 448 + 4 * U * scale)
            s = scale.repeat_interleave(256)[: len(x)]
            within(held(opt, name, i), x, (2.0 ** -4 + 32 * U) * x.abs() + 1.1 * tx + least * 1.001 * s + off.repeat_interleave(256)[: len(x)] / 448)
        q = opt.views("exp_avg_sq")[i].detach().float().cpu().reshape(-1)
        assert bool((q[v > 2.0 ** -140] > 0).all()) and bool((q >= 0).all())


def run(params, steps=2, max_norm=None, bits=32, lr=LR, **more):
    from mobilefinetuner_amd.adamw import AdamW
    opt = AdamW(params, lr, BETAS, EPS, state_bits=bits, **more)
    for t in range(1, steps + 1):
        before = snapshot(opt)
        norm = opt.step(max_norm)
        assert int(opt.state["step"]) == t
        check(opt, before, t, max_norm, norm)
        for p in params:
            if p.grad is not None:
                p.grad.mul_(-0.7)
    return opt


# one value, around a group and a chunk, several tensors, more than a launch takes of either kind
SIZES = [[1], [3], [255, 256, 257], [1, 2, 5, 64, 1000], [2047, 2048, 2049, 4096 + 3], [100003],
         [7 + 13 * i for i in range(150)]]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "both"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[-1]}")
def test_steps(dev, sizes, kind, bits):
    print(f"[case] {len(sizes)} {sizes[-1]} {kind} {bits}", flush=True)
    kinds = [("f32", "bf16")[i % 2] if kind == "both" else kind for i in range(len(sizes))]
    run(make(sizes, kinds, len(sizes)), bits=bits)
    run(make(sizes, kinds, len(sizes)), bits=bits, max_norm=0.5)
    run(make(sizes, kinds, len(sizes), offset=1), bits=bits, max_norm=1e6)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_tensor_among_small_ones(dev, bits):
    """Chunks longer than their least, for the sums and the step."""
    run(make([5, (1 << 24) + 77, 300], ["bf16", "f32", "f32"], 4), bits=bits, max_norm=1.0, steps=1)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_shapes_and_empty_tensors(dev, bits):
    from mobilefinetuner_amd.adamw import AdamW
    params = [torch.randn(s, device=dev).requires_grad_(True) for s in ((4, 5, 6), (0, 8), (), (300, 3))]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = AdamW(params, state_bits=bits)
    opt.step(1.0)
    assert [v.shape for v in opt.views("exp_avg")] == [p.shape for p in params]
    empty = torch.zeros(0, device=dev, requires_grad=True)
    empty.grad = torch.zeros_like(empty)
    opt = AdamW([empty], state_bits=bits)
    opt.step()
    assert int(opt.state["step"]) == 0  # nothing was stepped


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_a_gradient(dev, bits):
    params = make([300, 5, 1000, 70], ["f32", "bf16", "bf16", "f32"], 7)
    params[1].grad = params[3].grad = None
    opt = run(params, bits=bits, max_norm=0.1)
    opt.zero_grad()
    assert all(p.grad is None for p in params)
    before = snapshot(opt)
    assert opt.step(1.0) is None and int(opt.state["step"]) == 2
    assert all(torch.equal(a[k], b[k]) for a, b in zip(before, snapshot(opt)) for k in "pmv")
    params = make([9], ["f32"], 8)
    from mobilefinetuner_amd.adamw import AdamW
    opt = AdamW(params)
    opt.zero_grad(set_to_none=False)
    assert (params[0].grad == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 2, 1000, 10 ** 5, 10 ** 9])
def test_step_numbers(dev, t):
    """The bias corrections, from a small difference to one."""
    from mobilefinetuner_amd.adamw import AdamW
    params = make([700], ["f32"], 9)
    opt = AdamW(params, LR, BETAS, EPS)
    opt.step()
    opt.state["step"].fill_(t - 1)
    before = snapshot(opt)
    opt.step()
    check(opt, before, t, None, None)
    assert int(opt.state["step"]) == t


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas,eps", [((0.0, 0.0), 1e-3), ((0.0, 0.999), 1e-8), ((0.95, 0.9), 1e-6)])
def test_other_betas(dev, betas, eps, bits):
    from mobilefinetuner_amd.adamw import AdamW
    params = make([700], ["f32"], 9)
    opt = AdamW(params, LR, betas, eps, weight_decay=[0.5], state_bits=bits)
    before = snapshot(opt)
    opt.step()
    if betas != (0.0, 0.0):
        g = before[0]["g"]
        m, v = (1 - betas[0]) * g, (1 - betas[1]) * g * g
        size = LR / (1 - betas[0])
        p = before[0]["p"] * (1 - 0.5 * LR) - size * m / ((v / (1 - betas[1])).sqrt() + eps)
        within(snapshot(opt)[0]["p"], p, 8 * U * before[0]["p"].abs() + 40 * U * (p.abs() + LR))
    else:
        p = before[0]["p"] * (1 - 0.5 * LR) - LR * before[0]["g"] / (before[0]["g"].abs() + eps)
        within(snapshot(opt)[0]["p"], p, 8 * U * before[0]["p"].abs() + 40 * U * (p.abs() + LR))


@pytest.mark.gpu
def test_weight_decay_of_each_parameter(dev):
    params = make([100, 200, 300], ["f32", "bf16", "f32"], 10)
    opt = run(params, weight_decay=[0.0, 0.1, 10.0])
    before = snapshot(opt)
    opt.weight_decay[0] = 3.0  # set between steps
    opt.step()
    check(opt, before, 3, None, None)


@pytest.mark.gpu
def test_a_small_root_beside_large_ones_does_not_vanish(dev):
    """8 bits: a value whose root is far below its group's largest keeps the smallest number, so that its
    average over it stays bounded: m / (0 + eps) would be 10^5 times the step."""
    from mobilefinetuner_amd.adamw import AdamW
    p = torch.zeros(256, device=dev, requires_grad=True)
    opt = AdamW([p], 1e-3, BETAS, EPS, weight_decay=0.0, state_bits=8)
    p.grad = torch.full((256,), 1e-3, device=dev)
    p.grad[::2] = 1e4
    opt.step()
    assert (opt.views("exp_avg_sq")[0].float() > 0).all()
    p.grad.zero_()
    for _ in range(20):
        opt.step()
    assert p.abs().max() < 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_gradient_that_is_no_number(dev, bad, bits):
    """Without clipping it stays with its value (in 8 bits: its group's states); with, NaN reaches all, an
    infinity makes the others' gradients zero."""
    from mobilefinetuner_amd.adamw import AdamW

    def stepped(value, max_norm):
        params = make([1000, 40], ["f32", "bf16"], 11)
        if value is not None:
            params[0].grad[300] = value
        opt = AdamW(params, LR, BETAS, EPS, state_bits=bits)
        opt.step(max_norm)
        return opt

    clean, opt = stepped(None, None), stepped(bad, None)
    p, q = opt.params[0].detach(), clean.params[0].detach()
    assert torch.isnan(p[300])
    keep = torch.arange(1000, device=dev) != 300
    assert torch.equal(p[keep], q[keep]) and torch.equal(opt.params[1], clean.params[1])
    m, mc = (torch.stack([held(o, n, 0) for n in ("exp_avg", "exp_avg_sq")]) for o in (opt, clean))
    group = torch.arange(1000) // 256 == 1 if bits == 8 else torch.arange(1000) == 300
    assert torch.equal(m[:, ~group], mc[:, ~group]) and not torch.isfinite(m[:, 300]).any()
    opt = stepped(bad, 1.0)
    if math.isnan(bad):
        assert all(torch.isnan(p).all() for p in opt.params)
    else:
        assert torch.isnan(opt.params[0][300]) and torch.isfinite(opt.params[0][keep]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_past_32_bits(dev, bits):
    """More than 2^31 values: the last ones are stepped as in a call of their own."""
    from mobilefinetuner_amd.adamw import AdamW
    n = (1 << 31) + 300
    p = torch.zeros(n, dtype=torch.bfloat16, device=dev, requires_grad=True)
    p.grad = torch.zeros_like(p)
    small = make([300], ["bf16"], 12)
    with torch.no_grad():
        p[-300:] = small[0]
    p.grad[-300:] = small[0].grad
    opt, ref = (AdamW(v, LR, BETAS, EPS, state_bits=bits) for v in ([p], small))
    for _ in range(2):
        norms = opt.step(0.5), ref.step(0.5)
    assert torch.equal(*norms) and torch.equal(p[-300:], small[0]) and (p[:1000] == 0).all()
    for name in ref.state:
        a, b = opt.state[name], ref.state[name]
        assert torch.equal(a.float().view(-1)[-b.numel():], b.float().view(-1))
    del opt, p


@pytest.mark.gpu
def test_captured_steps_count_and_follow_their_inputs(dev):
    """Replays with the program's own work between them: as eager steps with the same gradients and rates."""
    from mobilefinetuner_amd.adamw import AdamW
    sizes, kinds = [300, 5000, 77], ["f32", "bf16", "f32"]
    for bits in (32, 8):
        a, b = make(sizes, kinds, 13), make(sizes, kinds, 13)
        lr = torch.tensor(1e-2, device=dev)
        captured, eager = AdamW(a, lr, state_bits=bits), AdamW(b, 1e-2, state_bits=bits)
        captured.step(1.0)  # warm
        eager.step(1.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = captured.step(1.0)
        for i in range(4):
            rate = 1e-2 / (i + 1)
            lr.fill_(rate)
            eager.lr = float(torch.tensor(rate, dtype=torch.float32))
            for p, q in zip(a, b):
                p.grad.mul_(-0.9)
                q.grad.mul_(-0.9)
            graph.replay()
            ref = eager.step(1.0)
            torch.cuda.synchronize()
            assert int(captured.state["step"]) == i + 2
            assert torch.equal(norm, ref) and all(torch.equal(p, q) for p, q in zip(a, b))
            assert all(torch.equal(captured.state[k].float(), eager.state[k].float()) for k in eager.state)


@pytest.mark.gpu
def test_streams_and_repeated_runs(dev):
    """The same bits on another stream, and of two optimizers on two streams at once."""
    from mobilefinetuner_amd.adamw import AdamW
    sizes, kinds = [4000 + i for i in range(90)], ["f32", "bf16"] * 45
    runs = [make(sizes, kinds, 14) for _ in range(3)]
    opts = [AdamW(p, LR, state_bits=8) for p in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o, s in zip(opts, streams):
            with torch.cuda.stream(s):
                o.step(0.3)
    torch.cuda.synchronize()
    for o in opts[1:]:
        assert all(torch.equal(p, q) for p, q in zip(o.params, opts[0].params))
        assert all(torch.equal(o.state[k].float(), opts[0].state[k].float()) for k in o.state)


@pytest.mark.gpu
def test_what_a_caller_changes_between_steps(dev):
    """New gradients and data, gradients that are not contiguous, masters after a load, saved state."""
    from mobilefinetuner_amd.adamw import AdamW
    w = torch.randn(40, 50, device=dev).requires_grad_(True)
    h = torch.randn(600, device=dev).bfloat16().requires_grad_(True)
    w.grad, h.grad = torch.randn(50, 40, device=dev).t(), torch.randn(600, device=dev).bfloat16()
    opt = AdamW([w, h], LR, BETAS, EPS, state_bits=8)
    before = snapshot(opt)
    opt.step()
    check(opt, before, 1, None, None)
    w.data = torch.randn(40, 50, device=dev)
    with torch.no_grad():
        h.copy_(torch.randn(600, device=dev))
    opt.reload_masters()
    before = snapshot(opt)
    assert torch.equal(before[1]["p"], h.detach().cpu().double())
    opt.step()
    check(opt, before, 2, None, None)
    saved, at = opt.state_dict(), [w.detach().clone(), h.detach().clone()]
    opt.step()
    want = [w.detach().clone(), h.detach().clone()]
    w2, h2 = (t.clone().requires_grad_(True) for t in at)
    w2.grad, h2.grad = w.grad, h.grad
    other = AdamW([w2, h2], LR, BETAS, EPS, state_bits=8)
    other.load_state_dict(saved)
    other.step()
    assert torch.equal(w2, want[0]) and torch.equal(h2, want[1])
    with pytest.raises(ValueError, match="bits"):
        AdamW([w2, h2]).load_state_dict(saved)
    with pytest.raises(ValueError, match="must be"):
        AdamW([w2.detach()[:20].clone().requires_grad_(True), h2], state_bits=8).load_state_dict(saved)
    y = (w * w).sum()  # saved for its backward, then stepped
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_copies_and_gradient_modes(dev):
    """A deep copy steps on its own; no_grad and inference_mode make no difference; states from host memory."""
    import copy
    from mobilefinetuner_amd.adamw import AdamW
    opt = AdamW(make([300, 70], ["f32", "bf16"], 15), LR, state_bits=8)
    opt.step(1.0)
    other = copy.deepcopy(opt)
    third = AdamW([p.detach().clone().requires_grad_(True) for p in opt.params], LR, state_bits=8)
    third.load_state_dict({"state": {k: v.cpu() for k, v in opt.state_dict()["state"].items()}, "state_bits": 8})
    for p, q, r in zip(opt.params, other.params, third.params):
        assert p.data_ptr() != q.data_ptr() and torch.equal(p, q)
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    with torch.no_grad():
        opt.step(1.0)
    with torch.inference_mode():
        other.step(1.0)
    third.step(1.0)
    for o in (other, third):
        assert all(torch.equal(p, q) for p, q in zip(opt.params, o.params))
        assert all(torch.equal(opt.state[k].float(), o.state[k].float()) for k in opt.state)


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


def table(capi, **change):
    t = (capi.AdamWTensor * 2)()
    for i in range(2):
        for j, (name, _) in enumerate(capi.AdamWTensor._fields_):
            setattr(t[i], name, 256 if name == "n" else 0.0 if name == "weight_decay" else 4096 * (10 * i + j + 1))
    for name, v in change.items():
        setattr(t[1], name, v)
    return t


@pytest.mark.parametrize("change,message", [
    (dict(state_bits=16), "state_bits"), (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta1 and beta2"),
    (dict(beta1=math.nan), "beta1"), (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(eps=-1e-8), "eps"),
    (dict(max_norm=math.inf), "max_norm"), (dict(max_norm=-1.0), "max_norm"),
])
def test_descriptors_refused(capi, change, message):
    d = capi.adamw_desc(**{**dict(lr=1e-3), **change})
    with pytest.raises(capi.MftError, match=message):
        capi.adamw_workspace_size(d, table(capi))
    with pytest.raises(capi.MftError, match=message):
        capi.adamw_step(d, table(capi), 64, None, 128, None)


@pytest.mark.parametrize("change,message", [
    (dict(n=-1), "n must be"), (dict(n=1 << 41), "2\\^40"), (dict(weight_decay=-1.0), "weight_decay"),
    (dict(weight_decay=math.nan), "weight_decay"), (dict(param=None), "non-NULL"), (dict(exp_avg=None), "non-NULL"),
    (dict(exp_avg_sq=None), "non-NULL"), (dict(exp_avg_scale=None), "non-NULL"),
    (dict(exp_avg_sq_scale=None), "non-NULL"), (dict(exp_avg=4096 * 12), "one another"),
    (dict(grad=4096 * 12), "gradient"),
])
def test_tensors_refused(capi, change, message):
    d = capi.adamw_desc(1e-3, state_bits=8)
    with pytest.raises(capi.MftError, match=message):
        capi.adamw_step(d, table(capi, **change), 64, None, 128, None)


def test_operands_refused(capi):
    d, t = capi.adamw_desc(1e-3), table(capi)
    for step, norm, ws, message in ((None, None, 128, "non-NULL"), (64, None, None, "non-NULL"), (64, 32, 128, "max_norm")):
        with pytest.raises(capi.MftError, match=message):
            capi.adamw_step(d, t, step, norm, ws, None)
    assert capi.lib().mft_adamw_step(C.byref(d), 2, None, 64, None, 128, None) == capi.MFT_ERR_INVALID_ARG
    assert capi.lib().mft_adamw_step(None, 0, None, 64, None, 128, None) == capi.MFT_ERR_INVALID_ARG
    assert capi.lib().mft_adamw_step(C.byref(d), -1, t, 64, None, 128, None) == capi.MFT_ERR_INVALID_ARG
    assert capi.lib().mft_adamw_step(C.byref(d), 0, None, None, None, None, None) == capi.MFT_OK
    for x in t:
        x.grad = None
    capi.adamw_step(d, t, None, None, None, None)  # nothing to step


def test_no_cpu_path():
    from mobilefinetuner_amd.adamw import AdamW
    with pytest.raises(ValueError, match="no CPU path"):
        AdamW([torch.zeros(4, requires_grad=True)])
    with pytest.raises(ValueError, match="at least one"):
        AdamW([])


@pytest.mark.gpu
def test_parameters_refused(dev):
    from mobilefinetuner_amd.adamw import AdamW
    p = torch.zeros(8, 8, device=dev, requires_grad=True)
    for bad in (lambda: AdamW([p, p]), lambda: AdamW([p.detach()[:5], p.detach()[4:]]), lambda: AdamW([p * 2]),
                lambda: AdamW([p.detach().t()[1:]]), lambda: AdamW([p.detach().half()]), lambda: AdamW([p], state_bits=16),
                lambda: AdamW([p], weight_decay=[0.1, 0.1]), lambda: AdamW([p, p.detach().cpu()])):
        with pytest.raises(ValueError):
            bad()
    opt = AdamW([p])
    p.grad = torch.zeros_like(p)
    for norm in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            opt.step(norm)
    for lr in (torch.zeros(2, device=dev), torch.zeros(()), torch.zeros((), device=dev, dtype=torch.float64)):
        opt.lr = lr
        with pytest.raises(ValueError, match="lr"):
            opt.step()
    opt.lr = 1e-3
    p.grad = None
    p.grad = torch.eye(8, device=dev).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        opt.step()
    p.grad = None
    p.grad = torch.zeros_like(p)
    p.data = torch.zeros(4, 8, device=dev)
    with pytest.raises(ValueError, match="size"):
        opt.step()
    p.data = torch.zeros(8, 8, device=dev)
    opt.state["exp_avg"] = torch.zeros(8, device=dev)
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    assert int(opt.state["step"]) == 0


@pytest.mark.gpu
def test_parameters_turned_in_place_refused(dev):
    from mobilefinetuner_amd.adamw import AdamW
    p = torch.randn(8, 4, device=dev, requires_grad=True)
    opt = AdamW([p])
    p.grad = torch.randn_like(p)
    opt.step()
    before = p.detach().clone()
    p.grad = None
    p.data = p.data.t()  # the same memory and size in another order
    p.grad = torch.ones(4, 8, device=dev)
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert int(opt.state["step"]) == 1 and torch.equal(p.detach().t(), before)
    p.data = p.data.t()
    p.grad = torch.ones(8, 4, device=dev)
    opt.step()
    assert int(opt.state["step"]) == 2 and not torch.equal(p.detach(), before)


@pytest.mark.gpu
def test_a_pending_backward_through_what_is_not_stepped(dev):
    from mobilefinetuner_amd.adamw import AdamW
    p, q = (torch.full((8,), v, device=dev, requires_grad=True) for v in (2.0, 3.0))
    opt = AdamW([p, q])
    loss = (q * q).sum()  # holds q until its backward
    p.grad = torch.ones_like(p)
    opt.step()
    loss.backward()
    assert torch.equal(q.grad, torch.full_like(q, 6.0))
    loss = (p * p).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_but_empty_gradients(dev, bits):
    from mobilefinetuner_amd.adamw import AdamW
    p, q = torch.zeros(0, 4, device=dev, requires_grad=True), torch.ones(4, device=dev, requires_grad=True)
    for params in ([p], [p, q]):
        opt = AdamW(params, state_bits=bits)
        p.grad = torch.zeros_like(p)
        assert opt.step(1.0) is None and opt.step() is None
        assert int(opt.state["step"]) == 0 and torch.equal(q.detach(), torch.ones_like(q))


@pytest.mark.gpu
def test_eight_bits_are_those_of_the_quotient(dev):
    """To the bit, scale = max |x| (1 / 448) and q = e4m3(x / scale), all in fp32, for x = m and sqrt(v): those
    of a first step are (1 - beta1) g and sqrt((1 - beta2) g^2), as with states in 32 bits.  Gradients with few
    digits, whose quotients often lie halfway between two numbers."""
    from mobilefinetuner_amd.adamw import AdamW
    g = torch.Generator().manual_seed(21)
    grad = (torch.randint(1, 256, (1 << 18,), generator=g) / 128 * (1 - 2 * torch.randint(0, 2, (1 << 18,), generator=g)))
    grad *= 2.0 ** torch.randint(-6, 1, (1 << 18,), generator=g)
    opts = []
    for bits in (32, 8):
        p = torch.zeros(1 << 18, device=dev, requires_grad=True)
        p.grad = grad.to(dev)
        opts.append(AdamW([p], LR, (0.5, 0.75), EPS, state_bits=bits))  # powers of two: m and v have few digits, too
        opts[-1].step()
    wide, narrow = (o.state for o in opts)
    for name, x in (("exp_avg", wide["exp_avg"].cpu()), ("exp_avg_sq", wide["exp_avg_sq"].cpu().sqrt())):
        x = x.view(-1, 256)
        scale = x.abs().amax(1) * (torch.tensor(1.0) / 448)
        assert torch.equal(narrow[name + "_scale"].cpu(), scale)
        q = (x / scale[:, None]).to(torch.float8_e4m3fn).float()
        if name == "exp_avg_sq":
            q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
        assert torch.equal(narrow[name].float().cpu().view(-1, 256), q)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_of_other_parameters_refused(dev, bits, tmp_path):
    """The same padded size in other parts: swapped, cut elsewhere, turned, the master beside the other parameter.  A
    state without the parameters' shapes loads as far as its sizes fit."""
    from mobilefinetuner_amd.adamw import AdamW

    def opt(*params):
        ps = [torch.ones(s, device=dev, dtype=t).requires_grad_(True) for s, t in params]
        for p in ps:
            p.grad = torch.ones_like(p)
        return AdamW(ps, state_bits=bits)

    f, b = torch.float32, torch.bfloat16
    first = opt(([300], f), ([200], f), ([16, 8], b), ([8, 16], f))
    first.step()
    torch.save(first.state_dict(), tmp_path / "state")
    saved = torch.load(tmp_path / "state", weights_only=True)
    for others in ([([200], f), ([300], f), ([16, 8], b), ([8, 16], f)], [([301], f), ([199], f), ([16, 8], b), ([8, 16], f)],
                   [([300], f), ([200], f), ([8, 16], b), ([8, 16], f)], [([300], f), ([200], f), ([16, 8], f), ([8, 16], b)],
                   [([300], f), ([200], f), ([16, 8], b), ([8, 16], f), ([0], f)], [([500], f), ([16, 8], b), ([8, 16], f)]):
        other = opt(*others)
        before = {k: v.clone() for k, v in other.state.items()}
        with pytest.raises(ValueError, match="they differ|must be"):
            other.load_state_dict(saved)
        assert all(torch.equal(before[k].float(), v.float()) for k, v in other.state.items())
    for d in (saved, {k: saved[k] for k in ("state", "state_bits")}):
        same = opt(([300], f), ([200], f), ([16, 8], b), ([8, 16], f))
        same.load_state_dict(d)
        assert all(torch.equal(first.state[k].float(), v.float()) for k, v in same.state.items())


@pytest.mark.gpu
def test_weight_decay_set_between_steps(dev):
    """A number, a list or one element of it, as at the start; lists of another length are refused and nothing is
    stepped."""
    params = make([100, 200, 300], ["f32", "bf16", "f32"], 10)
    opt = run(params, weight_decay=0.3)
    t = 2
    for decay in (0.1, [0.0, 0.2, 0.4], (0.5, 0.6, 0.7)):
        opt.weight_decay = decay
        assert opt.weight_decay == (list(decay) if isinstance(decay, (list, tuple)) else [decay] * 3)
        before, t = snapshot(opt), t + 1
        opt.step()
        check(opt, before, t, None, None)
    opt.weight_decay[1] = 5.0
    before, t = snapshot(opt), t + 1
    opt.step()
    check(opt, before, t, None, None)
    for decay in ([0.1], [0.1] * 4, []):
        with pytest.raises(ValueError, match="weight_decay has"):
            opt.weight_decay = decay
    before = snapshot(opt)
    for change in (lambda: opt.weight_decay.append(0.1), lambda: [opt.weight_decay.pop() for _ in range(2)]):
        change()
        with pytest.raises(ValueError, match="weight_decay has"):
            opt.step()
    assert int(opt.state["step"]) == t and all(torch.equal(a[k], b[k]) for a, b in zip(before, snapshot(opt)) for k in "pmv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eight_bits_of_several_steps(dev, dtype):
    """To the bit, over five steps: beta times the state rounded, then the gradient's share added with one rounding (in
    64 bits here, whose own rounding comes before that in one of 2^29), then numbers and scales as above.  A
    number off at a tie would move its group's scale by percents in a step after it."""
    from mobilefinetuner_amd.adamw import AdamW
    n = 1 << 22
    g = torch.Generator(device=dev).manual_seed(22)
    p = (0.02 * torch.randn(n, device=dev, generator=g)).to(dtype).requires_grad_(True)
    opt = AdamW([p], LR, BETAS, EPS, state_bits=8)
    m, v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    b1, b2, r1, r2 = (torch.tensor(x, device=dev) for x in (*BETAS, 1 - BETAS[0], 1 - BETAS[1]))
    by_448 = torch.tensor(1.0, device=dev) / torch.tensor(448.0, device=dev)

    def held(x, positive):
        x = x.view(-1, 256)
        scale = (x.abs().amax(1) * by_448).clamp(min=2.0 ** -126)
        q = x / scale[:, None]
        q = (torch.where(q > 0, q.clamp(min=2.0 ** -9), q) if positive else q).to(torch.float8_e4m3fn).float()
        return q, scale, (q * scale[:, None]).view(-1)

    for _ in range(5):
        p.grad = (1e-3 * torch.randn(n, device=dev, generator=g)).to(dtype)
        opt.step()
        grad = p.grad.float()
        m = ((b1 * m).double() + r1.double() * grad.double()).float()
        v = ((b2 * v).double() + (r2 * grad).double() * grad.double()).float()
        mq, ms, m = held(m, False)
        vq, vs, root = held(v.sqrt(), True)
        v = root.square()
        for name, q, scale in (("exp_avg", mq, ms), ("exp_avg_sq", vq, vs)):
            assert torch.equal(opt.state[name + "_scale"], scale)
            assert torch.equal(opt.state[name].float().view(-1, 256), q)
