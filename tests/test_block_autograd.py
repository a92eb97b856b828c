"""The nodes of the RMS norm and the gated linear layer, and a block's half as they make it with the linear layer
and the AdamW step.  The nodes on the CPU with plain functions in the kernels' place and on the GPU with the
kernels: their gradients are first-order, and a derivative through them raises."""
import itertools
import math

import pytest
import torch
import torch.nn.functional as F

U = 2.0 ** -24
ACT = {"relu": torch.relu, "silu": F.silu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}


def plain_rms_norm(x, weight=None, residual=None, norm="gemma", eps=1e-6):
    total = x if residual is None else x + residual
    rstd = torch.rsqrt(total.square().mean(-1) + eps)
    f = 1 if weight is None else weight + (norm == "gemma")
    return total * rstd[..., None] * f, None if residual is None else total, rstd


def plain_rms_norm_backward(x, weight, rstd, dy, dtotal=None, norm="gemma", want_x=True, want_weight=True):
    h = x * rstd[..., None]
    g = dy if weight is None else dy * (weight + (norm == "gemma"))
    dx = rstd[..., None] * (g - h * (g * h).mean(-1, keepdim=True)) + (0 if dtotal is None else dtotal)
    return dx if want_x else None, (dy * h).sum(0) if want_weight else None


def plain_gated_linear(x, W_gate, W_up, activation="gelu_tanh", w_transposed=False, want_preact=False):
    gate, up = (x @ (W.t() if w_transposed else W) for W in (W_gate, W_up))
    return ACT[activation](gate) * up, gate if want_preact else None, up if want_preact else None


def plain_gated_linear_backward(x, W_gate, W_up, gate, up, dh, activation="gelu_tanh", w_transposed=False, want_x=True,
                                want_gate=True, want_up=True):
    with torch.enable_grad():
        q = [t.detach().requires_grad_(True) for t in (x, W_gate, W_up)]
        grads = torch.autograd.grad(plain_gated_linear(*q, activation, w_transposed)[0], q, dh.detach())
    return tuple(g.clone(memory_format=torch.contiguous_format) if w else None
                 for g, w in zip(grads, (want_x, want_gate, want_up)))


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def place(request, monkeypatch):
    if request.param == "cuda":
        return request.getfixturevalue("dev")
    from mobilefinetuner_amd import gated_linear, rms_norm
    for module, names in ((rms_norm, ("rms_norm", "rms_norm_backward")),
                          (gated_linear, ("gated_linear", "gated_linear_backward"))):
        for name in names:
            monkeypatch.setattr(module, name, globals()["plain_" + name])
    return torch.device("cpu")


def leaves(place, *shapes):
    g = torch.Generator().manual_seed(len(shapes))
    return [torch.randn(s, generator=g).to(place).requires_grad_(True) for s in shapes]


def cases(place):
    """Leaves, and a node's outputs from them."""
    from mobilefinetuner_amd.gated_linear import GatedLinear
    from mobilefinetuner_amd.rms_norm import AddRMSNorm, RMSNorm
    yield leaves(place, (5, 24), (24,)), lambda x, w: RMSNorm.apply(x, w)
    yield leaves(place, (5, 24), (5, 24), (24,)), lambda *v: torch.stack(AddRMSNorm.apply(*v))
    yield leaves(place, (5, 24), (5, 24), (24,)), lambda *v: AddRMSNorm.apply(*v)[0]
    for w_t in (False, True):
        yield (leaves(place, (5, 24), *[(16, 24) if w_t else (24, 16)] * 2),
               lambda *v, w_t=w_t: GatedLinear.apply(*v, "silu", w_t))


@pytest.mark.parametrize("squared", [False, True], ids=["constant", "function"])
def test_a_second_derivative_raises(place, squared):
    """For each leaf's gradient, with respect to each leaf that it may depend on, by both ways that torch has;
    the incoming gradient constant or a function of the leaves.  The gradients themselves are as without a graph."""
    for at, f in cases(place):
        def loss():
            y = f(*at)
            return (y * y).sum() if squared else y.sum()

        first = torch.autograd.grad(loss(), at)
        grads = torch.autograd.grad(loss(), at, create_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(grads, first))
        for g, leaf in itertools.product(grads, at):
            for run in (lambda: torch.autograd.grad((g * g).sum() + leaf.sum(), leaf, retain_graph=True),
                        lambda: ((g * g).sum() + leaf.sum()).backward(retain_graph=True)):
                with pytest.raises(RuntimeError, match="no second order"):
                    run()
                leaf.grad = None


def test_gradients_that_are_not_wanted(place):
    """Frozen weights (an adapter's base), a frozen stream, and gradients of their own memory."""
    from mobilefinetuner_amd.gated_linear import GatedLinear
    from mobilefinetuner_amd.rms_norm import AddRMSNorm
    x, r, w = leaves(place, (5, 24), (5, 24), (24,))
    y, total = AddRMSNorm.apply(x, r, w, "gemma", 1e-6)
    (y.sum() + total.sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    for frozen in itertools.product((False, True), repeat=3):
        v = [t.detach().clone().requires_grad_(not f) for t, f in zip((x, r, w), frozen)]
        if all(frozen):
            assert not AddRMSNorm.apply(*v)[0].requires_grad
            continue
        y, total = AddRMSNorm.apply(*v)
        (y.sum() + total.sum()).backward()
        assert all((t.grad is None) if f else torch.equal(t.grad, g) for t, f, g in zip(v, frozen, (x.grad, r.grad, w.grad)))
    a, Wg, Wu = leaves(place, (5, 24), (16, 24), (16, 24))
    GatedLinear.apply(a, Wg, Wu, "silu", True).sum().backward()
    assert Wg.grad.data_ptr() != Wu.grad.data_ptr() and not Wg.grad._is_view()
    for frozen in itertools.product((False, True), repeat=3):
        v = [t.detach().clone().requires_grad_(not f) for t, f in zip((a, Wg, Wu), frozen)]
        h = GatedLinear.apply(*v, "silu", True)
        if all(frozen):
            assert not h.requires_grad
            continue
        h.sum().backward()
        # fp32 gradients alone or in one product: each within the other's bound, 2 (16 + 8) u of sums of magnitudes
        for t, f, g in zip(v, frozen, (a.grad, Wg.grad, Wu.grad)):
            assert (t.grad is None) if f else float((t.grad - g).abs().max()) <= 1e-4


def test_the_sums_are_kept_for_a_backward_only(place, monkeypatch):
    from mobilefinetuner_amd import gated_linear as L
    asked, real = [], L.gated_linear
    monkeypatch.setattr(L, "gated_linear", lambda *a, **k: (asked.append(a[5] if len(a) > 5 else k.get("want_preact", False)),
                                                            real(*a, **k))[1])
    x, Wg, Wu = leaves(place, (5, 24), (24, 16), (24, 16))
    L.GatedLinear.apply(x, Wg, Wu)
    with torch.no_grad():
        L.GatedLinear.apply(x, Wg, Wu)
    with torch.inference_mode():
        L.GatedLinear.apply(x, Wg, Wu)
    L.GatedLinear.apply(x.detach(), Wg.detach(), Wu.detach())
    L.GatedLinear.apply(x.detach(), Wg, Wu.detach())
    assert asked == [True, False, False, False, True]


# ------------------------------------------------------------ a run of them together
IN, FF, ROWS = 96, 160, 24


def block_weights(t, dev):
    g = torch.Generator().manual_seed(3)
    shapes = dict(norm1=(IN,), gate=(FF, IN), up=(FF, IN), down=(IN, FF), norm2=(IN,))
    return {k: ((0.1 * torch.randn(s, generator=g)) if len(s) == 1 else
                torch.randn(s, generator=g) / math.sqrt(s[1])).to(torch.float32 if len(s) == 1 else t).to(dev)
            for k, s in shapes.items()}


def block(p, x, attn):
    """The second half of a block and the next one's norm: (its normed input, the stream)."""
    from mobilefinetuner_amd.gated_linear import GatedLinear
    from mobilefinetuner_amd.linear import Linear
    from mobilefinetuner_amd.rms_norm import AddRMSNorm
    y, stream = AddRMSNorm.apply(attn, x, p["norm1"], "gemma", 1e-6)
    h = GatedLinear.apply(y, p["gate"], p["up"], "gelu_tanh", True)
    out = Linear.apply(h, p["down"], None, None, "none", True)
    return AddRMSNorm.apply(out, stream, p["norm2"], "gemma", 1e-6)


def ref_block(p, x, attn):
    def norm(s, w):
        return s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * (1 + w)

    stream = x + attn
    y = norm(stream, p["norm1"])
    h = F.gelu(y @ p["gate"].t(), approximate="tanh") * (y @ p["up"].t())
    stream = stream + h @ p["down"].t()
    return norm(stream, p["norm2"]), stream


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_blocks_half_and_its_step(dev, dtype):
    """Gradients against torch's in 64 bits, then the step of all parameters with clipping against the formula.
    Normwise: a product of K terms is off by 2 (K + 8) u of its sum of magnitudes, for normal operands
    sqrt(K) times its norm, so by 3e-4 in fp32 at K 160, and in bf16 each stored value by half a step, 2^-9 in
    the mean; eight such stages in a row, with slopes under 1.13 and norms that double an error at most."""
    from mobilefinetuner_amd.adamw import AdamW
    g = torch.Generator().manual_seed(4)
    x, attn, c, e = (torch.randn(ROWS, IN, generator=g).to(dtype).to(dev) for _ in range(4))
    p = {k: v.requires_grad_(True) for k, v in block_weights(dtype, dev).items()}
    y, stream = block(p, x, attn)
    torch.autograd.backward([y, stream], [c, e])
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    ry, rs = ref_block(q, x.double(), attn.double())
    torch.autograd.backward([ry, rs], [c.double(), e.double()])
    tol = 8 * 2 * (3e-4 if dtype == torch.float32 else 2.0 ** -9 * 1.13)
    for got, ref in ((y, ry), (stream, rs), *((p[k].grad, q[k].grad) for k in p)):
        assert float((got.detach().double() - ref.detach()).norm()) <= tol * float(ref.detach().norm())
    names = list(p)
    opt = AdamW([p[k] for k in names], lr=1e-2, weight_decay=[0.0 if "norm" in k else 0.1 for k in names])
    before = {k: v.detach().double().clone() for k, v in p.items()}
    grads = {k: v.grad.double() for k, v in p.items()}
    norm = opt.step(max_norm=1.0)
    ref = math.sqrt(sum(float(v.square().sum()) for v in grads.values()))
    assert abs(float(norm) - ref) <= 2 * U * ref
    for k in names:
        d = min(1.0, 1.0 / (ref + 1e-6)) * grads[k]  # the first step: m / sqrt(v) is the gradient's sign but for eps
        want = before[k] * (1 - 1e-2 * (0.0 if "norm" in k else 0.1)) - 1e-2 * d / (d.abs() + 1e-8)
        step = torch.finfo(p[k].dtype).eps / 2
        off = (p[k].detach().double() - want).abs()
        assert bool((off <= (step + 8 * U) * want.abs() + 4 * U * before[k].abs() + 1e-2 * 32 * U).all())
    opt.zero_grad()
    block(p, x, attn)[0].sum().backward()  # the next step's graph, of the stepped parameters
    opt.step(max_norm=1.0)
    assert int(opt.state["step"]) == 2


@pytest.mark.gpu
def test_a_prompt_through_eight_bit_weights(dev):
    """The norm's 8-bit rows into the gated layer and the linear layer behind it, against the 8-bit numbers in 64
    bits: gate and up lose 7 2^-13 of their sums of magnitudes at most, sqrt(96) times their norms, and h, the
    down product and both outputs half a step each."""
    from mobilefinetuner_amd.gated_linear import gated_linear_e4m3
    from mobilefinetuner_amd.linear import linear
    from mobilefinetuner_amd.rms_norm import quantize_rows, rms_norm_e4m3
    g = torch.Generator().manual_seed(5)
    x, attn = (torch.randn(ROWS, IN, generator=g).bfloat16().to(dev) for _ in range(2))
    p = block_weights(torch.bfloat16, dev)
    (gq, gs), (uq, us) = quantize_rows(p["gate"]), quantize_rows(p["up"])
    q, scale, stream = rms_norm_e4m3(attn, p["norm1"], x)
    h = gated_linear_e4m3(q, scale, gq, gs, uq, us)
    out, _ = linear(h, p["down"], residual=stream, w_transposed=True)
    wide = [v.float().double() * s.double()[:, None] for v, s in ((q, scale), (gq, gs), (uq, us))]
    rh = F.gelu(wide[0] @ wide[1].t(), approximate="tanh") * (wide[0] @ wide[2].t())
    ref = (attn.float() + x.float()).bfloat16().double() + rh @ p["down"].double().t()
    tol = 2 * 1.13 * 7 * 2.0 ** -13 * math.sqrt(IN) + 4 * 2.0 ** -9
    assert float((out.double() - ref).norm()) <= tol * float(ref.norm())


@pytest.mark.gpu
def test_lora_adapters_are_stepped(dev):
    """LoRALinear's parameters by AdamW: as many steps as calls, and the adapter's output follows them."""
    from mobilefinetuner_amd.adamw import AdamW
    from mobilefinetuner_amd.lora import LoRALinear
    g = torch.Generator().manual_seed(6)
    layers = []
    for i in range(3):
        layer = LoRALinear(torch.randn(IN, 40, generator=g).to(dev))
        layer.attach_lora(torch.randn(IN, 4, generator=g).to(dev) * 0.1, torch.zeros(4, 40, device=dev), 2.0)
        layers.append(layer)
    opt = AdamW([t for layer in layers for t in layer.trainable_parameters()], lr=1e-2, state_bits=8)
    x, c = torch.randn(7, IN, generator=g).to(dev), torch.randn(7, 40, generator=g).to(dev)
    start = [t.detach().clone() for t in opt.params]
    for _ in range(2):
        opt.zero_grad()
        (sum(layer.forward(x) for layer in layers) * c).sum().backward()
        grads = [t.grad.clone() for t in opt.params]
        opt.step(max_norm=0.5)
    assert int(opt.state["step"]) == 2
    for i, layer in enumerate(layers):
        A, B = layer.trainable_parameters()
        assert not torch.equal(B, start[2 * i + 1]) and all(bool(torch.isfinite(v).all()) for v in (A, B, *grads))
        ref = x.double() @ layer.W.double() + 2.0 * (x.double() @ A.double()) @ B.double()
        mags = x.double().abs() @ layer.W.double().abs() + 2.0 * (x.double().abs() @ A.double().abs()) @ B.double().abs()
        assert bool(((layer.forward(x).double() - ref).abs() <= 4 * (IN + 12) * U * mags + 1e-30).all())
