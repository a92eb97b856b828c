"""The autograd nodes of the layer norm, the linear layer and the token log
probabilities: their gradients are first-order, and a derivative through them
raises.  On the CPU with plain functions in the kernels' place, on the GPU with
the kernels."""
import itertools

import pytest
import torch

ACT = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
       "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}


def plain_layer_norm(x, weight=None, bias=None, eps=1e-5):
    var, mean = torch.var_mean(x, -1, unbiased=False)
    return torch.nn.functional.layer_norm(x, x.shape[-1:], weight, bias, eps), mean, torch.rsqrt(var + eps)


def plain_layer_norm_backward(x, weight, mean, rstd, dy, want_x=True, want_params=True):
    h = (x - mean[..., None]) * rstd[..., None]
    g = dy if weight is None else dy * weight
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx if want_x else None, (dy * h).sum(0) if want_params else None, dy.sum(0) if want_params else None


def plain_linear(x, W, bias=None, activation="none", residual=None, w_transposed=False, want_preact=False):
    z = x @ (W.t() if w_transposed else W) + (0 if bias is None else bias)
    y = ACT[activation](z).clone() + (0 if residual is None else residual)
    return y, z if want_preact else None


def plain_linear_backward(x, W, z, dy, activation="none", w_transposed=False, want_x=True, want_weight=True,
                          want_bias=True):
    dz = dy.clone()
    if activation != "none":
        with torch.enable_grad():
            q = z.detach().requires_grad_(True)
            dz, = torch.autograd.grad(ACT[activation](q), q, dy.detach())
    dW = dz.t() @ x if w_transposed else x.t() @ dz
    return (dz @ (W if w_transposed else W.t()) if want_x else None, dW if want_weight else None,
            dz.sum(0) if want_bias else None)


def plain_token_logprobs(logits, tokens, top=0, ignore_index=-100, check_tokens=True):
    q = torch.log_softmax(logits, -1)
    m = logits.max(-1).values
    lp = q.gather(-1, tokens.long()[..., None])[..., 0]
    return lp, -(q.exp() * q).sum(-1), torch.stack([m, (logits - m[..., None]).exp().sum(-1).log()], -1), None, None


def plain_token_logprobs_backward(logits, tokens, stats, entropy, grad_logprob, grad_entropy=None, ignore_index=-100):
    q = torch.log_softmax(logits, -1)
    p = q.exp()
    g = torch.zeros_like(logits)
    if grad_logprob is not None:
        hot = torch.nn.functional.one_hot(tokens.long(), logits.shape[-1])
        g += grad_logprob[..., None] * (hot - p)
    if grad_entropy is not None:
        g -= grad_entropy[..., None] * p * (q + entropy[..., None])
    return g


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def place(request, monkeypatch):
    if request.param == "cuda":
        return request.getfixturevalue("dev")
    from mobilefinetuner_amd import layer_norm, linear, logprobs
    for module, names in ((layer_norm, ("layer_norm", "layer_norm_backward")), (linear, ("linear", "linear_backward")),
                          (logprobs, ("token_logprobs", "token_logprobs_backward"))):
        for name in names:
            monkeypatch.setattr(module, name, globals()["plain_" + name])
    return torch.device("cpu")


def leaves(place, *shapes):
    g = torch.Generator().manual_seed(len(shapes))
    return [torch.randn(s, generator=g).to(place).requires_grad_(True) for s in shapes]


def cases(place):
    """Leaves, and a node's outputs from them."""
    from mobilefinetuner_amd.layer_norm import LayerNorm
    from mobilefinetuner_amd.linear import Linear
    from mobilefinetuner_amd.logprobs import TokenLogprobs
    t = torch.tensor([3, 0, 8, 1, 5], dtype=torch.int32, device=place)
    yield leaves(place, (5, 24), (24,), (24,)), lambda x, w, b: LayerNorm.apply(x, w, b, 1e-5)
    for act, w_t in itertools.product(("none", "gelu_tanh"), (False, True)):
        yield (leaves(place, (5, 24), (16, 24) if w_t else (24, 16), (16,), (5, 16)),
               lambda *v, act=act, w_t=w_t: Linear.apply(*v, act, w_t))
    yield leaves(place, (5, 9)), lambda z: torch.stack(TokenLogprobs.apply(z, t))
    yield leaves(place, (5, 9)), lambda z: TokenLogprobs.apply(z, t)[0]


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
        for g, leaf in itertools.product(grads[:3], at[:2]):  # the residual's gradient is the incoming one
            for run in (lambda: torch.autograd.grad((g * g).sum() + leaf.sum(), leaf, retain_graph=True),
                        lambda: ((g * g).sum() + leaf.sum()).backward(retain_graph=True)):
                with pytest.raises(RuntimeError, match="no second order"):
                    run()
                leaf.grad = None


def test_a_bias_behind_the_activation(place):
    """Only the bias is trained: the gradient is a function of it by the activation."""
    from mobilefinetuner_amd.linear import Linear
    x, W, b = leaves(place, (5, 24), (24, 16), (16,))
    y = Linear.apply(x.detach(), W.detach(), b, None, "silu", False)
    g, = torch.autograd.grad(y.sum(), b, create_graph=True)
    with pytest.raises(RuntimeError, match="no second order"):
        torch.autograd.grad(g.sum() + b.sum(), b)


def test_the_residuals_gradient_has_its_own(place):
    """It is the incoming one: its derivative is right, and only one that goes through the node's own gradients
    raises."""
    from mobilefinetuner_amd.linear import Linear
    x, W, b, r = leaves(place, (5, 24), (24, 16), (16,), (5, 16))
    y = Linear.apply(x, W, b, r, "none", False)
    dx, dr = torch.autograd.grad((y * y).sum(), (x, r), create_graph=True)
    again, = torch.autograd.grad(dr.sum(), r, retain_graph=True)
    assert torch.equal(again, torch.full_like(r, 2.0))
    with pytest.raises(RuntimeError, match="no second order"):
        torch.autograd.grad(dr.sum() + dx.sum(), r)


def test_nothing_to_differentiate_stays_without_a_graph(place):
    """create_graph over gradients that depend on nothing trained, and backward without it."""
    from mobilefinetuner_amd.linear import Linear
    x, W, r = leaves(place, (5, 24), (24, 16), (5, 16))
    y = Linear.apply(x.detach(), W.detach(), None, r, "none", False)
    g, = torch.autograd.grad(y.sum(), r, create_graph=True)
    assert not g.requires_grad
    y = Linear.apply(x, W, None, r, "none", False)
    y.sum().backward()
    assert not any(t.grad.requires_grad for t in (x, W, r))


def test_the_pre_activation_is_kept_for_a_backward_only(place, monkeypatch):
    """Not under no_grad or inference_mode, nor where only the residual is trained."""
    from mobilefinetuner_amd import linear as L
    asked, real = [], L.linear
    monkeypatch.setattr(L, "linear", lambda *a, **k: (asked.append(a[6] if len(a) > 6 else k.get("want_preact", False)),
                                                      real(*a, **k))[1])
    x, W, b, r = leaves(place, (5, 24), (24, 16), (16,), (5, 16))
    y = L.Linear.apply(x, W, b, r, "silu")
    with torch.no_grad():
        quiet = L.Linear.apply(x, W, b, r, "silu", False)
    with torch.inference_mode():
        L.Linear.apply(x, W, b, r, "silu", False)
    L.Linear.apply(x.detach(), W.detach(), b.detach(), r, "silu")
    L.Linear.apply(x, W, b)
    assert asked == [True, False, False, False, False]
    assert torch.equal(quiet, y) and not quiet.requires_grad
    y.sum().backward()
    assert all(t.grad is not None for t in (x, W, b, r))
