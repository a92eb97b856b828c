"""The operators around attention in a transformer block, as cases that can be timed.

  norm    layer norm over the last dimension, and its gradients
  linear  a matrix product with bias, activation and residual in its epilogue, and its gradients
  tokens  log probabilities of given tokens with the entropy and the top alternatives, and the gradient

A case is one call of one of them.  With `own` false it is computed in plain
torch operations in 32 bits; with `own` true by the package's operator.

Parameters (a norm's weight and bias, a linear layer's bias) are fp32 and so
are their gradients; activations, the matrix W and logits have the case's type
and so do their gradients.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
IGNORE = -100


# --------------------------------------------------------------------- cases
def _norm(dtype, N, D, grad=False):
    return dict(kind="norm", dtype=dtype, N=N, D=D, grad=grad)


def _linear(dtype, N, n_in, n_out, act="none", residual=False, w_out_in=False, grad=False):
    return dict(kind="linear", dtype=dtype, N=N, n_in=n_in, n_out=n_out, act=act, residual=residual,
                w_out_in=w_out_in, grad=grad)


def _tokens(dtype, N, V, top=0, grad=False):
    return dict(kind="tokens", dtype=dtype, N=N, V=V, top=top, grad=grad)


def listed():
    return [
        # the norm in front of a block for a single generated token, GPT-2 small: latency
        dict(_norm("bf16", 1, 768), name="norm token"),
        # the same norm in fp32 over a batch of 4 x 1024 tokens
        dict(_norm("f32", 4096, 768), name="norm forward f32"),
        # a training step's norm backward, GPT-2 medium, 16 x 1024 tokens
        dict(_norm("bf16", 16384, 1024, grad=True), name="norm backward bf16"),
        # a ragged batch, packed to its valid tokens, and a width off every vector boundary
        dict(_norm("f32", 1001, 1153, grad=True), name="norm backward ragged"),
        # the up projection of a single generated token: every weight is read once
        dict(_linear("bf16", 1, 1024, 4096, act="gelu"), name="linear token"),
        # the up projection of a training step, its pre-activation kept for the backward pass
        dict(_linear("bf16", 8192, 1024, 4096, act="gelu"), name="linear forward gelu"),
        # its gradients
        dict(_linear("bf16", 8192, 1024, 4096, act="gelu", grad=True), name="linear backward gelu"),
        # the down projection of Gemma-3's gated layer into the residual stream, W stored [out, in]
        dict(_linear("bf16", 4096, 6912, 1152, residual=True, w_out_in=True), name="linear down residual"),
        # the qkv projection of a packed batch in fp32, GPT-2 small
        dict(_linear("f32", 1021, 768, 2304, grad=True), name="linear backward f32"),
        # a decoding step that reports its 20 best alternatives, Gemma's vocabulary
        dict(_tokens("bf16", 1, 262144, top=20), name="tokens decode"),
        # scoring of 2 x 1024 given tokens with five alternatives each, GPT-2's vocabulary
        dict(_tokens("f32", 2048, 50257, top=5), name="tokens score"),
        # the gradient of a policy objective with an entropy bonus
        dict(_tokens("bf16", 1000, 262144, grad=True), name="tokens backward"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind, grad, dtype = rng.choice(["norm", "linear", "tokens"]), rng.random() < 0.5, rng.choice(["f32", "bf16"])
    if kind == "norm":
        D = _log(rng, 64, 8192)
        return _norm(dtype, _log(rng, 1, max(2, (1 << 24) // D)), D, grad)
    if kind == "linear":
        n_in, n_out = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.6:  # most layers' widths are multiples of 64
            n_in, n_out = (n_in + 63) // 64 * 64, (n_out + 63) // 64 * 64
        N = _log(rng, 1, max(2, min(8192, (1 << 34) // (n_in * n_out))))
        return _linear(dtype, N, n_in, n_out, rng.choice(["none", "gelu", "silu", "relu"]),
                       rng.random() < 0.4 and not grad, rng.random() < 0.5, grad)
    V = _log(rng, 1000, 262144)
    return _tokens(dtype, _log(rng, 1, max(2, (1 << 26) // V)), V, 0 if grad else rng.choice([0, 1, 5, 20]), grad)


# ------------------------------------------------------------------- prepare
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(c, seed):
    """The call's tensors by name."""
    g, t = _gen(seed), DT[c["dtype"]]

    def randn(*shape, sigma=1.0):
        return sigma * torch.randn(*shape, device="cuda", generator=g)

    if c["kind"] == "norm":
        N, D = c["N"], c["D"]
        # a residual stream: rows of different size, a few channels far above the others
        x = randn(N, D) * (0.5 + torch.rand(N, 1, device="cuda", generator=g)) + randn(D, sigma=0.3)
        x[:, :: max(1, D // 5)] *= 6.0
        s = dict(x=x.to(t), weight=1.0 + randn(D, sigma=0.2), bias=randn(D, sigma=0.1))
        if c["grad"]:
            mean = s["x"].double().mean(1)
            var = s["x"].double().var(1, unbiased=False)
            s.update(mean=mean.float(), rstd=(1.0 / torch.sqrt(var + EPS)).float(), dy=randn(N, D, sigma=0.1).to(t))
        return s
    if c["kind"] == "linear":
        N, n_in, n_out = c["N"], c["n_in"], c["n_out"]
        x, w = randn(N, n_in).to(t), randn(n_in, n_out, sigma=n_in ** -0.5).to(t)
        s = dict(x=x, W=w.t().contiguous() if c["w_out_in"] else w, bias=randn(n_out, sigma=0.1), residual=None)
        if not c["grad"]:
            if c["residual"]:
                s["residual"] = randn(N, n_out).to(t)
            return s
        # what the forward pass has kept
        s["z"] = (x.float() @ w.float() + s["bias"]).to(t) if c["act"] != "none" else None
        s["dy"] = randn(N, n_out, sigma=0.1).to(t)
        return s
    N, V = c["N"], c["V"]
    # logits of a language model: a wide bulk, a row's own sharpness, and some entries that a sampler has excluded
    z = randn(N, V, sigma=2.0) * (0.7 + 0.6 * torch.rand(N, 1, device="cuda", generator=g))
    z[:, :: max(2, V // 7)] = -math.inf
    tokens = 1 + torch.randint(0, V // 7 - 2, (N,), device="cuda", generator=g, dtype=torch.int32)
    if N > 4:
        tokens[::10] = IGNORE  # prompt tokens
    s = dict(logits=z.to(t), tokens=tokens)
    if c["grad"]:
        zd = s["logits"].double()
        m = zd.max(1).values
        log_s = (zd - m[:, None]).exp_().sum(1).log()
        q = zd - (m + log_s)[:, None]
        p = q.exp()
        entropy = -(p * q.clamp(min=-1e300)).sum(1)
        skip = tokens == IGNORE
        s.update(stats=torch.stack([m, log_s], 1).masked_fill(skip[:, None], 0.0).float(),
                 entropy=entropy.masked_fill(skip, 0.0).float(), grad_logprob=randn(N), grad_entropy=randn(N, sigma=0.1))
    return s


def prepare(case, seed):
    return dict(case=dict(case), **_inputs(case, seed))


# ----------------------------------------------------------------------- run
_ACT = {"none": "none", "gelu": "gelu_tanh", "silu": "silu", "relu": "relu"}
_GELU_C, _GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(_GELU_C * (z + _GELU_A * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return torch.where(z > 0, z, torch.zeros_like(z)) if act == "relu" else z


def _dact(z, act):
    if act == "gelu":
        th = torch.tanh(_GELU_C * (z + _GELU_A * z * z * z))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * _GELU_C * (1.0 + 3.0 * _GELU_A * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return (z > 0).float()


def _plain_norm(s, c):
    t, x = s["x"].dtype, s["x"].float()
    if not c["grad"]:
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        return ((d * rstd) * s["weight"] + s["bias"]).to(t), mean[:, 0], rstd[:, 0]
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(t), (dy * xhat).sum(0), dy.sum(0)


def _plain_linear(s, c):
    t, x = s["x"].dtype, s["x"].float()
    w = s["W"].float().t() if c["w_out_in"] else s["W"].float()
    if not c["grad"]:
        z = x @ w + s["bias"]
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(t), z.to(t)) if c["act"] != "none" else (y.to(t),)
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _dact(s["z"].float(), c["act"])
    dw = dz.t() @ x if c["w_out_in"] else x.t() @ dz
    return (dz @ w.t()).to(t), dw.to(t), dz.sum(0)


def _plain_tokens(s, c):
    z, tok = s["logits"].float(), s["tokens"].long()
    on = tok != IGNORE
    at = torch.where(on, tok, torch.zeros_like(tok))[:, None]
    if not c["grad"]:
        m = z.max(1, keepdim=True).values
        d = z - m
        e = torch.exp(d)
        total = e.sum(1)
        log_s = torch.log(total)
        mean_d = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / total
        zero = torch.zeros_like(log_s)
        out = [torch.where(on, d.gather(1, at)[:, 0] - log_s, zero), torch.where(on, log_s - mean_d, zero)]
        if c["top"]:
            # equal logits in the order of their indices
            ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : c["top"]]
            best = d.gather(1, ids) - log_s[:, None]
            out += [torch.where(on[:, None], best, torch.full_like(best, -math.inf)),
                    torch.where(on[:, None], ids, torch.full_like(ids, -1)).int()]
        return tuple(out)
    logp = (z - s["stats"][:, :1]) - s["stats"][:, 1:]
    p = torch.exp(logp)
    gl, ge = s["grad_logprob"][:, None], s["grad_entropy"][:, None]
    g = -gl * p - ge * torch.where(p > 0, p * (logp + s["entropy"][:, None]), torch.zeros_like(p))
    g.scatter_add_(1, at, gl)
    return (torch.where(on[:, None], g, torch.zeros_like(g)).to(s["logits"].dtype),)


_package = None


def _ops():
    global _package
    if _package is None:
        from mobilefinetuner_amd import layer_norm, linear, logprobs
        _package = layer_norm, linear, logprobs
    return _package


def _own(s, c):
    layer_norm, linear, logprobs = _ops()
    if c["kind"] == "norm":
        if not c["grad"]:
            return layer_norm.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        return layer_norm.layer_norm_backward(s["x"], s["weight"], s["mean"], s["rstd"], s["dy"])
    if c["kind"] == "linear":
        act = _ACT[c["act"]]
        if not c["grad"]:
            y, z = linear.linear(s["x"], s["W"], s["bias"], act, s["residual"], w_transposed=c["w_out_in"],
                                 want_preact=act != "none")
            return (y,) if z is None else (y, z)
        return linear.linear_backward(s["x"], s["W"], s["z"], s["dy"], act, w_transposed=c["w_out_in"])
    if not c["grad"]:
        logprob, entropy, _, best, ids = logprobs.token_logprobs(s["logits"], s["tokens"], c["top"], IGNORE,
                                                                 check_tokens=False)
        return (logprob, entropy, best, ids) if c["top"] else (logprob, entropy)
    return (logprobs.token_logprobs_backward(s["logits"], s["tokens"], s["stats"], s["entropy"], s["grad_logprob"],
                                             s["grad_entropy"], IGNORE),)


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"norm": _plain_norm, "linear": _plain_linear, "tokens": _plain_tokens}[c["kind"]](s, c)


# ---------------------------------------------------------------------- work
def work(c):
    e = SIZE[c["dtype"]]
    if c["kind"] == "norm":
        N, D = c["N"], c["D"]
        if c["grad"]:
            return {"bytes": 3 * N * D * e + 8 * N + 12 * D, "flops": 14 * N * D}
        return {"bytes": 2 * N * D * e + 8 * N + 8 * D, "flops": 8 * N * D}
    if c["kind"] == "linear":
        N, i, o = c["N"], c["n_in"], c["n_out"]
        kept = c["act"] != "none"
        if c["grad"]:  # x, W, dy and z in; dx, dW and the bias gradient out
            return {"bytes": e * (2 * N * i + 2 * i * o + N * o * (1 + kept)) + 4 * o, "flops": 4 * N * i * o}
        return {"bytes": e * (N * i + i * o + N * o * (1 + kept + c["residual"])) + 4 * o, "flops": 2 * N * i * o}
    N, V = c["N"], c["V"]
    live = N - (-(-N // 10) if N > 4 else 0)  # rows that are not ignored
    if c["grad"]:
        return {"bytes": (live + N) * V * e + 24 * N, "flops": 8 * live * V}
    return {"bytes": live * V * e + N * (12 + 8 * c["top"]), "flops": 6 * live * V}


# --------------------------------------------------------------------- exact
def exact(c, seed):
    s = _inputs(c, seed)
    up = {k: v.double() for k, v in s.items() if v is not None and v.is_floating_point()}
    F = torch.nn.functional
    if c["kind"] == "norm":
        x = up["x"]
        if not c["grad"]:
            var, mean = torch.var_mean(x, dim=1, unbiased=False)
            return F.layer_norm(x, (c["D"],), up["weight"], up["bias"], EPS), mean, torch.rsqrt(var + EPS)
        # the statistics are inputs of this call: the formula on the given ones
        h = torch.addcmul(-up["mean"] * up["rstd"], x.t(), up["rstd"]).t()
        g = up["dy"] * up["weight"]
        c1, c2 = g.sum(1) / c["D"], torch.einsum("nd,nd->n", g, h) / c["D"]
        return ((g - c1[:, None] - h * c2[:, None]) * up["rstd"][:, None], torch.einsum("nd,nd->d", up["dy"], h),
                up["dy"].sum(0))
    if c["kind"] == "linear":
        act = {"none": lambda v: v, "gelu": lambda v: F.gelu(v, approximate="tanh"), "silu": F.silu,
               "relu": F.relu}[c["act"]]
        w = up["W"] if c["w_out_in"] else up["W"].t()  # [out, in]
        if not c["grad"]:
            z = F.linear(up["x"], w, up["bias"])
            y = act(z) + (up["residual"] if c["residual"] else 0.0)
            return (y, z) if c["act"] != "none" else (y,)
        dz = up["dy"]
        if c["act"] != "none":
            z = up["z"].requires_grad_(True)
            dz, = torch.autograd.grad(act(z), z, up["dy"])
        dw = torch.mm(dz.t(), up["x"])
        return torch.mm(dz, w), dw if c["w_out_in"] else dw.t(), dz.sum(0)
    tok, on = s["tokens"].long(), s["tokens"] != IGNORE
    best, ids, out = [], [], []
    for lo in range(0, c["N"], 256):  # a part of the rows at a time: a row is a vocabulary of doubles
        rows = slice(lo, lo + 256)
        z, live = up["logits"][rows], on[rows]
        q = torch.log_softmax(z, 1)
        if c["grad"]:
            q = z - up["stats"][rows].sum(1, keepdim=True)
            p = q.exp()
            g = -p * (up["grad_logprob"][rows, None] + up["grad_entropy"][rows, None]
                      * (q.clamp(min=-1e30) + up["entropy"][rows, None]))
            n = torch.arange(len(z), device=z.device)[live]
            g[n, tok[rows][live]] += up["grad_logprob"][rows][live]
            g[~live] = 0.0
            out.append(g)
            continue
        logp = q.gather(1, tok[rows].clamp(min=0)[:, None])[:, 0]
        pair = torch.stack([logp, torch.special.entr(q.exp()).sum(1)], 1)
        pair[~live] = 0.0
        out.append(pair)
        if c["top"]:
            v = torch.topk(q, c["top"], dim=1).values
            v[~live] = -math.inf
            best.append(v)
    if c["grad"]:
        return (torch.cat(out),)
    out = torch.cat(out)
    return (out[:, 0], out[:, 1]) + ((torch.cat(best), None) if c["top"] else ())
