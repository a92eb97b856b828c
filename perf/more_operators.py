"""The gated half of a transformer block and the step that trains it, as cases that can be timed.

  norm   root-mean-square norm of a residual stream with the addition in front of it, in the stream's
         type or in 8 bits (e4m3) with one scale a row, and its gradients
  gated  act(x W_gate) * (x W_up), the first half of a gated feed-forward block, and its gradients; with
         operands in e4m3 and a scale a row, too
  adamw  one AdamW step over a list of parameters, gradients clipped by their global norm, with states in
         fp32 or in 8 bits (e4m3, a scale for each 256 values)

A case is one call of one of them.  With `own` false it is computed in plain torch operations in 32 bits;
with `own` true by the package's operator.

Activations, weights of products and their gradients have the case's type; a norm's weight and its
gradient are fp32.  A parameter in bf16 is stepped on its fp32 master copy.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}
TOP = 448.0          # the largest e4m3 number
LEAST = 2.0 ** -9    # the smallest
TINY = 2.0 ** -126   # a scale's lower bound
GROUP = 256          # values of an 8-bit state with one scale
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01


# --------------------------------------------------------------------- cases
def _norm(dtype, N, D, residual=True, out="same", grad=False):
    return dict(kind="norm", dtype=dtype, N=N, D=D, residual=residual, out=out, grad=grad)


def _gated(dtype, N, n_in, n_ff, act="gelu", w_out_in=True, grad=False, keep=False):
    return dict(kind="gated", dtype=dtype, N=N, n_in=n_in, n_ff=n_ff, act=act, w_out_in=w_out_in, grad=grad, keep=keep)


def _adamw(dtype, bits, count, total, clip=True, of="sizes"):
    return dict(kind="adamw", dtype=dtype, bits=bits, count=count, total=total, clip=clip, of=of)


# a LoRA adapter of rank 8 on q, k, v and o of each of Gemma-3-1B's 26 layers: (in + out) * 8 values each
_LORA = [s for i, o in ((1152, 1024), (1152, 256), (1152, 256), (1024, 1152)) for s in (8 * i, 8 * o)] * 26
# a block of Gemma-3-1B: q, k, v, o, gate, up, down, its four norms of the stream and two of the heads
_BLOCK = [1152 * 1024, 1152 * 256, 1152 * 256, 1024 * 1152, 1152 * 6912, 1152 * 6912, 6912 * 1152, 1152, 1152, 1152,
          1152, 256, 256]


def listed():
    return [
        # the addition and the norm in front of a block for a single generated token, Gemma-3-1B: latency
        dict(_norm("bf16", 1, 1152), name="norm token"),
        # the same of 8 x 1024 prompt tokens, in 8 bits for the products behind it
        dict(_norm("bf16", 8192, 1152, out="e4m3"), name="norm forward e4m3"),
        # a training step's backward pass of 16 x 1024 tokens, the residual stream's gradient added
        dict(_norm("bf16", 16384, 1152, grad=True), name="norm backward bf16"),
        # a ragged batch in fp32, packed to its valid tokens, and a width off every vector boundary
        dict(_norm("f32", 1001, 1153, grad=True), name="norm backward ragged"),
        # gate and up of a single generated token, Gemma-3-1B: every weight is read once
        dict(_gated("bf16", 1, 1152, 6912), name="gated token"),
        # gate and up of a training step of 8 x 1024 tokens, both kept for the backward pass
        dict(_gated("bf16", 8192, 1152, 6912, keep=True), name="gated forward"),
        # their gradients for 4 x 1024 tokens
        dict(_gated("bf16", 4096, 1152, 6912, w_out_in=False, grad=True), name="gated backward"),
        # the gradients of a packed batch in fp32, Gemma-3-270M
        dict(_gated("f32", 509, 640, 2048, grad=True), name="gated backward f32"),
        # a prompt of 4096 tokens through weights held in 8 bits
        dict(_gated("e4m3", 4096, 1152, 6912), name="gated forward e4m3"),
        # the step of a LoRA adapter of rank 8: 208 small tensors
        dict(_adamw("f32", 32, len(_LORA), sum(_LORA), of="lora"), name="adamw lora"),
        # the step of a block in fp32 with all its states
        dict(_adamw("f32", 32, len(_BLOCK), sum(_BLOCK), of="block"), name="adamw block"),
        # the step of Gemma-3-270M's embedding table in bf16, its states in 8 bits
        dict(_adamw("bf16", 8, 1, 262144 * 640, clip=False, of="table"), name="adamw table 8 bit"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "gated", "adamw"])
    if kind == "norm":
        D = _log(rng, 64, 8192)
        N, dtype, residual = _log(rng, 1, max(2, (1 << 24) // D)), rng.choice(["f32", "bf16"]), rng.random() < 0.7
        if rng.random() < 0.4:
            return _norm(dtype, N, D, residual, grad=True)
        return _norm(dtype, N, D, residual, rng.choice(["same", "e4m3"]))
    if kind == "gated":
        n_in, n_ff, dtype = _log(rng, 64, 4096), _log(rng, 64, 8192), rng.choice(["f32", "bf16", "bf16", "e4m3"])
        if rng.random() < 0.6:  # most layers' widths are multiples of 64
            n_in, n_ff = (n_in + 63) // 64 * 64, (n_ff + 63) // 64 * 64
        N = _log(rng, 1, max(2, min(8192, (1 << 33) // (n_in * n_ff))))
        act = rng.choice(["gelu", "silu"])
        if dtype == "e4m3":
            return _gated(dtype, N, n_in, n_ff, act)
        grad = rng.random() < 0.5
        return _gated(dtype, N, n_in, n_ff, act, rng.random() < 0.5, grad, not grad and rng.random() < 0.5)
    count = _log(rng, 1, 300)
    return _adamw(rng.choice(["f32", "bf16"]), rng.choice([32, 8]), count, _log(rng, 4 * count, 1 << 26),
                  rng.random() < 0.5)


def _sizes(c):
    """Values of each parameter of an adamw case."""
    if c["of"] == "lora":
        return list(_LORA)
    if c["of"] == "block":
        return list(_BLOCK)
    if c["of"] == "table":
        return [c["total"]]
    r = random.Random(c["count"] * 1000003 + c["total"])
    cuts = sorted(r.sample(range(1, c["total"]), c["count"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [c["total"]])]


# ------------------------------------------------------------------- prepare
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _to_rows(x):
    """(e4m3 values, fp32 scale of each row) of a matrix."""
    scale = (x.abs().amax(1) / TOP).clamp(min=TINY)
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def _to_groups(x, positive):
    """(e4m3 values, fp32 scales) of a flat state; a positive value is not rounded to zero where `positive`."""
    g = x.view(-1, GROUP)
    scale = (g.abs().amax(1) / TOP).clamp(min=TINY)
    q = g / scale[:, None]
    if positive:
        q = torch.where(q > 0, q.clamp(min=LEAST), q)
    return q.to(torch.float8_e4m3fn).view(-1), scale


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
        s = dict(x=x.to(t), weight=randn(D, sigma=0.2), residual=None)
        if c["grad"]:
            total = s["x"].double()
            s.update(rstd=(1.0 / torch.sqrt((total * total).mean(1) + EPS)).float(), dy=randn(N, D, sigma=0.1).to(t),
                     dtotal=randn(N, D, sigma=0.1).to(t) if c["residual"] else None)
        elif c["residual"]:
            s["residual"] = randn(N, D).to(t)
        return s
    if c["kind"] == "gated":
        N, n_in, n_ff = c["N"], c["n_in"], c["n_ff"]
        x = randn(N, n_in)
        # rows of the weights: [out, in]
        wg, wu = randn(n_ff, n_in, sigma=n_in ** -0.5), randn(n_ff, n_in, sigma=n_in ** -0.5)
        if c["dtype"] == "e4m3":
            (x, xs), (wg, gs), (wu, us) = _to_rows(x), _to_rows(wg), _to_rows(wu)
            return dict(x=x, W_gate=wg, W_up=wu, x_scale=xs, gate_scale=gs, up_scale=us)
        x, wg, wu = x.to(t), wg.to(t), wu.to(t)
        s = dict(x=x, W_gate=wg if c["w_out_in"] else wg.t().contiguous(),
                 W_up=wu if c["w_out_in"] else wu.t().contiguous())
        if c["grad"]:  # what the forward pass has kept
            s.update(gate=(x.float() @ wg.float().t()).to(t), up=(x.float() @ wu.float().t()).to(t),
                     dh=randn(N, n_ff, sigma=0.1).to(t))
        return s
    sizes = _sizes(c)
    total, starts = sum(sizes), _starts(sizes)
    flat = starts[-1]
    master = randn(total, sigma=0.02)
    grad = randn(total, sigma=1e-3).to(t)
    # mid-training: averages of gradients of about this size, none for the values behind a tensor's end
    inside = torch.zeros(flat, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        inside[a : a + n] = True
    m = torch.where(inside, randn(flat, sigma=3e-4), torch.zeros((), device="cuda"))
    v = torch.where(inside, 1e-6 * (0.2 + torch.rand(flat, device="cuda", generator=g)), torch.zeros((), device="cuda"))
    s = dict(grad=grad, step=torch.full((), 100, dtype=torch.int64, device="cuda"))
    s["param"] = master if c["dtype"] == "f32" else master.to(t)
    if c["dtype"] != "f32":
        whole = torch.zeros(flat, device="cuda")
        for a, n, p in zip(starts, sizes, master.split(sizes)):
            whole[a : a + n] = p
        s["master"] = whole
    if c["bits"] == 32:
        s.update(exp_avg=m, exp_avg_sq=v)
    else:
        (s["exp_avg"], s["exp_avg_scale"]), (s["exp_avg_sq"], s["exp_avg_sq_scale"]) = _to_groups(m, False), _to_groups(v.sqrt(), True)
    return s


def _starts(sizes):
    """Where each parameter's states begin in the flat ones, and where the last ends: multiples of a group."""
    at = [0]
    for n in sizes:
        at.append(at[-1] + (n + GROUP - 1) // GROUP * GROUP)
    return at


def _parts(flat, sizes):
    return [flat[a : a + n] for a, n in zip(_starts(sizes), sizes)]


_STATES = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")


def prepare(case, seed):
    s = dict(case=dict(case), **_inputs(case, seed))
    if case["kind"] == "adamw":
        sizes = _sizes(case)
        # a program holds its parameters and gradients as tensors of their own; here they lie one behind the other
        s["params"], s["grads"] = list(s["param"].split(sizes)), list(s["grad"].split(sizes))
        if own:
            optimizer = _ops()[2].AdamW([p.requires_grad_(True) for p in s["params"]], lr=LR, betas=(BETA1, BETA2),
                                        eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"])
            for p, d in zip(s["params"], s["grads"]):
                p.grad = d
            for name, state in optimizer.state.items():
                state.copy_(s[name])
            s["optimizer"] = optimizer
        else:
            s["masters"] = s["params"] if "master" not in s else _parts(s["master"], sizes)
    return s


# ----------------------------------------------------------------------- run
_ACT = {"gelu": "gelu_tanh", "silu": "silu"}
_GELU_C, _GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(_GELU_C * (z + _GELU_A * z * z * z)))
    return z / (1.0 + torch.exp(-z))


def _dact(z, act):
    if act == "gelu":
        th = torch.tanh(_GELU_C * (z + _GELU_A * z * z * z))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * _GELU_C * (1.0 + 3.0 * _GELU_A * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_norm(s, c):
    t, factor = s["x"].dtype, 1.0 + s["weight"]
    if c["grad"]:
        h = s["x"].float() * s["rstd"][:, None]
        dy = s["dy"].float()
        g = dy * factor
        dx = s["rstd"][:, None] * (g - h * (g * h).mean(1, keepdim=True))
        if s["dtotal"] is not None:
            dx = dx + s["dtotal"].float()
        return {"dx": dx.to(t), "dweight": (dy * h).sum(0)}
    out = {}
    total = s["x"]
    if s["residual"] is not None:  # the stream is kept in its own type, and the norm is of what is kept
        total = out["total"] = (s["x"].float() + s["residual"].float()).to(t)
    x = total.float()
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    y = x * rstd * factor
    if c["out"] == "e4m3":
        out["y"], out["scale"] = _to_rows(y)
    else:
        out["y"], out["rstd"] = y.to(t), rstd[:, 0]
    return out


def _plain_gated(s, c):
    if c["dtype"] == "e4m3":
        x = s["x"].float() * s["x_scale"][:, None]
        gate = x @ (s["W_gate"].float() * s["gate_scale"][:, None]).t()
        up = x @ (s["W_up"].float() * s["up_scale"][:, None]).t()
        return {"h": (_act(gate, c["act"]) * up).bfloat16()}
    t, x = s["x"].dtype, s["x"].float()
    wg, wu = s["W_gate"].float(), s["W_up"].float()
    if c["w_out_in"]:
        wg, wu = wg.t(), wu.t()
    if not c["grad"]:
        gate, up = x @ wg, x @ wu
        out = {"h": (_act(gate, c["act"]) * up).to(t)}
        return {**out, "gate": gate.to(t), "up": up.to(t)} if c["keep"] else out
    gate, up, dh = s["gate"].float(), s["up"].float(), s["dh"].float()
    dgate, dup = dh * up * _dact(gate, c["act"]), dh * _act(gate, c["act"])
    dwg, dwu = x.t() @ dgate, x.t() @ dup
    if c["w_out_in"]:
        dwg, dwu = dwg.t(), dwu.t()
    return {"dx": (dgate @ wg.t() + dup @ wu.t()).to(t), "dW_gate": dwg.to(t), "dW_up": dwu.to(t)}


def _plain_adamw(s, c):
    sizes, out = _sizes(c), {}
    t = s["step"].add_(1).double()
    grads = [g.float() for g in s["grads"]]
    if c["clip"]:
        norm = torch.stack(torch._foreach_norm(grads, 2, dtype=torch.float64)).square().sum().sqrt()
        grads = torch._foreach_mul(grads, (1.0 / (norm + 1e-6)).clamp(max=1.0).float())
        out["norm"] = norm.float()
    m, v = s["exp_avg"], s["exp_avg_sq"]
    if c["bits"] == 8:
        m = (m.float().view(-1, GROUP) * s["exp_avg_scale"][:, None]).view(-1)
        v = (v.float().view(-1, GROUP) * s["exp_avg_sq_scale"][:, None]).square().view(-1)
    ms, vs = _parts(m, sizes), _parts(v, sizes)
    torch._foreach_mul_(ms, BETA1)
    torch._foreach_add_(ms, grads, alpha=1.0 - BETA1)
    torch._foreach_mul_(vs, BETA2)
    torch._foreach_addcmul_(vs, grads, grads, 1.0 - BETA2)
    under = torch._foreach_sqrt(vs)
    torch._foreach_mul_(under, (1.0 / torch.sqrt(1.0 - BETA2 ** t)).float())
    torch._foreach_add_(under, ADAM_EPS)
    change = torch._foreach_div(ms, under)
    torch._foreach_mul_(change, (LR / (1.0 - BETA1 ** t)).float())
    torch._foreach_mul_(s["masters"], 1.0 - LR * DECAY)
    torch._foreach_sub_(s["masters"], change)
    if c["dtype"] != "f32":
        torch._foreach_copy_(s["params"], s["masters"])
    if c["bits"] == 8:
        q, scale = _to_groups(m, False)
        s["exp_avg"].copy_(q)
        s["exp_avg_scale"].copy_(scale)
        q, scale = _to_groups(torch.sqrt(v), True)
        s["exp_avg_sq"].copy_(q)
        s["exp_avg_sq_scale"].copy_(scale)
    return {**out, "param": s["param"], "step": s["step"], **{n: s[n] for n in _STATES if n in s}}


_package = None


def _ops():
    global _package
    if _package is None:
        from mobilefinetuner_amd import adamw, gated_linear, rms_norm
        _package = rms_norm, gated_linear, adamw
    return _package


def _own(s, c):
    rms_norm, gated_linear, _ = _ops()
    if c["kind"] == "norm":
        if c["grad"]:
            dx, dweight = rms_norm.rms_norm_backward(s["x"], s["weight"], s["rstd"], s["dy"], s["dtotal"])
            return {"dx": dx, "dweight": dweight}
        if c["out"] == "e4m3":
            y, scale, total = rms_norm.rms_norm_e4m3(s["x"], s["weight"], s["residual"], eps=EPS)
            out = {"y": y, "scale": scale}
        else:
            y, total, rstd = rms_norm.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
            out = {"y": y, "rstd": rstd}
        return {**out, "total": total} if s["residual"] is not None else out
    if c["kind"] == "gated":
        act = _ACT[c["act"]]
        if c["dtype"] == "e4m3":
            return {"h": gated_linear.gated_linear_e4m3(s["x"], s["x_scale"], s["W_gate"], s["gate_scale"], s["W_up"],
                                                        s["up_scale"], act)}
        if c["grad"]:
            dx, dwg, dwu = gated_linear.gated_linear_backward(s["x"], s["W_gate"], s["W_up"], s["gate"], s["up"],
                                                              s["dh"], act, w_transposed=c["w_out_in"])
            return {"dx": dx, "dW_gate": dwg, "dW_up": dwu}
        h, gate, up = gated_linear.gated_linear(s["x"], s["W_gate"], s["W_up"], act, w_transposed=c["w_out_in"],
                                                want_preact=c["keep"])
        return {"h": h, "gate": gate, "up": up} if c["keep"] else {"h": h}
    optimizer = s["optimizer"]
    norm = optimizer.step(max_norm=1.0 if c["clip"] else None)
    out = {"param": s["param"].detach(), **optimizer.state}
    return {**out, "norm": norm} if c["clip"] else out


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"norm": _plain_norm, "gated": _plain_gated, "adamw": _plain_adamw}[c["kind"]](s, c)


# ---------------------------------------------------------------------- work
def work(c):
    e = SIZE[c["dtype"]]
    if c["kind"] == "norm":
        N, D, r = c["N"], c["D"], int(c["residual"])
        if c["grad"]:  # the stream, dy and the stream's gradient in; dx and the weight's gradient out
            return {"bytes": (3 + r) * N * D * e + 4 * N + 8 * D, "flops": 11 * N * D}
        # x and the residual in; the sum and y out
        return {"bytes": (1 + 2 * r) * N * D * e + N * D * (1 if c["out"] == "e4m3" else e) + 4 * N + 4 * D,
                "flops": 6 * N * D}
    if c["kind"] == "gated":
        N, i, f = c["N"], c["n_in"], c["n_ff"]
        if c["dtype"] == "e4m3":
            return {"bytes": N * i + 2 * i * f + 4 * (N + 2 * f) + 2 * N * f, "flops": 4 * N * i * f}
        if c["grad"]:  # x, both weights, gate, up and dh in; dx and both weights' gradients out
            return {"bytes": e * (2 * N * i + 4 * i * f + 3 * N * f), "flops": 8 * N * i * f}
        return {"bytes": e * (N * i + 2 * i * f + N * f * (3 if c["keep"] else 1)), "flops": 4 * N * i * f}
    n = c["total"]
    state = 16 if c["bits"] == 32 else 4 + 16 / GROUP  # both read and written
    param = 8 if c["dtype"] == "f32" else 8 + 2
    return {"bytes": n * (e + state + param), "flops": (16 if c["clip"] else 13) * n}


# --------------------------------------------------------------------- exact
def exact(c, seed):
    s = _inputs(c, seed)
    up = {k: v.double() for k, v in s.items() if v is not None and v.is_floating_point()}
    F = torch.nn.functional
    if c["kind"] == "norm":
        if c["grad"]:
            n = torch.arange(c["D"], device="cuda")
            scaled = up["x"] * up["rstd"].unsqueeze(1)
            back = up["dy"] + up["dy"] * up["weight"]
            along = torch.einsum("nd,nd->n", back, scaled) / len(n)
            dx = torch.addcmul(back, scaled, along.unsqueeze(1), value=-1.0) * up["rstd"].unsqueeze(1)
            return {"dx": dx if s["dtotal"] is None else dx + up["dtotal"],
                    "dweight": torch.einsum("nd,nd->d", up["dy"], scaled)}
        out, x = {}, up["x"]
        if c["residual"]:
            out["total"] = x + up["residual"]
            x = out["total"].to(s["x"].dtype).double()
        rstd = torch.rsqrt(x.pow(2).sum(1) / c["D"] + EPS)
        y = torch.einsum("nd,n->nd", x, rstd)
        y += y * up["weight"]
        if c["out"] == "e4m3":
            out["scale"] = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / TOP
            out["y"] = y / out["scale"].unsqueeze(1)  # before its rounding to 8 bits
        else:
            out.update(y=y, rstd=rstd)
        return out
    if c["kind"] == "gated":
        act = {"gelu": lambda v: F.gelu(v, approximate="tanh"), "silu": F.silu}[c["act"]]
        wg, wu = up["W_gate"], up["W_up"]
        if c["dtype"] == "e4m3":
            gate = torch.outer(up["x_scale"], up["gate_scale"]) * F.linear(up["x"], wg)
            return {"h": act(gate) * torch.outer(up["x_scale"], up["up_scale"]) * F.linear(up["x"], wu)}
        both = torch.cat([wg, wu], 0 if c["w_out_in"] else 1)
        both = both if c["w_out_in"] else both.t()  # [2 ff, in]
        if not c["grad"]:
            gate, rise = F.linear(up["x"], both).chunk(2, 1)
            return {"h": act(gate) * rise, **({"gate": gate, "up": rise} if c["keep"] else {})}
        leaves = [up["gate"].requires_grad_(True), up["up"].requires_grad_(True)]
        dz = torch.cat(torch.autograd.grad(act(leaves[0]) * leaves[1], leaves, up["dh"]), 1)
        dw = torch.mm(dz.t(), up["x"])
        dwg, dwu = dw.chunk(2, 0)
        return {"dx": torch.mm(dz, both), "dW_gate": dwg if c["w_out_in"] else dwg.t(),
                "dW_up": dwu if c["w_out_in"] else dwu.t()}
    sizes = _sizes(c)
    starts, t = _starts(sizes), 101
    at = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(starts, sizes)])  # values of the flat states
    g = torch.zeros(starts[-1], dtype=torch.float64, device="cuda")
    g[at] = up["grad"]
    out = {"step": s["step"] + 1}
    if c["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g *= min(1.0, 1.0 / (float(out["norm"]) + 1e-6))
    m, v = up["exp_avg"], up["exp_avg_sq"]
    if c["bits"] == 8:
        m = (m.view(-1, GROUP) * up["exp_avg_scale"].unsqueeze(1)).flatten()
        v = (v.view(-1, GROUP) * up["exp_avg_sq_scale"].unsqueeze(1)).flatten() ** 2
    m, v = torch.lerp(g, m, BETA1), torch.lerp(g * g, v, BETA2)
    p = torch.zeros_like(g)
    p[at] = up["param"]
    p = up["master"] if "master" in up else p
    p = p * (1.0 - LR * DECAY) - LR / (1.0 - BETA1 ** t) * m / ((v / (1.0 - BETA2 ** t)).sqrt() + ADAM_EPS)
    out["param"] = p[at]
    if "master" in s:
        out["master"] = p
    if c["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    for name, x in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):  # before their rounding to 8 bits
        scale = (torch.linalg.vector_norm(x.view(-1, GROUP), ord=math.inf, dim=1) / TOP).clamp(min=TINY)
        out[name], out[name + "_scale"] = (x.view(-1, GROUP) / scale.unsqueeze(1)).flatten(), scale
    return out
