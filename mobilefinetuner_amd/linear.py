"""Linear layer with bias, activation and residual in its epilogue on the GPU,
forward and backward, over the C ABI of include/mft/linear.h.

  z = x W + bias,  y = act(z) + residual

x [..., in], W [in, out] or, with w_transposed, [out, in], residual and y
[..., out] are all fp32 or all bf16; bias [out] and its gradient are fp32.  act
is "none", "relu", "gelu_tanh" or "silu".  Operands that are not contiguous are
copied on every call: pass a weight stored [out, in] with w_transposed, not its
transposed view.  In bf16 the backward rounds dz = dy act'(z) to bf16 for both
products, with an activation.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import capi
from .device import DTYPES, first_order, guard, like, operand, ptr, stream, workspace

ACTIVATIONS = {"none": capi.MFT_ACT_NONE, "relu": capi.MFT_ACT_RELU, "gelu_tanh": capi.MFT_ACT_GELU_TANH,
               "silu": capi.MFT_ACT_SILU}


def _desc(x, W, activation, w_transposed):
    """(desc, lead, in, out) of x [*lead, in] and W."""
    if operand(x, "x").dim() < 1:
        raise ValueError("x must be [..., in]")
    if operand(W, "W", x, x.dtype).dim() != 2:
        raise ValueError("W must be 2-D")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    n_in = x.shape[-1]
    n_out, w_in = W.shape if w_transposed else (W.shape[1], W.shape[0])
    if w_in != n_in:
        raise ValueError(f"matmul dimension mismatch: x has {n_in} columns, W {w_in} "
                         f"({'[out, in]' if w_transposed else '[in, out]'})")
    lead = x.shape[:-1]
    return (capi.linear_desc(lead.numel(), n_in, n_out, DTYPES[x.dtype], w_transposed, ACTIVATIONS[activation]),
            lead, n_in, n_out)


def linear(x, W, bias=None, activation="none", residual=None, w_transposed=False, want_preact=False):
    """(y, z): y = act(x W + bias) + residual, and z = x W + bias, the backward's
    input with an activation (None unless want_preact)."""
    d, lead, _, n_out = _desc(x, W, activation, w_transposed)
    if want_preact and activation == "none":
        raise ValueError("the pre-activation is kept with an activation only")
    if bias is not None:
        bias = operand(bias, "bias", x, torch.float32, (n_out,)).contiguous()
    if residual is not None:
        residual = operand(residual, "residual", x, x.dtype, (*lead, n_out)).contiguous()
    with guard(x):
        xc, Wc = x.contiguous(), W.contiguous()
        y = torch.empty(*lead, n_out, dtype=x.dtype, device=x.device)
        z = torch.empty_like(y) if want_preact else None
        ws = workspace(capi.linear_fwd_workspace_size(d), x)
        capi.linear_fwd(d, xc.data_ptr(), Wc.data_ptr(), ptr(bias), ptr(residual), y.data_ptr(), ptr(z), ptr(ws),
                        stream(x))
    return y, z


def linear_backward(x, W, z, dy, activation="none", w_transposed=False, want_x=True, want_weight=True,
                    want_bias=True):
    """(dx, dW, dbias) from dy = dL/dy and, with an activation, the forward's z;
    None where not wanted.  dx and dW have x's type and x's and W's shapes, dbias
    is fp32 [out].  The residual's gradient is dy."""
    d, lead, _, n_out = _desc(x, W, activation, w_transposed)
    dy = operand(dy, "dy", x, x.dtype, (*lead, n_out)).contiguous()
    if activation != "none":
        z = operand(z, "z", x, x.dtype, (*lead, n_out)).contiguous()
    else:
        z = None
    with guard(x):
        xc, Wc = x.contiguous(), W.contiguous()
        dx = like(x) if want_x else None
        dW = like(W) if want_weight else None
        db = torch.empty(n_out, dtype=torch.float32, device=x.device) if want_bias else None
        ws = workspace(capi.linear_workspace_size(d)[1], x)
        capi.linear_bwd(d, xc.data_ptr(), Wc.data_ptr(), ptr(z), dy.data_ptr(), ptr(dx), ptr(dW), ptr(db), ptr(ws),
                        stream(x))
    return dx, dW, db


class Linear(torch.autograd.Function):
    """y = Linear.apply(x, W, bias, residual, activation, w_transposed)."""

    @classmethod
    def apply(cls, x, W, bias=None, residual=None, activation="none", w_transposed=False):
        # Whether a backward can follow is seen here alone: needs_input_grad is the leaves', also under no_grad.
        return super().apply(x, W, bias, residual, activation, w_transposed, torch.is_grad_enabled())

    @staticmethod
    def forward(ctx, x, W, bias, residual, activation, w_transposed, grad_mode):
        need = ctx.needs_input_grad
        y, z = linear(x, W, bias, activation, residual, w_transposed,
                      grad_mode and activation != "none" and (need[0] or need[1] or need[2]))
        ctx.save_for_backward(x, W, z)
        ctx.also = bias if z is not None else None  # z is a function of it, too
        ctx.cfg = (activation, w_transposed)
        return y

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, W, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dW = db = None
        if need[0] or need[1] or need[2]:
            dx, dW, db = linear_backward(x, W, z, dy, *ctx.cfg, want_x=need[0], want_weight=need[1],
                                         want_bias=need[2])
        return dx, dW, db, dy if need[3] else None, None, None, None
