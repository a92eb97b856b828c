"""Layer norm over the last dimension on the GPU, forward and backward, over the
C ABI of include/mft/layer_norm.h.

x [..., D] is fp32 or bf16, with any strides between rows; weight and bias [D]
are fp32 (the trainable parameters), as are the row statistics and the
parameters' gradients.  y and dx have x's type.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import capi
from .device import DTYPES, first_order, guard, like, operand, optional, ptr, rows, stream, workspace


def _param(p, name, x):
    return optional(p, name, x, torch.float32, (x.shape[-1],))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias in x's type and shape,
    and the statistics (fp32, x's shape without its last dimension) for the
    backward.  weight and bias may be None (1 and 0)."""
    if operand(x, "x").dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x must be [..., D] with D > 0")
    D, x2 = x.shape[-1], rows(x, x.shape[-1])
    w, b = _param(weight, "weight", x), _param(bias, "bias", x)
    with guard(x):
        y = like(x)
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        d = capi.layer_norm_desc(x2.shape[0], D, DTYPES[x.dtype], eps, x2.stride(0))
        capi.layer_norm_fwd(d, x2.data_ptr(), ptr(w), ptr(b), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                            stream(x))
    return y, mean, rstd


def layer_norm_backward(x, weight, mean, rstd, dy, want_x=True, want_params=True):
    """(dx, dweight, dbias) from dy = dL/dy and the forward's statistics; None where
    not wanted.  dx has x's type and shape, the parameters' gradients are fp32 [D]."""
    if operand(x, "x").dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x must be [..., D] with D > 0")
    D, x2 = x.shape[-1], rows(x, x.shape[-1])
    g2 = rows(operand(dy, "dy", x, x.dtype, x.shape), D)
    w = _param(weight, "weight", x)
    mean = operand(mean, "mean", x, torch.float32, x.shape[:-1]).contiguous()
    rstd = operand(rstd, "rstd", x, torch.float32, x.shape[:-1]).contiguous()
    with guard(x):
        dx = like(x) if want_x else None
        dw = torch.empty(D, dtype=torch.float32, device=x.device) if want_params else None
        db = torch.empty_like(dw) if want_params else None
        d = capi.layer_norm_desc(x2.shape[0], D, DTYPES[x.dtype], 0.0, x2.stride(0), 0, g2.stride(0))
        ws = workspace(capi.layer_norm_workspace_size(d), x)
        capi.layer_norm_bwd(d, x2.data_ptr(), ptr(w), mean.data_ptr(), rstd.data_ptr(), g2.data_ptr(), ptr(dx),
                            ptr(dw), ptr(db), ptr(ws), stream(x))
    return dx, dw, db


class LayerNorm(torch.autograd.Function):
    """y = LayerNorm.apply(x, weight, bias, eps)."""

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        y, mean, rstd = layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(x, weight, mean, rstd, dy, need[0], need[1] or need[2])
        return dx, dw if need[1] else None, db if need[2] else None, None
