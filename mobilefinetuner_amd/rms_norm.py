"""Root-mean-square norm of a residual stream on the GPU, with the addition in front
of it, in the stream's type or in 8 bits, and its gradients, over the C ABI of
include/mft/rms_norm.h.

x, residual [..., D] are fp32 or bf16, with any strides between rows; weight [D]
is fp32 (the trainable parameter), as are rstd, the scales and the weight's
gradient.  norm "gemma" multiplies by 1 + weight (ops::rms_norm), "affine" by
weight (ops::rms_norm_affine).  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import capi
from .device import DTYPES, first_order, guard, like, operand, optional, ptr, rows, stream, workspace

NORMS = {"gemma": capi.MFT_NORM_GEMMA, "affine": capi.MFT_NORM_AFFINE}


def _norm(norm):
    if norm not in NORMS:
        raise ValueError(f"norm must be one of {sorted(NORMS)}, got {norm!r}")
    return NORMS[norm]


def _stream(x, residual):
    """(D, x's rows, the residual's rows or None)."""
    if operand(x, "x").dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x must be [..., D] with D > 0")
    D = x.shape[-1]
    return D, rows(x, D), None if residual is None else rows(operand(residual, "residual", x, x.dtype, x.shape), D)


def rms_norm(x, weight=None, residual=None, norm="gemma", eps=1e-6):
    """(y, total, rstd): total = x + residual in x's type (None without residual),
    y = total * rstd * f in x's type and shape with f = 1 + weight ("gemma") or
    weight ("affine") (1 without weight), and rstd (fp32, x's shape without its
    last dimension) for the backward."""
    how = _norm(norm)
    D, x2, r2 = _stream(x, residual)
    w = optional(weight, "weight", x, torch.float32, (D,))
    with guard(x):
        y = like(x)
        total = None if r2 is None else like(x)
        rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
        d = capi.rms_norm_desc(x2.shape[0], D, DTYPES[x.dtype], how, eps, x2.stride(0),
                               0 if r2 is None else r2.stride(0))
        capi.rms_norm_fwd(d, x2.data_ptr(), ptr(r2), ptr(w), ptr(total), y.data_ptr(), rstd.data_ptr(), stream(x))
    return y, total, rstd


def _e4m3(x, weight, residual, how, eps):
    D, x2, r2 = _stream(x, residual)
    w = optional(weight, "weight", x, torch.float32, (D,))
    with guard(x):
        q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
        total = None if r2 is None else like(x)
        scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
        d = capi.rms_norm_desc(x2.shape[0], D, DTYPES[x.dtype], how, eps, x2.stride(0),
                               0 if r2 is None else r2.stride(0))
        capi.rms_norm_e4m3_fwd(d, x2.data_ptr(), ptr(r2), ptr(w), ptr(total), q.data_ptr(), scale.data_ptr(),
                               stream(x))
    return q, scale, total


def rms_norm_e4m3(x, weight=None, residual=None, norm="gemma", eps=1e-6):
    """(q, scale, total): rms_norm's y, before any rounding, as e4m3 numbers (x's
    shape, torch.float8_e4m3fn) with one fp32 scale a row, y = q * scale: the largest
    |y| of a row becomes 448.  What gated_linear_e4m3 takes."""
    return _e4m3(x, weight, residual, _norm(norm), eps)


def quantize_rows(x):
    """(q, scale): x itself [..., D] as e4m3 numbers with one fp32 scale a row, as
    rms_norm_e4m3 holds y.  For weights, stored [out, in]."""
    return _e4m3(x, None, None, capi.MFT_NORM_NONE, 0.0)[:2]


def rms_norm_backward(x, weight, rstd, dy, dtotal=None, norm="gemma", want_x=True, want_weight=True):
    """(dx, dweight) from dy = dL/dy and the forward's rstd; x is the forward's total,
    or its x without a residual.  dtotal, what reaches the total from the stream
    behind it, is added to dx, the gradient of x and of the residual.  None where
    not wanted; dx has x's type and shape, dweight is fp32 [D]."""
    how = _norm(norm)
    D, x2, _ = _stream(x, None)
    g2 = rows(operand(dy, "dy", x, x.dtype, x.shape), D)
    t2 = None if dtotal is None else rows(operand(dtotal, "dtotal", x, x.dtype, x.shape), D)
    w = optional(weight, "weight", x, torch.float32, (D,))
    rstd = operand(rstd, "rstd", x, torch.float32, x.shape[:-1]).contiguous()
    with guard(x):
        dx = like(x) if want_x else None
        dw = x.new_empty(D, dtype=torch.float32) if want_weight else None
        d = capi.rms_norm_desc(x2.shape[0], D, DTYPES[x.dtype], how, 0.0, x2.stride(0), 0, g2.stride(0),
                               0 if t2 is None else t2.stride(0))
        ws = workspace(capi.rms_norm_workspace_size(d), x)
        capi.rms_norm_bwd(d, x2.data_ptr(), ptr(w), rstd.data_ptr(), g2.data_ptr(), ptr(t2), ptr(dx), ptr(dw), ptr(ws),
                          stream(x))
    return dx, dw


class RMSNorm(torch.autograd.Function):
    """y = RMSNorm.apply(x, weight, norm, eps)."""

    @staticmethod
    def forward(ctx, x, weight=None, norm="gemma", eps=1e-6):
        y, _, rstd = rms_norm(x, weight, None, norm, eps)
        ctx.save_for_backward(x, weight, rstd)
        ctx.norm = norm
        return y

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw = rms_norm_backward(x, weight, rstd, dy, None, ctx.norm, need[0], need[1])
        return dx, dw, None, None


class AddRMSNorm(torch.autograd.Function):
    """y, total = AddRMSNorm.apply(x, residual, weight, norm, eps): the stream that goes
    on past a block is total."""

    @staticmethod
    def forward(ctx, x, residual, weight=None, norm="gemma", eps=1e-6):
        y, total, rstd = rms_norm(x, weight, residual, norm, eps)
        ctx.save_for_backward(total, weight, rstd)
        ctx.norm = norm
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @first_order
    def backward(ctx, dy, dtotal):
        total, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None:
            return dtotal, dtotal, None, None, None
        dx, dw = rms_norm_backward(total, weight, rstd, dy, dtotal, ctx.norm, need[0] or need[1], need[2])
        return dx if need[0] else None, dx if need[1] else None, dw, None, None
