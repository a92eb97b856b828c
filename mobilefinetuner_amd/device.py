"""What the torch helpers share: checks of operands, the device and stream a
call is enqueued on, and workspaces.

A call runs on the device of its first operand, whichever is current, and on
torch's current stream of that device.  Outputs and workspaces are torch
tensors allocated under that stream, so the caching allocator hands their
memory out again only in its order.
"""
from __future__ import annotations

import contextlib
import functools

import torch

from . import capi

DTYPES = {torch.float32: capi.MFT_F32, torch.bfloat16: capi.MFT_BF16}
_HERE = contextlib.nullcontext()
# The handle without a Stream object around it (0.1 us a call for 2).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def guard(t):
    """Makes t's device current for a `with` block."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def stream(t):
    if _raw_stream is not None:
        return _raw_stream(t.get_device())
    return torch.cuda.current_stream(t.device).cuda_stream


def like(t):
    """A new contiguous tensor of t's shape and type (empty_like costs half of empty)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def ptr(t):
    return None if t is None else t.data_ptr()


def operand(t, name, like=None, dtype=None, shape=None):
    """t, checked: on the GPU (`like`'s, if given), of `dtype` and `shape` (a tuple) where they are given."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (there is no CPU path)")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, the call on {like.device}")
    if dtype is None:
        if t.dtype not in DTYPES:
            raise ValueError(f"{name}: unsupported dtype {t.dtype}")
    elif t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t


def optional(t, name, like, dtype, shape):
    """A contiguous operand that may be None."""
    return None if t is None else operand(t, name, like, dtype, shape).contiguous()


def rows(t, last):
    """t [..., last] as [N, last] with one stride between rows: a view where its
    strides allow, else a copy."""
    if t.dim() != 2:
        t = t.view(-1, last) if t.is_contiguous() else t.reshape(-1, last)
    if t.stride(1) == 1 or last == 1:
        if t.stride(0) >= last:
            return t
        if t.shape[0] <= 1:
            return t.as_strided(t.shape, (last, 1))
    return t.contiguous()


def workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


class _NoSecondDerivative(torch.autograd.Function):
    """The first `n` tensors, gradients that kernels have computed, as functions of the others, whose derivative raises."""

    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        ctx.mark_dirty(*tensors[:n])
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name}: its gradients have no derivative (no second order)")


def first_order(backward):
    """Decorates the backward of a node whose gradients the kernels compute.  With create_graph they
    depend on the incoming gradients and on what the forward saved (and on ctx.also, where it
    is set), and a derivative through them raises rather than leaving these terms out.  A gradient handed
    on as it came in keeps its graph."""
    name = backward.__qualname__.split(".")[0]

    @functools.wraps(backward)
    def checked(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        of = [t for t in (*grads, *ctx.saved_tensors, getattr(ctx, "also", None)) if t is not None and t.requires_grad]
        own = [i for i, t in enumerate(out) if t is not None and not any(t is g for g in grads)]
        if not of or not own:
            return out
        out = list(out)
        for i, t in zip(own, _NoSecondDerivative.apply(name, len(own), *(out[i] for i in own), *of)):
            out[i] = t
        return tuple(out)

    return checked
