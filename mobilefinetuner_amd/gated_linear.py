"""Gated linear layer on the GPU, the first half of a gated feed-forward block, forward
and backward, over the C ABI of include/mft/gated_linear.h.

  gate = x W_gate,  up = x W_up,  h = act(gate) * up

x [..., in], W_gate and W_up [in, ff] or, with w_transposed, [ff, in], and h, gate and
up [..., ff] are all fp32 or all bf16.  act is "relu", "gelu_tanh" or "silu".
Operands that are not contiguous are copied on every call.  In bf16 the backward
rounds the gradients of gate and up to bf16 for the products.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import capi
from .device import DTYPES, first_order, guard, like, operand, ptr, stream, workspace

ACTIVATIONS = {"relu": capi.MFT_ACT_RELU, "gelu_tanh": capi.MFT_ACT_GELU_TANH, "silu": capi.MFT_ACT_SILU}


def _desc(x, W_gate, W_up, activation, w_transposed, dtype=None):
    """(desc, lead, ff) of x [*lead, in] and the weights."""
    if operand(x, "x", dtype=dtype).dim() < 1:
        raise ValueError("x must be [..., in]")
    if operand(W_gate, "W_gate", x, x.dtype).dim() != 2:
        raise ValueError("W_gate must be 2-D")
    operand(W_up, "W_up", x, x.dtype, W_gate.shape)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    n_in = x.shape[-1]
    n_ff, w_in = W_gate.shape if w_transposed else (W_gate.shape[1], W_gate.shape[0])
    if w_in != n_in:
        raise ValueError(f"matmul dimension mismatch: x has {n_in} columns, W_gate {w_in} "
                         f"({'[ff, in]' if w_transposed else '[in, ff]'})")
    lead = x.shape[:-1]
    return (capi.gated_linear_desc(lead.numel(), n_in, n_ff, DTYPES.get(x.dtype, capi.MFT_BF16), w_transposed,
                                   ACTIVATIONS[activation]), lead, n_ff)


def gated_linear(x, W_gate, W_up, activation="gelu_tanh", w_transposed=False, want_preact=False):
    """(h, gate, up): h = act(gate) * up, and gate = x W_gate and up = x W_up, the
    backward's inputs (None unless want_preact)."""
    d, lead, n_ff = _desc(x, W_gate, W_up, activation, w_transposed)
    with guard(x):
        xc, Wg, Wu = x.contiguous(), W_gate.contiguous(), W_up.contiguous()
        h = x.new_empty((*lead, n_ff))
        gate, up = (torch.empty_like(h), torch.empty_like(h)) if want_preact else (None, None)
        ws = workspace(capi.gated_linear_fwd_workspace_size(d), x)
        capi.gated_linear_fwd(d, xc.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), h.data_ptr(), ptr(gate), ptr(up), ptr(ws),
                              stream(x))
    return h, gate, up


def gated_linear_e4m3(x, x_scale, W_gate, gate_scale, W_up, up_scale, activation="gelu_tanh"):
    """h [..., ff] in bf16 from e4m3 numbers: x [..., in] with its rows' fp32 scales [...]
    (rms_norm_e4m3), W_gate and W_up [ff, in] with theirs [ff] (quantize_rows)."""
    d, lead, n_ff = _desc(x, W_gate, W_up, activation, True, torch.float8_e4m3fn)
    scales = [operand(s, n, x, torch.float32, shape).contiguous()
              for s, n, shape in ((x_scale, "x_scale", lead), (gate_scale, "gate_scale", (n_ff,)),
                                  (up_scale, "up_scale", (n_ff,)))]
    with guard(x):
        xc, Wg, Wu = x.contiguous(), W_gate.contiguous(), W_up.contiguous()
        h = x.new_empty((*lead, n_ff), dtype=torch.bfloat16)
        ws = workspace(capi.gated_linear_e4m3_workspace_size(d), x)
        capi.gated_linear_e4m3_fwd(d, xc.data_ptr(), scales[0].data_ptr(), Wg.data_ptr(), scales[1].data_ptr(),
                                   Wu.data_ptr(), scales[2].data_ptr(), h.data_ptr(), ptr(ws), stream(x))
    return h


def gated_linear_backward(x, W_gate, W_up, gate, up, dh, activation="gelu_tanh", w_transposed=False, want_x=True,
                          want_gate=True, want_up=True):
    """(dx, dW_gate, dW_up) from dh = dL/dh and the forward's gate and up; None where
    not wanted.  They have x's type, and x's and the weights' shapes."""
    d, lead, n_ff = _desc(x, W_gate, W_up, activation, w_transposed)
    gate, up, dh = (operand(t, n, x, x.dtype, (*lead, n_ff)).contiguous()
                    for t, n in ((gate, "gate"), (up, "up"), (dh, "dh")))
    with guard(x):
        xc, Wg, Wu = x.contiguous(), W_gate.contiguous(), W_up.contiguous()
        dx = like(x) if want_x else None
        dWg, dWu = like(W_gate) if want_gate else None, like(W_up) if want_up else None
        ws = workspace(capi.gated_linear_workspace_size(d)[1], x)
        capi.gated_linear_bwd(d, xc.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), gate.data_ptr(), up.data_ptr(),
                              dh.data_ptr(), ptr(dx), ptr(dWg), ptr(dWu), ptr(ws), stream(x))
    return dx, dWg, dWu


class GatedLinear(torch.autograd.Function):
    """h = GatedLinear.apply(x, W_gate, W_up, activation, w_transposed)."""

    @classmethod
    def apply(cls, x, W_gate, W_up, activation="gelu_tanh", w_transposed=False):
        # Whether a backward can follow is seen here alone: needs_input_grad is the leaves', also under no_grad.
        return super().apply(x, W_gate, W_up, activation, w_transposed, torch.is_grad_enabled())

    @staticmethod
    def forward(ctx, x, W_gate, W_up, activation, w_transposed, grad_mode):
        h, gate, up = gated_linear(x, W_gate, W_up, activation, w_transposed,
                                   grad_mode and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, W_gate, W_up, gate, up)
        ctx.cfg = (activation, w_transposed)
        return h

    @staticmethod
    @first_order
    def backward(ctx, dh):
        need = ctx.needs_input_grad
        return (*gated_linear_backward(*ctx.saved_tensors, dh, *ctx.cfg, *need[:3]), None, None, None)
