"""Log probabilities of given tokens on the GPU, with each row's entropy and its
top alternatives, and their gradient, over the C ABI of include/mft/logprobs.h.

logits [..., V] are fp32 or bf16, with any strides between rows; tokens [...]
are int32, one to a row (no shift, unlike the language-model loss).  There is no
CPU path.
"""
from __future__ import annotations

import torch

from . import capi
from .device import DTYPES, first_order, guard, like, operand, optional, ptr, rows, stream, workspace


def _operands(logits, tokens):
    if operand(logits, "logits").dim() < 1 or logits.shape[-1] == 0:
        raise ValueError("logits must be [..., V] with V > 0")
    operand(tokens, "tokens", logits, torch.int32, logits.shape[:-1])
    return rows(logits, logits.shape[-1]), tokens.contiguous()


def token_logprobs(logits, tokens, top=0, ignore_index=-100, check_tokens=True):
    """(logprob, entropy, stats, top_logprobs, top_ids), fp32 but for top_ids (int32).
    logprob and entropy [...]; stats [..., 2] is kept for the backward;
    top_logprobs and top_ids [..., top] hold the largest log probabilities in
    falling order, equal ones in the order of their indices (None with top = 0).
    A row whose token is ignore_index is not read (0, 0, and -inf, -1 as its
    alternatives).  check_tokens synchronises and raises on a token outside
    [0, V); without it such a token's logprob is NaN."""
    z, t = _operands(logits, tokens)
    lead, V = logits.shape[:-1], logits.shape[-1]
    with guard(logits):
        dev = logits.device
        logprob = torch.empty(lead, dtype=torch.float32, device=dev)
        entropy = torch.empty_like(logprob)
        stats = torch.empty(*lead, 2, dtype=torch.float32, device=dev)
        best = torch.empty(*lead, top, dtype=torch.float32, device=dev) if top else None
        ids = torch.empty_like(best, dtype=torch.int32) if top else None
        status = torch.zeros(1, dtype=torch.int32, device=dev) if check_tokens else None
        d = capi.logprobs_desc(z.shape[0], V, z.stride(0), 0, DTYPES[z.dtype], ignore_index, top)
        ws = workspace(capi.logprobs_workspace_size(d), logits)
        capi.logprobs_fwd(d, z.data_ptr(), t.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                          ptr(best), ptr(ids), ptr(status), ptr(ws), stream(logits))
        if check_tokens and int(status.item()) != 0:
            raise ValueError("token_logprobs: token out of range")
    return logprob, entropy, stats, best, ids


def token_logprobs_backward(logits, tokens, stats, entropy, grad_logprob, grad_entropy=None, ignore_index=-100):
    """grad_logits, in logits' type and shape, from the gradients of logprob and
    entropy (each may be None) and the forward's stats and entropy.  Rows that
    are ignored or whose token is out of range get a zero gradient."""
    z, t = _operands(logits, tokens)
    lead = logits.shape[:-1]
    stats = operand(stats, "stats", logits, torch.float32, (*lead, 2)).contiguous()
    entropy = optional(entropy, "entropy", logits, torch.float32, lead)
    gl = optional(grad_logprob, "grad_logprob", logits, torch.float32, lead)
    ge = optional(grad_entropy, "grad_entropy", logits, torch.float32, lead)
    with guard(logits):
        g = like(logits)
        d = capi.logprobs_desc(z.shape[0], logits.shape[-1], z.stride(0), 0, DTYPES[z.dtype], ignore_index, 0)
        capi.logprobs_bwd(d, z.data_ptr(), t.data_ptr(), stats.data_ptr(), ptr(entropy), ptr(gl), ptr(ge),
                          g.data_ptr(), stream(logits))
    return g


class TokenLogprobs(torch.autograd.Function):
    """logprob, entropy = TokenLogprobs.apply(logits, tokens, ignore_index, check_tokens)."""

    @staticmethod
    def forward(ctx, logits, tokens, ignore_index=-100, check_tokens=True):
        logprob, entropy, stats, _, _ = token_logprobs(logits, tokens, 0, ignore_index, check_tokens)
        ctx.save_for_backward(logits, tokens, stats, entropy)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        return logprob, entropy

    @staticmethod
    @first_order
    def backward(ctx, grad_logprob, grad_entropy):
        if grad_logprob is None and grad_entropy is None:
            return None, None, None, None
        logits, tokens, stats, entropy = ctx.saved_tensors
        return token_logprobs_backward(logits, tokens, stats, entropy, grad_logprob, grad_entropy,
                                       ctx.ignore_index), None, None, None
