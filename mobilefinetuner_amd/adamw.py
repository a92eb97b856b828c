"""AdamW over many tensors at once on the GPU, over the C ABI of include/mft/adamw.h:
the step that trains LoRA adapters (LoRALinear.trainable_parameters), norms'
weights and whole matrices.

Parameters are fp32, or bf16 with an fp32 master copy among the states.  States
are fp32 or 8 bits wide.  One step is two launches and one more for each further
48 (8 bits) or 64 tensors, and with clipping one for each 120.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import attrgetter

import torch

from . import capi
from .device import guard, operand, ptr, stream, workspace

GROUP = capi.ADAMW_GROUP  # values of an 8-bit state with one scale
_FIELDS = C.sizeof(capi.AdamWTensor) // 8
_GRAD = capi.AdamWTensor.grad.offset // 8
_ADDRESS, _SIZE, _WHOLE = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_GRADIENT, _DTYPE = attrgetter("grad"), attrgetter("dtype")


class AdamW:
    """AdamW(params, lr, betas, eps, weight_decay, state_bits): steps params, a list of
    contiguous leaf tensors on one GPU, by their .grad.

    weight_decay is a number or one for each parameter.  lr may be an fp32 GPU
    tensor of one value, which a captured step reads at each replay (a float is
    part of the capture); both may be set between steps.  With state_bits 8 the
    averages are e4m3 numbers with an fp32 scale for each 256 values of a tensor
    (exp_avg_sq: of the square root), 2 bytes a value in place of 8.

    state: {"step": int64 [], "exp_avg", "exp_avg_sq": flat, "exp_avg_scale",
    "exp_avg_sq_scale": with 8 bits, "master": fp32, of the bf16 parameters}.  In
    the flat ones each parameter's part starts at a multiple of 256 values
    (views()); state_dict() says whose they are.  One step's number serves all
    parameters, also one that had no gradient in some steps."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        first = self.params[0]
        for p in self.params:
            operand(p, "a parameter", first)
            if not p.is_leaf or not p.is_contiguous():
                raise ValueError("a parameter must be a contiguous leaf tensor")
        ends = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(ends, ends[1:])):
            raise ValueError("a parameter is given twice, or shares memory with another")
        self.lr, self.betas, self.eps = lr, tuple(betas), eps
        self.weight_decay, self.state_bits = weight_decay, state_bits
        self._sizes = [p.numel() for p in self.params]
        half = [p.dtype == torch.bfloat16 for p in self.params]
        self._dtypes = [p.dtype for p in self.params]
        self._starts, total = self._places(self._sizes)
        self._master_starts, masters = self._places([n if h else 0 for n, h in zip(self._sizes, half)])
        with guard(first):
            def zeros(n, dtype=torch.float32):
                return torch.zeros(n, dtype=dtype, device=first.device)

            self.state = {"step": zeros((), torch.int64)}
            if state_bits == 32:
                self.state.update(exp_avg=zeros(total), exp_avg_sq=zeros(total))
            else:
                self.state.update({n: zeros(total, torch.uint8).view(torch.float8_e4m3fn)
                                   for n in ("exp_avg", "exp_avg_sq")})
                self.state.update({n: zeros(total // GROUP) for n in ("exp_avg_scale", "exp_avg_sq_scale")})
            if any(half):
                self.state["master"] = zeros(masters)
        self._layout = {k: (v.shape, v.dtype) for k, v in self.state.items()}
        self._words = None  # the C ABI's table of the tensors
        self.reload_masters()

    @property
    def weight_decay(self):
        """A list of one for each parameter."""
        return self.__dict__["weight_decay"]

    @weight_decay.setter
    def weight_decay(self, decay):
        decay = list(decay) if isinstance(decay, (list, tuple)) else [decay] * len(self.params)
        self.__dict__["weight_decay"] = self._one_each(decay)

    def _one_each(self, decay):
        if len(decay) != len(self.params):
            raise ValueError(f"weight_decay has {len(decay)} values for {len(self.params)} parameters")
        return decay

    def __getstate__(self):
        return {**self.__dict__, "_words": None, "_table": None}  # addresses are a process's own

    @staticmethod
    def _places(sizes):
        at, starts = 0, []
        for n in sizes:
            starts.append(at)
            at += (n + GROUP - 1) // GROUP * GROUP
        return starts, at

    def views(self, name):
        """state[name] by parameter: views of the parameters' shapes (of [ceil(n / 256)] for scales; for
        "master" None beside an fp32 parameter)."""
        flat, out = self.state[name], []
        starts = self._master_starts if name == "master" else self._starts
        for p, n, a in zip(self.params, self._sizes, starts):
            if name.endswith("_scale"):
                out.append(flat[a // GROUP : a // GROUP + (n + GROUP - 1) // GROUP])
            elif name == "master" and p.dtype != torch.bfloat16:
                out.append(None)
            else:
                out.append(flat[a : a + n].view(p.shape))
        return out

    @torch.no_grad()
    def reload_masters(self):
        """The masters start again from the bf16 parameters: after these have been written by anything
        but step(), which writes them from the masters."""
        if "master" in self.state:
            for p, m in zip(self.params, self.views("master")):
                if m is not None:
                    m.copy_(p)

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    def state_dict(self):
        return {"state": {k: v.clone() for k, v in self.state.items()}, "state_bits": self.state_bits,
                "params": self._parts()}

    def _parts(self):
        """Whose the flat states' parts are: each parameter's shape and type."""
        return [(list(p.shape), str(t)) for p, t in zip(self.params, self._dtypes)]

    def load_state_dict(self, d):
        """Takes over a copy of another's state; the parameters are the caller's to load, before or after.  They
        must have the other's shapes and types, in its order (what a state without "params" does not tell)."""
        state = d["state"]
        if d["state_bits"] != self.state_bits or state.keys() != self.state.keys():
            raise ValueError(f"the state has {d['state_bits']} bits and {sorted(state)}, "
                             f"this optimizer {self.state_bits} and {sorted(self.state)}")
        for k, (shape, dtype) in self._layout.items():
            if state[k].shape != shape or state[k].dtype != dtype:
                raise ValueError(f"{k} must be {dtype} {list(shape)}, got {state[k].dtype} {list(state[k].shape)}")
        if "params" in d:
            given, own = [(list(s), t) for s, t in d["params"]], self._parts()
            if given != own:
                i = next((i for i, (a, b) in enumerate(zip(given, own)) if a != b), min(len(given), len(own)))
                raise ValueError(f"the state is of {len(given)} parameters, this optimizer has {len(own)}: they differ "
                                 f"from parameter {i} on, {given[i:i + 1]} and {own[i:i + 1]}")
        for k, v in state.items():
            self.state[k].copy_(v)

    def _fill(self):
        """The C ABI's table of the tensors, but for their gradients."""
        params, first = self.params, self.params[0]
        decay = self._one_each(self.weight_decay)
        for p, n, t in zip(params, self._sizes, self._dtypes):
            operand(p, "a parameter", first, t)
            if p.numel() != n or not p.is_contiguous():
                raise ValueError("a parameter has changed its size or is no longer contiguous")
        for k, (shape, dtype) in self._layout.items():
            if not operand(self.state[k], f"state[{k!r}]", first, dtype, shape).is_contiguous():
                raise ValueError(f"state[{k!r}] must be contiguous")
        table = bytearray(len(params) * C.sizeof(capi.AdamWTensor))
        at = {k: v.data_ptr() for k, v in self.state.items()}
        wide = self.state["exp_avg"].element_size()
        for i, (t, p) in enumerate(zip((capi.AdamWTensor * len(params)).from_buffer(table), params)):
            a, half = self._starts[i], p.dtype == torch.bfloat16
            t.n = self._sizes[i]
            t.param = at["master"] + 4 * self._master_starts[i] if half else p.data_ptr()
            t.param_bf16 = p.data_ptr() if half else None
            t.exp_avg, t.exp_avg_sq = at["exp_avg"] + wide * a, at["exp_avg_sq"] + wide * a
            if self.state_bits == 8:
                t.exp_avg_scale = at["exp_avg_scale"] + 4 * (a // GROUP)
                t.exp_avg_sq_scale = at["exp_avg_sq_scale"] + 4 * (a // GROUP)
            t.weight_decay = decay[i]
        self._table = (capi.AdamWTensor * len(params)).from_buffer(table)
        self._words = memoryview(table).cast("Q")

    def step(self, max_norm=None):
        """One step of the parameters that have a gradient.  With max_norm all gradients are scaled
        by min(1, max_norm / (their norm + 1e-6)) on their way in, and the norm is returned (fp32 [],
        on the GPU; None without max_norm or where no value has a gradient)."""
        params, sizes, dtypes = self.params, self._sizes, self._dtypes
        stepped = params
        grads = on = list(map(_GRADIENT, params))
        if any(g is None for g in grads):
            on = [g for g in grads if g is not None]
            if not on:
                return None
            sizes, dtypes, stepped = map(list, zip(*(c for *c, g in zip(sizes, dtypes, params, grads) if g is not None)))
        if not any(sizes):
            return None
        # what a caller can have changed since the last step: data replaced or moved by p.data, the decays
        seen = (list(map(_ADDRESS, params)), [v.data_ptr() for v in self.state.values()], list(self.weight_decay))
        if (self._words is None or seen != self._seen or list(map(_SIZE, params)) != self._sizes
                or not all(map(_WHOLE, params))):
            self._fill()
            self._seen = seen
        if list(map(_SIZE, on)) != sizes or list(map(_DTYPE, on)) != dtypes:
            raise ValueError("a gradient must have its parameter's size and type")
        if not all(map(_WHOLE, on)):
            if any(g.layout is not torch.strided for g in on):
                raise ValueError("a gradient must be dense")
            on = [g.contiguous() for g in on]  # alive until the launches are enqueued
        addresses = list(map(_ADDRESS, on))
        if len(on) != len(grads):
            left = iter(addresses)
            addresses = [0 if g is None else next(left) for g in grads]
        self._words[_GRAD::_FIELDS] = memoryview(array("Q", addresses))
        lr, address = self.lr, None
        if isinstance(lr, torch.Tensor):
            if operand(lr, "lr", params[0], torch.float32).numel() != 1:
                raise ValueError("lr must be a number or a GPU tensor of one value")
            lr, address = 0.0, lr.data_ptr()
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        d = capi.adamw_desc(lr, *self.betas, self.eps, max_norm or 0.0, self.state_bits, address)
        with guard(params[0]):
            norm = None if max_norm is None else params[0].new_empty((), dtype=torch.float32)
            ws = workspace(capi.adamw_workspace_size(d, self._table), params[0])
            capi.adamw_step(d, self._table, self.state["step"].data_ptr(), ptr(norm), ws.data_ptr(), stream(params[0]))
        torch.autograd.graph.increment_version(stepped)
        return norm
