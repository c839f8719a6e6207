"""Dropout from a counter-based generator, on the kernels of csrc/dropout.hip: the mask is a function of (seed, step, site,
element index) and is never stored - the backward computes it again.

  state = dropout_state(seed, device)            {seed, step} in device memory
  y = dropout(x, p, state, site=0)               x / (1 - p) where kept, 0 elsewhere
  y = dropout_add(x, residual, p, state, site)   residual + dropout(x), one pass
  advance(state)                                 next step: new masks everywhere

`site` tells the dropout layers of a network apart that share one state.  The pair is read on the device when the kernel runs, so
a captured graph that contains advance(state) draws new masks at every replay; the forward keeps a copy of the pair it used, and
the backward takes that copy whatever has become of the state meanwhile.

An element is kept iff its 32-bit draw is >= round(p * 2^32): p is honoured to 2^-33, and the same (seed, step, site, shape) gives
the same mask for every type, layout and device.  A dropped element is 0 even where x is inf or NaN.  Draws: see csrc/dropout.hip
(Philox-4x32-10)."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ._lib import HipCallError, ptr
from .launch import ELEM, first_order, launch, need_device, need_elem


def dropout_state(seed: int, device, step: int = 0) -> torch.Tensor:
    """{seed, step} as the int64 device tensor that the operators read; seed: any 64 bits, step: 0 .. 2^32 - 1"""
    seed = int(seed) & (2 ** 64 - 1)
    return torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed, int(step)], dtype=torch.int64, device=device)


def advance(state: torch.Tensor) -> None:
    """the next step's masks from here on (stream-ordered, graph-capturable; the step counts modulo 2^32)"""
    state[1].add_(1)


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, scale, site, state):
        dev = x.device
        x = x.contiguous()
        res = None if residual is None else residual.contiguous()
        y = torch.empty(x.shape, dtype=x.dtype if res is None else torch.promote_types(x.dtype, res.dtype), device=dev)
        used = torch.empty(2, dtype=torch.int64, device=dev) if ctx.needs_input_grad[0] else None
        if y.numel():
            launch("nnz_dropout_forward", dev, x.data_ptr(), ELEM[x.dtype], ptr(res), 0 if res is None else ELEM[res.dtype],
                   y.data_ptr(), y.numel(), threshold, scale, site, state.data_ptr(), ptr(used))
        ctx.save_for_backward(used)
        ctx.cfg = (threshold, scale, site, x.dtype, None if res is None else res.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _backward(ctx, dy)
        with torch.no_grad():
            grads = _backward(ctx, dy)
        return first_order("dropout", grads, (dy,))


def _backward(ctx, dy):
    used, = ctx.saved_tensors
    threshold, scale, site, xt, rt = ctx.cfg
    dx = None
    if ctx.needs_input_grad[0]:
        g = dy.contiguous()
        dx = torch.empty(g.shape, dtype=xt, device=g.device)
        if dx.numel():
            launch("nnz_dropout_backward", g.device, g.data_ptr(), ELEM[g.dtype], dx.data_ptr(), ELEM[xt], dx.numel(), threshold,
                   scale, site, used.data_ptr())
    return dx, dy.to(rt) if rt is not None and ctx.needs_input_grad[1] else None, None, None, None, None


def _check_p(name, p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name}: p must lie in [0, 1], got {p}")


def _apply(name, x, residual, p, state, site, training):
    _check_p(name, p)
    need_device(name, x, residual, state)
    need_elem(name, x=x, residual=residual)
    if not isinstance(state, torch.Tensor) or state.dtype != torch.int64 or state.shape != (2,) or not state.is_contiguous():
        raise HipCallError(f"{name}: `state` is the int64 pair of dropout_state()")
    if not 0 <= site < 2 ** 31:
        raise ValueError(f"{name}: site must lie in [0, 2^31), got {site}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{name}: x {tuple(x.shape)} and residual {tuple(residual.shape)} differ in shape")
    threshold = round(p * 2 ** 32) if training else 0
    scale = 1.0 / (1.0 - p) if training and p < 1.0 else 1.0
    return _DropoutFn.apply(x, residual, threshold, scale, int(site), state)


def dropout(x: torch.Tensor, p: float, state: torch.Tensor, site: int = 0, training: bool = True) -> torch.Tensor:
    """x / (1 - p) where the mask keeps an element and 0 elsewhere; x itself when not training or p is 0"""
    _check_p("dropout", p)
    if (not training or p == 0.0) and x.is_cuda:
        return x
    return _apply("dropout", x, None, p, state, site, training)


def dropout_add(x: torch.Tensor, residual: torch.Tensor, p: float, state: torch.Tensor, site: int = 0,
                training: bool = True) -> torch.Tensor:
    """residual + dropout(x) in one pass, in the wider of the two types (fp16 beside bf16: fp32)"""
    return _apply("dropout_add", x, residual, p, state, site, training)


class Dropout(nn.Module):
    """dropout(x) or, called with a residual, dropout_add(x, residual), on a state shared with the network's other dropouts"""

    def __init__(self, p: float, state: torch.Tensor, site: int):
        super().__init__()
        _check_p("Dropout", p)
        self.p, self.state, self.site = p, state, site

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if residual is None:
            return dropout(x, self.p, self.state, self.site, self.training)
        return dropout_add(x, residual, self.p, self.state, self.site, self.training)

    def extra_repr(self) -> str:
        return f"p={self.p}, site={self.site}"
