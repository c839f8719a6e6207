"""Group norm with an activation on channels-last tensors, on the kernels of csrc/group_norm.hip: what nn.GroupNorm followed by
an activation computes in the residual blocks of the LightMUNet family (reference: monai's get_norm_layer / get_act_layer at
nnunetv2/nets/lm2net.py:119-121,160-171, light_mamba2net.py:480-482,519-531, LightMUNet.py:105-107,144-156), one operator with its
gradient.

  group_norm_act(x, num_groups, weight, bias, eps, activation, negative_slope)      x (N, *spatial, C), C innermost
  GroupNormAct(num_groups, num_channels, ..., activation=...)                       nn.GroupNorm's parameters, x (N, C, *spatial)
  norm_act(norm, act, x)                                                            act(norm(x)) of two modules on either path

fp32 / fp16 / bf16 in; the output has the input's type, or fp32 under autocast (group_norm is on autocast's fp32 list).
Statistics are fp64 sums, everything else is computed in fp32 and rounded once.  Results are bit-identical from run to run.
There is no CPU path and, but for norm_act, which stands for two modules that have one, no second derivative."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd import forward_ad

from ._lib import load, ptr
from .launch import ELEM, first_order, launch, need_device, need_elem

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "leaky_relu": 2, "silu": 3}
MAX_CHANNELS = 4096     # csrc/group_norm.hip GN_MAX_C


def _rows(x: torch.Tensor):
    """(x or its contiguous copy, batch stride, row stride): rows of C adjacent elements, evenly spaced within a sample.  The copy is made
    in front of the autograd function, so that what the function saves is part of the graph"""
    C = x.shape[-1]
    if x.stride(-1) == 1 or C == 1:
        step = want = None
        for d in range(x.dim() - 2, 0, -1):
            if x.shape[d] != 1:
                if step is None:
                    step = want = x.stride(d)
                elif x.stride(d) != want:
                    break
                want *= x.shape[d]
        else:
            return x, x.stride(0), C if step is None else step
    x = x.contiguous()
    return x, x.numel() // max(1, x.shape[0]), C


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, xb, xs, weight, bias, groups, eps, act, slope, out_dtype, twice):
        dev = x.device
        y = torch.empty(x.shape, dtype=out_dtype, device=dev)
        N, C = x.shape[0], x.shape[-1]
        stats = None
        if y.numel():
            S = x.numel() // (N * C)
            ws_bytes = load().nnz_group_norm_act_workspace_bytes(N, S, C, groups, 0)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
            stats = torch.empty(2 * N * groups, dtype=torch.float32, device=dev)
            launch("nnz_group_norm_act_forward", dev, x.data_ptr(), ELEM[x.dtype], xb, xs, ptr(weight), ptr(bias), y.data_ptr(),
                   ELEM[out_dtype], stats.data_ptr(), ptr(ws), ws_bytes, N, S, C, groups, eps, act, slope)
            # asked here: whatever Python the backward runs, on the engine's own thread, takes it three to four times as long
            ctx.bwd_bytes = load().nnz_group_norm_act_workspace_bytes(N, S, C, groups, 1)
            ctx.cfg = (xb, xs, N, S, C, groups, act, slope)
        ctx.save_for_backward(x, weight, bias)
        ctx.stats = stats       # of this node's own making: neither input nor output
        ctx.twice = (groups, eps, act, slope) if twice else None
        return y

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _backward(ctx, dy)
        if ctx.twice:
            return _recorded_backward(ctx, dy)
        with torch.no_grad():
            grads = _backward(ctx, dy)
        return first_order("group_norm_act", grads, (dy, *ctx.saved_tensors))


def _backward(ctx, dy):
    x, weight, bias = ctx.saved_tensors
    need_x, _, _, need_w, need_b, *_ = ctx.needs_input_grad
    dev, C, stats = x.device, x.shape[-1], ctx.stats
    make = torch.zeros if stats is None else torch.empty
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    dw = make(C, dtype=torch.float32, device=dev) if need_w else None
    db = make(C, dtype=torch.float32, device=dev) if need_b else None
    if stats is not None:
        xb, xs, N, S, C, groups, act, slope = ctx.cfg
        dy = dy.contiguous()
        ws_bytes = ctx.bwd_bytes
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        launch("nnz_group_norm_act_backward", dev, x.data_ptr(), ELEM[x.dtype], xb, xs, dy.data_ptr(), ELEM[dy.dtype],
               ptr(weight), ptr(bias), stats.data_ptr(), ptr(dx), ptr(dw), ptr(db), ptr(ws), ws_bytes, N, S, C, groups, act, slope)
    return dx, None, None, dw, db, None, None, None, None, None, None


def _recorded_backward(ctx, dy):
    """the gradients as functions that can be differentiated again (create_graph=True), from the library's group norm: what a caller
    of the modules that norm_act stands for gets"""
    x, weight, bias = ctx.saved_tensors
    groups, eps, act, slope = ctx.twice
    z = F.group_norm(x.movedim(-1, 1).float(), groups, weight, bias, eps)
    y = {0: lambda t: t, 1: F.relu, 2: lambda t: F.leaky_relu(t, slope), 3: F.silu}[act](z).movedim(1, -1).to(dy.dtype)
    grads = [None] * 11
    which = [i for i in (0, 3, 4) if ctx.needs_input_grad[i]]
    ins = {0: x, 3: weight, 4: bias}
    for i, g in zip(which, torch.autograd.grad(y, [ins[i] for i in which], dy, create_graph=True)):
        grads[i] = g
    return tuple(grads)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: Optional[str] = None,
                   negative_slope: float = 0.01) -> torch.Tensor:
    """activation(group_norm(x)) for x (N, *spatial, C); activation: None / "none", "relu", "leaky_relu", "silu"."""
    return _group_norm_act(x, num_groups, weight, bias, eps, activation, negative_slope, twice=False)


def _group_norm_act(x, num_groups, weight, bias, eps, activation, negative_slope, twice):
    dev = need_device("group_norm_act", x, weight, bias)
    need_elem("group_norm_act", x=x, weight=weight, bias=bias)
    if activation not in ACTIVATIONS:
        raise NotImplementedError(f"group_norm_act: activation {activation!r} (one of {sorted(k for k in ACTIVATIONS if k)})")
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: x must be (N, *spatial, C), got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups < 1 or C % num_groups or C < 1:
        raise ValueError(f"group_norm_act: {C} channels in {num_groups} groups")
    if C > MAX_CHANNELS:
        raise NotImplementedError(f"group_norm_act: at most {MAX_CHANNELS} channels, got {C}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and p.shape != (C,):
            raise ValueError(f"group_norm_act: `{name}` has shape {tuple(p.shape)}, expected ({C},)")
    if weight is not None:
        weight = weight.float().contiguous()
    if bias is not None:
        bias = bias.float().contiguous()
    out_dtype = torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype
    return _GroupNormActFn.apply(*_rows(x), weight, bias, int(num_groups), float(eps), ACTIVATIONS[activation],
                                 float(negative_slope), out_dtype, twice)


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm (same constructor, parameters, state_dict) followed by an activation, for x (N, C, *spatial): a tensor whose
    channels lie innermost (torch.channels_last, token-major views) is read in place and the output has the same layout; any
    other layout is copied to it first."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, device=None, dtype=None,
                 activation: Optional[str] = None, negative_slope: float = 0.01):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        if activation not in ACTIVATIONS:
            raise NotImplementedError(f"GroupNormAct: activation {activation!r}")
        self.activation, self.negative_slope = activation, negative_slope

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = group_norm_act(x.movedim(1, -1), self.num_groups, self.weight, self.bias, self.eps, self.activation,
                           self.negative_slope)
        return y.movedim(-1, 1)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"


def _token_order(x: torch.Tensor):
    """the permutation that turns x (N, C, *spatial) into contiguous (N, *spatial in memory order, C), or None where there is none
    or where x is just as well stored channel by channel"""
    if x.dim() < 3 or x.shape[1] < 2 or x.is_contiguous():
        return None
    perm = (0, *sorted(range(2, x.dim()), key=lambda d: -x.stride(d)), 1)
    return perm if x.permute(perm).is_contiguous() else None


def _hooked(m: nn.Module) -> bool:
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


_hooks_of_all = nn.modules.module._has_any_global_hook      # register_module_forward_hook and its kin


def _transformed(*tensors) -> bool:
    """whether torch.func transforms (vmap, jvp, ..) or forward-mode tangents are at work, which the operator has no rules for"""
    if torch._C._are_functorch_transforms_active():
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def norm_act(norm: nn.Module, act: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """act(norm(x)): the operator where `norm` is an nn.GroupNorm, `act` one of its activations and x a device tensor whose channels
    lie innermost (what the token-major mixers of the LightMUNet family hand on; the spatial axes may lie in any order); the two
    modules one after the other otherwise."""
    name = {nn.ReLU: "relu", nn.SiLU: "silu", nn.LeakyReLU: "leaky_relu", nn.Identity: "none"}.get(type(act))
    if (type(norm) is nn.GroupNorm and name is not None and x.is_cuda and x.dtype in ELEM and norm.num_channels <= MAX_CHANNELS
            and not _hooked(norm) and not _hooked(act) and not _hooks_of_all()
            and not _transformed(x, norm.weight, norm.bias)):
        perm = _token_order(x)
        if perm is not None:
            from . import backends
            backends.note(norm, "hip", "group norm + activation")
            y = _group_norm_act(x.permute(perm), norm.num_groups, norm.weight, norm.bias, norm.eps, name,
                                getattr(act, "negative_slope", 0.01), twice=True)
            return y.permute([perm.index(d) for d in range(x.dim())])
    return act(norm(x))
