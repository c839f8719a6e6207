"""The state-carrying operators of a Mamba block - its short causal convolution and its selective scan - for prompts and for single
tokens, on the kernels of csrc/mamba_state.hip.  What the reference's Mamba module does in `step` and with `inference_params`
(nnunetv2/nets/seg_mamba/mamba_simple.py:190-215, 357-411) in token-major form: rows are (B, L, D) with the channels innermost, as
the projections around them write and read them.

  causal_conv1d_prompt(x, weight, bias, activation, conv_state, lengths)                  (B, L, D) -> (B, L, D)
  causal_conv1d_token(x, conv_state, weight, bias, activation, active)                    (B, D) -> (B, D)
  selective_scan_prompt(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths, ...)  (B, L, D) -> (B, L, D)
  selective_scan_token(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, active, ...)    (B, D) -> (B, D)

conv_state (B, D, W) holds the last W inputs of every sequence, state (B, D, N) its scan state; both are read and brought up to date
IN PLACE.  A prompt may continue an earlier one.  lengths (B,): tokens of each sequence in a padded batch; nothing behind them is
read, outputs there are 0, and a sequence of length 0 keeps its states (values outside 0 .. L are clamped).  active (B,) bool: the
sequences that take part in a token step; the others keep their states and get 0.

Heads: dt is (B, L, H) with D = H * P channels, head by head; A is (H, N) or, one decay a head, (H,); D and dt_bias are (H,).
B and C are (B, L, G, N), or (B, L, N) for one group; group g serves the channels g * D / G ...  H = D is Mamba, A (H,) is Mamba2.
N: 4, 8, 16 or 32; W: up to 8; the scan over prompts takes at most 65535 sequences a call.  Activations fp32, fp16 or bf16, all of one
type; parameters are taken in fp32, states are fp32 (conv_state: the activations' type or fp32).

These operators have no backward (training: nnuzoo_amd.mamba_block, nnuzoo_amd.selective_scan): an input that requires a gradient
is refused while gradients are being recorded, one that carries a forward-mode tangent always.  There is no CPU path."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from ._lib import load, ptr
from .launch import ELEM, launch, need_device, need_elem

MAX_WIDTH = 8
STATE_WIDTHS = (4, 8, 16, 32)
MAX_PROMPTS = 65535         # sequences of a scan over prompts: the rows of a launch's grid


def _no_grad(name, *tensors):
    if forward_ad._current_level >= 0:      # within a dual level, which no_grad() does not end
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() (training goes through "
                                   "nnuzoo_amd.mamba_block.causal_conv1d_fn and nnuzoo_amd.selective_scan.selective_scan_fn)")


def _shape(name, arg, t, shape):
    if t.shape != shape:
        raise ValueError(f"{name}: `{arg}` has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _inner(t):
    """t with adjacent elements along the last axis"""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().float().contiguous()


def _own_memory(name, arg, t):
    """a state is written in place: no two of its elements may share memory"""
    if t.is_contiguous():
        return
    need = 1
    for stride, size in sorted((t.stride(d), t.shape[d]) for d in range(t.dim()) if t.shape[d] > 1):
        if stride < need:
            raise ValueError(f"{name}: elements of `{arg}` share memory (shape {tuple(t.shape)}, strides {t.stride()})")
        need = stride * (size - 1) + need


def _which(name, arg, t, batch, kinds):
    if t is None:
        return None
    if t.dtype not in kinds:
        raise TypeError(f"{name}: `{arg}` must be {' or '.join(str(k).replace('torch.', '') for k in kinds)}, got {t.dtype}")
    _shape(name, arg, t, (batch,))
    return t.contiguous()


def _conv_checks(name, x, weight, bias, activation, conv_state, rows):
    need_elem(name, x=x, weight=weight, bias=bias)
    _no_grad(name, x, weight, bias, conv_state)
    if activation not in (None, "silu", "swish"):
        raise NotImplementedError(f"{name}: activation {activation!r} (None, 'silu' or 'swish')")
    if x.dim() != rows:
        raise ValueError(f"{name}: x must be {'(B, L, D)' if rows == 3 else '(B, D)'}, got {tuple(x.shape)}")
    B, D = x.shape[0], x.shape[-1]
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight.squeeze(1)      # nn.Conv1d's layout
    W = weight.shape[-1]
    if weight.dim() != 2:
        raise ValueError(f"{name}: `weight` has shape {tuple(weight.shape)}, expected {(D, 'W')}")
    _shape(name, "weight", weight, (D, W))
    if not 1 <= W <= MAX_WIDTH:
        raise NotImplementedError(f"{name}: kernel widths 1 .. {MAX_WIDTH}, got {W}")
    if bias is not None:
        _shape(name, "bias", bias, (D,))
    if conv_state is not None:
        _shape(name, "conv_state", conv_state, (B, D, W))
        if conv_state.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name}: `conv_state` must be {x.dtype} or float32, got {conv_state.dtype}")
        _own_memory(name, "conv_state", conv_state)
    return _param(weight), _param(bias), B, D, W


def _state_args(st):
    return (0, 0, 0, 0, 0) if st is None else (st.data_ptr(), ELEM[st.dtype], *st.stride())


def causal_conv1d_prompt(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         activation: Optional[str] = "silu", conv_state: Optional[torch.Tensor] = None,
                         lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y_t = act(bias + sum_j weight[:, j] x_{t - W + 1 + j}) for the tokens of every sequence; what lies before its first token
    comes from conv_state (zeros without one)"""
    name = "causal_conv1d_prompt"
    dev = need_device(name, x, weight, bias, conv_state, lengths)
    weight, bias, B, D, W = _conv_checks(name, x, weight, bias, activation, conv_state, 3)
    lengths = _which(name, "lengths", lengths, B, (torch.int32, torch.int64))
    x = _inner(x)
    L = x.shape[1]
    y = torch.empty((B, L, D), dtype=x.dtype, device=dev)
    if y.numel():
        launch("nnz_causal_conv1d_prompt", dev, x.data_ptr(), ELEM[x.dtype], x.stride(0), x.stride(1), weight.data_ptr(), ptr(bias),
               y.data_ptr(), *_state_args(conv_state), ptr(lengths), int(lengths is not None and lengths.dtype == torch.int64),
               B, L, D, W, int(activation is not None))
    return y


def causal_conv1d_token(x: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        activation: Optional[str] = "silu", active: Optional[torch.Tensor] = None) -> torch.Tensor:
    """one token of every active sequence: conv_state moves on by one column, y = act(bias + sum_j weight[:, j] conv_state[:, :, j])"""
    name = "causal_conv1d_token"
    dev = need_device(name, x, conv_state, weight, bias, active)
    weight, bias, B, D, W = _conv_checks(name, x, weight, bias, activation, conv_state, 2)
    active = _which(name, "active", active, B, (torch.bool,))
    x = _inner(x)
    y = torch.empty((B, D), dtype=x.dtype, device=dev)
    if y.numel():
        launch("nnz_causal_conv1d_token", dev, x.data_ptr(), ELEM[x.dtype], x.stride(0), weight.data_ptr(), ptr(bias), y.data_ptr(),
               *_state_args(conv_state), ptr(active), B, D, W, int(activation is not None))
    return y


def _scan_checks(name, x, dt, A, B, C, D, z, dt_bias, state, rows):
    """checks and brings into form: (x, dt, B, C, z, A, D, dt_bias, channels, heads, groups, state width)"""
    if x.dim() != rows:
        raise ValueError(f"{name}: x must be {'(B, L, D)' if rows == 3 else '(B, D)'}, got {tuple(x.shape)}")
    need_elem(name, x=x, A=A, D=D, dt_bias=dt_bias)
    _no_grad(name, x, dt, A, B, C, D, z, dt_bias, state)
    for arg, t in (("dt", dt), ("B", B), ("C", C), ("z", z)):
        if t is not None and t.dtype is not x.dtype:
            raise TypeError(f"{name}: x is {x.dtype}, `{arg}` is {t.dtype}: activations share one type")
    *lead, d = x.shape
    h = dt.shape[-1]
    _shape(name, "dt", dt, (*lead, h))
    if z is not None:
        _shape(name, "z", z, x.shape)
    if B.dim() == rows:
        B = B.unsqueeze(-2)
    if C.dim() == rows:
        C = C.unsqueeze(-2)
    if B.dim() != rows + 1:
        raise ValueError(f"{name}: `B` has {B.dim()} dimensions, expected {rows} or {rows + 1}")
    g, n = B.shape[-2:]
    _shape(name, "B", B, (*lead, g, n))
    _shape(name, "C", C, B.shape)
    if n not in STATE_WIDTHS:
        raise NotImplementedError(f"{name}: state widths {STATE_WIDTHS}, got {n}")
    if h < 1 or g < 1 or d % h or h % g:
        raise ValueError(f"{name}: {d} channels, {h} heads, {g} groups: heads divide the channels, groups divide the heads")
    if A.shape != (h, n) and A.shape != (h,):
        raise ValueError(f"{name}: `A` has shape {tuple(A.shape)}, expected {(h, n)} or {(h,)}")
    if D is not None:
        _shape(name, "D", D, (h,))
    if dt_bias is not None:
        _shape(name, "dt_bias", dt_bias, (h,))
    if state is not None:
        if state.dtype is not torch.float32:
            raise TypeError(f"{name}: `state` must be float32, got {state.dtype}")
        _shape(name, "state", state, (lead[0], d, n))
        if d and not state.is_contiguous():
            if state.stride(2) != 1 or (d > 1 and state.stride(1) != n):
                raise ValueError(f"{name}: `state` is updated in place and must be contiguous within a sequence, strides {state.stride()}")
            _own_memory(name, "state", state)
    return _inner(x), _inner(dt), _inner(B), _inner(C), _inner(z), _param(A), _param(D), _param(dt_bias), d, h, g, n


_Long7, _Long12 = ctypes.c_long * 7, ctypes.c_long * 12


def selective_scan_prompt(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                          D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                          dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                          state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                          A_is_log: bool = False) -> torch.Tensor:
    """h_t = exp(s_t A) h_{t-1} + s_t x_t B_t, y_t = (<C_t, h_t> + D x_t) * silu(z_t) with s_t = [softplus](dt_t + dt_bias) over the
    tokens of every sequence; h starts from `state` (zeros without one) and is left there.  A_is_log: A holds log(-A), the form in which
    the blocks keep it"""
    name = "selective_scan_prompt"
    dev = need_device(name, x, dt, A, B, C, D, z, dt_bias, state, lengths)
    x, dt, B, C, z, A, D, dt_bias, d, h, g, n = _scan_checks(name, x, dt, A, B, C, D, z, dt_bias, state, 3)
    batch, L = x.shape[:2]
    if batch > MAX_PROMPTS:
        raise NotImplementedError(f"{name}: at most {MAX_PROMPTS} sequences a call, got {batch}")
    lengths = _which(name, "lengths", lengths, batch, (torch.int32, torch.int64))
    y = torch.empty((batch, L, d), dtype=x.dtype, device=dev)
    if y.numel():
        strides = _Long12(*x.stride()[:2], *dt.stride()[:2], *B.stride()[:3], *C.stride()[:3],
                          *(z.stride()[:2] if z is not None else (0, 0)))
        ws_bytes = load().nnz_selective_scan_prompt_workspace_bytes(batch, L, d, h, g, n)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        launch("nnz_selective_scan_prompt", dev, x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), ptr(z), ELEM[x.dtype],
               strides, A.data_ptr(), A.dim() - 1 + 2 * bool(A_is_log), ptr(D), ptr(dt_bias), int(dt_softplus), ptr(state),
               0 if state is None else state.stride(0), y.data_ptr(), ptr(lengths),
               int(lengths is not None and lengths.dtype == torch.int64), ptr(ws), ws_bytes, batch, L, d, h, g, n)
    return y


def selective_scan_token(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                         D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                         dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False, *, state: torch.Tensor,
                         active: Optional[torch.Tensor] = None, A_is_log: bool = False) -> torch.Tensor:
    """selective_scan_prompt for one token of every active sequence: x, z (B, D), dt (B, H), B, C (B, G, N) or (B, N)"""
    name = "selective_scan_token"
    dev = need_device(name, x, dt, A, B, C, D, z, dt_bias, state, active)
    x, dt, B, C, z, A, D, dt_bias, d, h, g, n = _scan_checks(name, x, dt, A, B, C, D, z, dt_bias, state, 2)
    batch = x.shape[0]
    active = _which(name, "active", active, batch, (torch.bool,))
    y = torch.empty((batch, d), dtype=x.dtype, device=dev)
    if y.numel():
        strides = _Long7(x.stride(0), dt.stride(0), *B.stride()[:2], *C.stride()[:2], 0 if z is None else z.stride(0))
        launch("nnz_selective_scan_token", dev, x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), ptr(z), ELEM[x.dtype],
               strides, A.data_ptr(), A.dim() - 1 + 2 * bool(A_is_log), ptr(D), ptr(dt_bias), int(dt_softplus), state.data_ptr(), state.stride(0),
               y.data_ptr(), ptr(active), batch, d, h, g, n)
    return y
