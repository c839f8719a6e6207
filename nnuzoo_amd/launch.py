"""What the operators with fp32 / fp16 / bf16 tensors share on the host: element types as the C boundary names them, and a launch
on the tensors' own device and that device's current stream."""
from __future__ import annotations

import torch

from ._lib import HipCallError, check, load

ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def need_device(name: str, *tensors) -> torch.device:
    """the one device of all tensors (None is skipped); CPU tensors and mixed devices are refused"""
    dev = None
    for t in tensors:
        if t is not None:
            d = t.device
            if dev is None:
                dev = d
            if d != dev or d.type != "cuda":
                if d.type != "cuda" or dev.type != "cuda":
                    raise RuntimeError(f"nnuzoo_amd.{name} runs on MI355X through libnnuzoo_hip.so only (no CPU fallback)")
                raise HipCallError(f"{name}: tensors on {dev} and {d}")
    return dev


def need_elem(name: str, **tensors) -> None:
    for arg, t in tensors.items():
        if t is not None and t.dtype not in ELEM:
            raise NotImplementedError(f"{name}: `{arg}` must be float32, float16 or bfloat16, got {t.dtype}")


_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream() without the Stream object: 0.1 us, not 2
_current = torch.cuda.current_device


def launch(name: str, device: torch.device, *args) -> None:
    """`_lib.call` with the device's current stream as the last argument, whatever device is current"""
    fn = getattr(load(), name)
    if device.index == _current():
        rc = fn(*args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device.index))
    if rc:
        check(rc, name)


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, out, *sources):
        ctx.name = name
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} has no second derivative")


def first_order(name: str, grads, sources):
    """`grads` of a backward that is itself being recorded (create_graph=True): usable as values, an error once something is
    differentiated through them - also where only the saved `sources`, not the incoming gradient, require one"""
    return tuple(g if g is None else _Once.apply(name, g, *(s for s in sources if s is not None)) for g in grads)
