"""Global norm of the adapters' gradients and clipping by it, between ``i8lora_backward`` and the
optimizer (the reference's training loop, src/training/wan_runner.jl:108-289), over
``reels_hip_grad_norm`` and ``reels_hip_clip_gradients``.
"""
from __future__ import annotations

import math
from array import array
from typing import Optional, Sequence

import torch

from . import _lib
from .layers import _DTYPE_CODE, _need_device, _ptr, _stream, on_device


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one run of memory, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz > 1):
        if stride != n:
            return False
        n *= size
    return True


def _tensors(grads, name):
    if not all(isinstance(g, torch.Tensor) for g in grads):
        raise TypeError(f"{name} must be tensors")
    for g in grads:
        if g.dtype not in _DTYPE_CODE:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {g.dtype}")
        _need_device(g, name)
    if len({g.device for g in grads}) > 1:
        raise ValueError(f"{name} lie on several devices")


def _pointers(ts):
    return array("q", [t.data_ptr() for t in ts])


def _call(grads, max_norm, outs):
    _tensors(grads, "gradients")
    if not all(map(_dense, grads)):
        raise ValueError("gradients must be dense")
    dev = grads[0].device
    n = len(grads)
    L = _lib.lib()
    ptrs, sizes = _pointers(grads), array("q", [g.numel() for g in grads])
    types = array("i", [_DTYPE_CODE[g.dtype] for g in grads])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = L.reels_hip_grad_workspace_bytes(n)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)

    def at(a):
        return a.buffer_info()[0]

    with on_device(dev):
        if max_norm is None:
            _lib.check("reels_hip_grad_norm", L.reels_hip_grad_norm(
                at(ptrs), at(sizes), at(types), n, _ptr(norm), _ptr(ws), nbytes, _stream(dev)))
        else:
            to = ptrs if outs is grads else _pointers(outs)
            _lib.check("reels_hip_clip_gradients", L.reels_hip_clip_gradients(
                at(ptrs), at(to), at(sizes), at(types), n, float(max_norm), _ptr(norm), _ptr(ws),
                nbytes, _stream(dev)))
    return norm


def gradient_norm(grads: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """sqrt of the sum of squares of all elements of all tensors (None entries are skipped), float32
    on their device; the sum runs in 64 bits."""
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("no gradients")
    return _call(grads, None, None)


def clip_gradients(grads: Sequence[Optional[torch.Tensor]], max_norm: float,
                   out: Optional[Sequence[Optional[torch.Tensor]]] = None) -> torch.Tensor:
    """Multiplies the gradients by min(1, max_norm / (norm + 1e-6)), norm their ``gradient_norm``,
    which it returns (without waiting for it). In place, or into ``out``: tensors of the gradients'
    shapes, strides and types, such as the pieces of an optimizer's buffer. None entries are skipped
    in both. Gradients whose norm is not finite are left (or copied) as they are. A gradient that
    occurs twice, and outputs that overlap, raise."""
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError("max_norm must not be negative or NaN")
    if out is not None:
        if len(out) != len(grads) or any((g is None) != (o is None) for g, o in zip(grads, out)):
            raise ValueError("out must match the gradients one by one")
        out = [o for o in out if o is not None]
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("no gradients")
    if out is not None:
        _tensors(out, "out")
        for g, o in zip(grads, out):
            if o.shape != g.shape or o.dtype != g.dtype or o.device != g.device:
                raise ValueError(f"out must match its gradient: {tuple(g.shape)} {g.dtype} on {g.device}, "
                                 f"got {tuple(o.shape)} {o.dtype} on {o.device}")
            if o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
                raise ValueError("out must have its gradient's strides")
    return _call(grads, max_norm, grads if out is None else out)
