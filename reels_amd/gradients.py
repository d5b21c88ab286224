"""Global norm of the adapters' gradients and clipping by it, between ``i8lora_backward`` and the
optimizer (the reference's training loop, src/training/wan_runner.jl:108-289), over
``reels_hip_grad_norm`` and ``reels_hip_clip_gradients``.
"""
from __future__ import annotations

import math
from array import array
from operator import attrgetter
from typing import Optional, Sequence

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .layers import _DTYPE_CODE, _launch, _need_device, _stream


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


# A call's host time is that of these loops, 25 to 50 ns a tensor for each property that is read (800
# tensors and their outputs: 0.74 ms with a statement for each check, 0.22 ms alone to compare their
# shapes), so every property is read once, by one map over the list.
_T = torch.Tensor
_dtype = attrgetter("dtype")


def _tensors(ts, name):
    """(types, sizes, whether all are contiguous) of a list of tensors on one device."""
    if not all(issubclass(c, _T) for c in set(map(type, ts))):
        raise TypeError(f"{name} must be tensors")
    types = list(map(_dtype, ts))
    for d in set(types):
        if d not in _DTYPE_CODE:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {d}")
    devices = set(map(_T.get_device, ts))
    if -1 in devices:
        for t in ts:
            _need_device(t, name)
    if len(devices) > 1:
        raise ValueError(f"{name} lie on several devices")
    return types, array("q", map(_T.numel, ts)), all(map(_T.is_contiguous, ts))


def _pointers(ts):
    return array("q", map(_T.data_ptr, ts))


def _call(grads, checked, max_norm, out):
    types, sizes, contiguous = checked
    if not contiguous and not all(map(_dense, grads)):
        raise ValueError("gradients must be dense")
    dev, n = grads[0].device, len(grads)
    ptrs, codes = _pointers(grads), array("i", map(_DTYPE_CODE.__getitem__, types))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = _lib.lib().reels_hip_grad_workspace_bytes(n)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    of, to = ptrs.buffer_info()[0], (sizes.buffer_info()[0], codes.buffer_info()[0], n)
    end = (norm.data_ptr(), ws.data_ptr(), nbytes, _stream(dev))
    if max_norm is None:
        _launch("reels_hip_grad_norm", dev, of, *to, *end)
    else:
        outs = ptrs if out is None else _pointers(out)
        _launch("reels_hip_clip_gradients", dev, of, outs.buffer_info()[0], *to, max_norm, *end)
        # the kernel writes behind torch's back: a graph that has saved one of these has to see it (50 ns
        # a tensor, while the kernels run)
        increment_version(grads if out is None else out)
    return norm


def _none_at(ts):
    """The places of None, looked for only where the list's types have it."""
    return [i for i, t in enumerate(ts) if t is None] if type(None) in set(map(type, ts)) else []


def _without_none(ts):
    return [t for t in ts if t is not None]


def gradient_norm(grads: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """sqrt of the sum of squares of all elements of all tensors (None entries are skipped), float32
    on their device; the sum runs in 64 bits."""
    grads = _without_none(grads)
    if not grads:
        raise ValueError("no gradients")
    return _call(grads, _tensors(grads, "gradients"), None, None)


def clip_gradients(grads: Sequence[Optional[torch.Tensor]], max_norm: float,
                   out: Optional[Sequence[Optional[torch.Tensor]]] = None) -> torch.Tensor:
    """Multiplies the gradients by min(1, max_norm / (norm + 1e-6)), norm their ``gradient_norm``,
    which it returns (without waiting for it). In place, or into ``out``: tensors of the gradients'
    sizes and types (and, where they are not contiguous, shapes and strides), such as the pieces of an
    optimizer's buffer. None entries are skipped in both. Gradients whose norm is not finite in float32
    are left (or copied) as they are. Outputs that overlap each other or another gradient raise, a
    gradient that is given twice to be clipped in place among them. Tensors that are written count as
    changed in place (a replay of a captured call does not count)."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError("max_norm must not be negative or NaN")
    grads = list(grads)
    none = _none_at(grads)
    if out is not None:
        out = list(out)
        if len(out) != len(grads) or _none_at(out) != none:
            raise ValueError("out must match the gradients one by one")
    if none:
        grads, out = _without_none(grads), None if out is None else _without_none(out)
    if not grads:
        raise ValueError("no gradients")
    checked = _tensors(grads, "gradients")
    if out is not None:
        types, sizes, contiguous = _tensors(out, "out")
        if types != checked[0] or sizes != checked[1] or out[0].device != grads[0].device:
            raise ValueError("out must have its gradients' sizes and types, on their device")
        if not (contiguous and checked[2]) and any(
                (o.shape != g.shape or o.stride() != g.stride())
                and not (o.is_contiguous() and g.is_contiguous()) for o, g in zip(out, grads)):
            raise ValueError("out must have its gradients' strides")
    return _call(grads, checked, max_norm, out)
