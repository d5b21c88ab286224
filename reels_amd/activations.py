"""Activations kept in 8 bits for the backward, over ``reels_hip_act8_*``.

What a trainer keeps of a block for its backward (the inputs of the linears with adapters, of the GELU,
the sums before the norms) takes 33 bytes for 32 elements here instead of 64: blocks of 32 neighbours
of a row share a power of two, each element has 7 bits and a sign. The forward computes with the
activations themselves; only the backward sees the rounded ones.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .layers import _DTYPE_CODE, _act_dtype, _contig, _launch, _need_device, _ptr, _stream, gelu_tanh_backward

_BLOCK = 32


@dataclass
class CompressedActivations:
    """A tensor ``[..., C]`` in 8 bits: values int8 of its shape, scales uint8 ``[..., ceil(C / 32)]``
    (the exponent + 127 of each block's power of two 2^E; a value is code * 2^(E - 6); 255: the block
    held NaN or an infinity, its values are NaN); compute_dtype: the tensor's own type."""

    values: torch.Tensor
    scales: torch.Tensor
    compute_dtype: torch.dtype = torch.bfloat16

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def reshape(self, *shape) -> "CompressedActivations":
        """Another shape with the same rows."""
        shape = tuple(shape[0]) if len(shape) == 1 and not isinstance(shape[0], int) else shape
        values = self.values.reshape(shape)
        if values.dim() < 1 or values.shape[-1] != self.values.shape[-1]:
            raise ValueError(f"rows must keep their length {self.values.shape[-1]}, got shape {tuple(values.shape)}")
        return CompressedActivations(values, self.scales.reshape(values.shape[:-1] + self.scales.shape[-1:]),
                                     self.compute_dtype)

    def restore(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values in the tensor's own type or another (exact in bfloat16 and float32)."""
        dt = dtype or self.compute_dtype
        if dt not in _DTYPE_CODE:
            raise TypeError(f"unsupported dtype {dt}")
        k = _checked(self, "the activations")
        M, C = _rows_of(k.values)
        out = torch.empty_like(k.values, dtype=dt)
        _launch("reels_hip_act8_restore", k.device, _ptr(k.values), _ptr(k.scales), _DTYPE_CODE[dt],
                M, C, _ptr(out), _stream(k.device))
        return out


def _rows_of(t: torch.Tensor) -> Tuple[int, int]:
    C = t.shape[-1]
    return t.numel() // C, C


def _checked(k: CompressedActivations, name: str) -> CompressedActivations:
    """Types, shapes and device of the codes, dense."""
    v, s = k.values, k.scales
    _need_device(v, name)
    if v.dtype != torch.int8 or v.dim() < 1 or v.shape[-1] < 1:
        raise ValueError(f"{name} must have int8 values with rows of at least one, got {v.dtype} {tuple(v.shape)}")
    want = _scales_shape(v.shape)
    if s.dtype != torch.uint8 or s.shape != want or s.device != v.device:
        raise ValueError(f"{name} must have uint8 scales of shape {want} on the values' device")
    if v.is_contiguous() and s.is_contiguous():
        return k
    return CompressedActivations(v.contiguous(), s.contiguous(), k.compute_dtype)


@functools.lru_cache(maxsize=4096)
def _scales_shape(shape):
    return tuple(shape[:-1]) + (-(-shape[-1] // _BLOCK),)


def _empty(x: torch.Tensor, dtype) -> CompressedActivations:
    values = (torch.empty_like(x, dtype=torch.int8) if x.is_contiguous()
              else torch.empty(x.shape, dtype=torch.int8, device=x.device))
    return CompressedActivations(values, torch.empty(_scales_shape(x.shape), dtype=torch.uint8, device=x.device), dtype)


def _input(x: torch.Tensor):
    dt = _act_dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one element, got shape {tuple(x.shape)}")
    return dt, x.contiguous()


def compress_activations(x: torch.Tensor) -> CompressedActivations:
    """x ``[..., C]`` in 8 bits (bfloat16, float16 or float32)."""
    dt, x = _input(x)
    k = _empty(x, dt)
    M, C = _rows_of(x)
    _launch("reels_hip_act8_keep", x.device, _ptr(x), _DTYPE_CODE[dt], M, C, _ptr(k.values),
            _ptr(k.scales), _stream(x.device))
    return k


def gelu_tanh_compressed(x: torch.Tensor) -> Tuple[torch.Tensor, CompressedActivations]:
    """(gelu_tanh(x), x in 8 bits) in one pass; ``gelu_tanh_backward`` takes the second."""
    dt, x = _input(x)
    k, y = _empty(x, dt), torch.empty_like(x)
    M, C = _rows_of(x)
    _launch("reels_hip_act8_gelu_tanh", x.device, _ptr(x), _DTYPE_CODE[dt], M, C, _ptr(y),
            _ptr(k.values), _ptr(k.scales), _stream(x.device))
    return y, k


def _gelu_backward(x: CompressedActivations, dy: torch.Tensor) -> torch.Tensor:
    """dy gelu_tanh'(values of x), in dy's type (what ``gelu_tanh_backward`` does with such an x)."""
    dt = _act_dtype(dy, "dy")
    x = _checked(x, "x")
    if dy.shape != x.shape:
        raise ValueError(f"dy must have shape {tuple(x.shape)}, got {tuple(dy.shape)}")
    if dy.device != x.device:
        raise ValueError(f"dy is on {dy.device}, the activations on {x.device}")
    dy = _contig(dy, dt, "dy")
    dx = torch.empty_like(dy)
    M, C = _rows_of(x.values)
    _launch("reels_hip_act8_gelu_tanh_bwd", x.device, _ptr(x.values), _ptr(x.scales), _ptr(dy),
            _DTYPE_CODE[dt], M, C, _ptr(dx), _stream(x.device))
    return dx


class GeluTanhCompressedFunction(torch.autograd.Function):
    """Autograd rule: ``y = GeluTanhCompressedFunction.apply(x)`` keeps x in 8 bits."""

    @staticmethod
    def forward(ctx, x):
        y, kept = gelu_tanh_compressed(x)
        ctx.save_for_backward(kept.values, kept.scales)
        ctx.dtype = kept.compute_dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return gelu_tanh_backward(CompressedActivations(*ctx.saved_tensors, ctx.dtype), dy)
