"""Rotary positions over several axes (time, height, width of a video's patches), ``_rope!`` of
src/layers/rope.jl:13-32, over ``reels_hip_rotary``.

Queries and keys are ``[B][S][H][D]`` as in ``memory_efficient_attention``; positions are
``[S][axes]`` for every batch or ``[B][S][axes]``, int32 or float32 (fractions are fine). ``axes``
gives the pairs of each axis in order: ``rotary_axes(D)`` is the video model's split.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .layers import _DTYPE_CODE, _act_dtype, _launch, _ptr, _stream

_POS = {torch.float32: _lib.F32, torch.int32: _lib.I32}


def rotary_axes(head_dim: int) -> Tuple[int, int, int]:
    """Pairs of time, height and width: a third of the head's pairs (rounded down) for height and
    for width each, the rest for time (22, 21, 21 at head dim 128)."""
    if head_dim < 2 or head_dim % 2:
        raise ValueError(f"head_dim must be even and positive, got {head_dim}")
    pairs = head_dim // 2
    return pairs - 2 * (pairs // 3), pairs // 3, pairs // 3


def grid_positions(frames: int, height: int, width: int, device=None) -> torch.Tensor:
    """Positions ``[frames * height * width][3]`` (int32) of a grid of patches in its token order."""
    t, h, w = (torch.arange(n, dtype=torch.int32, device=device) for n in (frames, height, width))
    return torch.stack(torch.meshgrid(t, h, w, indexing="ij"), dim=-1).reshape(-1, 3)


@functools.lru_cache(maxsize=256)
def _pairs(axes: Tuple[int, ...], D: int):
    """The C array of the axes' pairs, checked against the head dim."""
    if not 1 <= len(axes) <= 4 or min(axes) < 0 or 2 * sum(axes) > D:
        raise ValueError(f"axes must be one to four numbers of pairs, together at most {D // 2}, got {axes}")
    return (ctypes.c_int32 * len(axes))(*axes)


def _tokens(t: torch.Tensor):
    """(tensor, token stride): heads that lie together are taken as they are, as the thirds of one
    fused projection do."""
    B, S, H, D = t.shape
    if t.is_contiguous():
        return t, H * D
    ld = t.stride(1) if S > 1 else (t.stride(0) if B > 1 else H * D)
    if ((t.stride(3) == 1 or D == 1) and (H == 1 or t.stride(2) == D) and ld >= H * D
            and (B == 1 or t.stride(0) == S * ld)):
        return t, ld
    return t.contiguous(), H * D


def _like(t, taken):
    return torch.empty_like(taken) if taken.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rotate(q, k, positions, axes, theta, interleaved, inverse):
    dt = _act_dtype(q, "q")
    if q.dim() != 4:
        raise ValueError(f"q must be 4-d [batch][tokens][heads][head_dim], got {tuple(q.shape)}")
    B, S, Hq, D = q.shape
    Hk = 0
    if k is not None:
        if k.dim() != 4 or k.shape != (B, S, k.shape[2], D):
            raise ValueError(f"k must be [{B}][{S}][heads][{D}], got {tuple(k.shape)}")
        if k.dtype != dt or k.device != q.device:
            raise TypeError(f"k must be {dt} on {q.device}, got {k.dtype} on {k.device}")
        Hk = k.shape[2]
    if D < 2 or D % 2 or D > 512:
        raise ValueError(f"head_dim must be even and at most 512, got {D}")
    axes = tuple(axes)
    pairs, n = _pairs(axes, D), len(axes)
    if not 0 < theta < math.inf:
        raise ValueError("theta must be finite and positive")
    if positions.dtype not in _POS:
        raise TypeError(f"positions must be int32 or float32, got {positions.dtype}")
    if positions.device != q.device:
        raise ValueError(f"positions are on {positions.device}, q on {q.device}")
    ps = positions.shape
    if not (ps == (S, n) or ps == (1, S, n) or ps == (B, S, n)):
        raise ValueError(f"positions must be [{S}][{n}] or [{B}][{S}][{n}], got {tuple(ps)}")
    p = positions.contiguous()
    qr, ld_q = _tokens(q)
    yq = _like(q, qr)
    kr, ld_k, yk = None, 0, None
    if k is not None:
        kr, ld_k = _tokens(k)
        yk = _like(k, kr)
    _launch("reels_hip_rotary", q.device, _ptr(qr), ld_q, _ptr(kr), ld_k, _ptr(p), _POS[p.dtype],
            1 if len(ps) == 2 else ps[0], _DTYPE_CODE[dt], B, S, Hq, Hk, D, pairs, n, theta,
            int(bool(interleaved)), inverse, _ptr(yq), _ptr(yk), _stream(q.device))
    return yq, yk


def rotary(x: torch.Tensor, positions: torch.Tensor, axes: Sequence[int], theta: float = 10000.0,
           interleaved: bool = True) -> torch.Tensor:
    """x with pair j of axis a turned by ``positions[..., a] * theta ** (-j / axes[a])``. The pairs
    of an axis follow those of the axis before it; pair p is elements 2p and 2p + 1 of a head, or
    with interleaved=False elements p and p + sum(axes). Elements past 2 sum(axes) are copied. theta
    is taken as a float32 value."""
    return _rotate(x, None, positions, axes, theta, interleaved, 0)[0]


def rotary_backward(dy: torch.Tensor, positions: torch.Tensor, axes: Sequence[int],
                    theta: float = 10000.0, interleaved: bool = True) -> torch.Tensor:
    """The gradient of ``rotary``'s input: dy turned back."""
    return _rotate(dy, None, positions, axes, theta, interleaved, 1)[0]


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes: Sequence[int],
              theta: float = 10000.0, interleaved: bool = True):
    """``rotary`` of the queries and the keys of one attention in one launch; k may have another
    number of heads."""
    return _rotate(q, k, positions, axes, theta, interleaved, 0)


def rotary_qk_backward(dq: torch.Tensor, dk: torch.Tensor, positions: torch.Tensor,
                       axes: Sequence[int], theta: float = 10000.0, interleaved: bool = True):
    """The gradients of ``rotary_qk``'s inputs."""
    return _rotate(dq, dk, positions, axes, theta, interleaved, 1)


class RotaryFunction(torch.autograd.Function):
    """Autograd rule: ``yq, yk = RotaryFunction.apply(q, k, positions, axes, theta, interleaved)``;
    k (and yk) may be None."""

    @staticmethod
    def forward(ctx, q, k, positions, axes, theta=10000.0, interleaved=True):
        ctx.save_for_backward(positions)
        ctx.args = (tuple(axes), theta, interleaved)
        return _rotate(q, k, positions, axes, theta, interleaved, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq, dk = _rotate(dq, dk, positions, *ctx.args, 1)
        return dq, dk, None, None, None, None
