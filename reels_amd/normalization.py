"""Root-mean-square norm of rows with the residual's addition, its int8 output and its backward
(rmsnorm, src/layers/normalization.jl:10-24) over ``reels_hip_rms_norm*``.

Rows are the last dimension of a tensor, ``[..., C]``, as in the linears; bfloat16, float16 or
float32, the weight in the rows' type or in float32. Every call runs the HIP kernels on the current
stream of the rows' device; CPU tensors raise.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .layers import _DTYPE_CODE, QuantizedMatrix, _act_dtype, _contig, _launch, _ptr, _stream


class RMSNormResult(NamedTuple):
    output: torch.Tensor   # [..., C] the normed rows
    sum: torch.Tensor      # [..., C] x + residual, what was normed (x itself without a residual)
    rstd: torch.Tensor     # [...] float32, what the backward takes


class RMSNormQuantized(NamedTuple):
    output: QuantizedMatrix  # values int8 [M][C], scales float32 [M]
    sum: torch.Tensor        # [M][C]


class RMSNormGradients(NamedTuple):
    x: torch.Tensor                  # of x, and of the residual
    weight: Optional[torch.Tensor]   # float32 [C]


def _rows(t: torch.Tensor, C: int):
    """(tensor, row stride): a matrix whose rows are contiguous is taken as it lies."""
    if t.is_contiguous():
        return t, C
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= C:
        return t, t.stride(0)
    return t.contiguous(), C


def _like(x, xr):
    return torch.empty_like(xr) if xr.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _operands(x, weight, residual, eps):
    dt = _act_dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one element, got shape {tuple(x.shape)}")
    C = x.shape[-1]
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype != dt:
            raise TypeError(f"residual must be {dt}, got {residual.dtype}")
        _same_device(residual, x, "residual")
    return dt, C, _weight(weight, C, dt, x)


def _same_device(t, x, name):
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, the rows on {x.device}")


def _weight(weight, C, dt, x):
    if weight is None:
        return None
    if weight.shape != (C,):
        raise ValueError(f"weight must have shape {(C,)}, got {tuple(weight.shape)}")
    if weight.dtype != dt and weight.dtype != torch.float32:
        raise TypeError(f"weight must be {dt} or float32, got {weight.dtype}")
    _same_device(weight, x, "weight")
    return weight.contiguous()


def _forward(x, weight, eps, residual, quantized):
    dt, C, weight = _operands(x, weight, residual, eps)
    dev = x.device
    M = x.numel() // C
    xr, ld_x = _rows(x, C)
    res, ld_r, s = None, C, x
    if residual is not None:
        res, ld_r = _rows(residual, C)
        s = _like(x, xr)
    if quantized:
        fn = "reels_hip_rms_norm_i8"
        out = torch.empty((M, C), dtype=torch.int8, device=dev)
        per_row = torch.empty((M,), dtype=torch.float32, device=dev)
    else:
        fn = "reels_hip_rms_norm"
        out = _like(x, xr)
        per_row = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    _launch(fn, dev, _ptr(xr), ld_x, _ptr(res), ld_r, _ptr(weight),
            _DTYPE_CODE[dt if weight is None else weight.dtype], _DTYPE_CODE[dt], M, C, eps,
            None if res is None else s.data_ptr(), out.data_ptr(), per_row.data_ptr(), _stream(dev))
    return out, s, per_row


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None) -> RMSNormResult:
    """s = x + residual (rounded to the type), output = s / sqrt(mean(s^2) + eps) * weight, each
    rounded once; also rstd = 1 / sqrt(mean(s^2) + eps) for ``rms_norm_backward``. Without a
    residual ``sum`` is x itself."""
    return RMSNormResult(*_forward(x, weight, eps, residual, False))


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       residual: Optional[torch.Tensor] = None) -> RMSNormQuantized:
    """The norm of a matrix ``[M][C]`` with its rows in 8 bits: symmetric codes with one scale per
    row, the layout of ``quantize_frozen_matrix``, tagged with x's type; ``quantized_linear`` takes
    it. A row that holds NaN or infinities has scale NaN."""
    if x.dim() != 2:
        raise ValueError(f"x must be a [M][C] matrix, got shape {tuple(x.shape)}")
    q, s, scales = _forward(x, weight, eps, residual, True)
    return RMSNormQuantized(QuantizedMatrix(q, scales, x.dtype), s)


def rms_norm_backward(dy: torch.Tensor, s: torch.Tensor, weight: Optional[torch.Tensor],
                      rstd: torch.Tensor, dsum: Optional[torch.Tensor] = None,
                      want_dweight: bool = True) -> RMSNormGradients:
    """Gradients of ``rms_norm`` from its ``sum`` and ``rstd``: of x (and of the residual, the same
    tensor), with ``dsum``, the gradient that reaches the sum from elsewhere, added before the one
    rounding; and of the weight in float32 unless want_dweight is False or there is none."""
    dt = _act_dtype(s, "s")
    if s.dim() < 1 or s.shape[-1] < 1:
        raise ValueError(f"s must have rows of at least one element, got shape {tuple(s.shape)}")
    C = s.shape[-1]
    for t, n in ((dy, "dy"), (dsum, "dsum")):
        if t is None:
            continue
        if t.shape != s.shape:
            raise ValueError(f"{n} must have shape {tuple(s.shape)}, got {tuple(t.shape)}")
        _same_device(t, s, n)
    if rstd.shape != s.shape[:-1]:
        raise ValueError(f"rstd must have shape {tuple(s.shape[:-1])}, got {tuple(rstd.shape)}")
    _same_device(rstd, s, "rstd")
    weight = _weight(weight, C, dt, s)
    dy, dsum, s = _contig(dy, dt, "dy"), _contig(dsum, dt, "dsum"), s.contiguous()
    rstd = _contig(rstd, torch.float32, "rstd")
    dev, M = s.device, s.numel() // C
    dx = torch.empty_like(s)
    dw, ws, nbytes = None, None, 0
    if want_dweight and weight is not None:
        dw = torch.empty((C,), dtype=torch.float32, device=dev)
        nbytes = _lib.lib().reels_hip_rms_norm_workspace_bytes(M, C)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    _launch("reels_hip_rms_norm_bwd", dev, _ptr(dy), _ptr(s), _ptr(dsum), _ptr(weight),
            _DTYPE_CODE[dt if weight is None else weight.dtype], _ptr(rstd), _DTYPE_CODE[dt], M, C,
            _ptr(dx), _ptr(dw), _ptr(ws), nbytes, _stream(dev))
    return RMSNormGradients(dx, dw)


class RMSNormFunction(torch.autograd.Function):
    """Autograd rule: ``y = RMSNormFunction.apply(x, weight, None, eps)``, or with a residual ``y, s =
    RMSNormFunction.apply(x, weight, residual, eps)`` and s the sum. The weight may be None; its
    gradient comes back in its own type."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps=1e-6):
        ctx.set_materialize_grads(False)
        r = rms_norm(x, weight, eps, residual)
        ctx.save_for_backward(r.sum, weight, r.rstd)
        return r.output if residual is None else (r.output, r.sum)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        s, weight, rstd = ctx.saved_tensors
        residual = ctx.needs_input_grad[2]
        if dy is None:  # nothing reaches the norm: the sum's gradient alone
            return dsum, None, (dsum if residual else None), None
        g = rms_norm_backward(dy, s, weight, rstd, dsum, want_dweight=ctx.needs_input_grad[1])
        dw = None if g.weight is None else g.weight.to(weight.dtype)
        return g.x, dw, (g.x if residual else None), None
