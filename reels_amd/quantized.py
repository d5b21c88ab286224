"""Activations in 8 bits: rows quantised with one scale each, and their product with a packed int8
weight, over ``reels_hip_i8_pack`` and ``reels_hip_i8i8_linear``. For sampling: where the int8
linears multiply 16-bit activations, this multiplies codes with codes at twice the rate. It has no
gradient of its own; the frozen weight's pullback is ``_weight_transpose_mul``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .layers import (_DTYPE_CODE, QuantizedMatrix, _act_dtype, _check_codes, _check_shape, _contig,
                     _launch, _need_device, _on_activation_device, _ptr, _stream)

_ACTIVATIONS = {None: _lib.ACT_NONE, "gelu_tanh": _lib.ACT_GELU_TANH}


def quantize_rows(x: torch.Tensor) -> QuantizedMatrix:
    """The rows of an activation matrix ``[M][K]`` as int8 codes with one scale each, by
    ``quantize_frozen_matrix``'s formula but without its check (and its wait) for values that are
    not finite: a row that holds one has zero codes and the scale NaN or Inf, so its values are NaN."""
    dt = _act_dtype(x, "x")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be a [M][K] matrix, got shape {tuple(x.shape)}")
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    M, K = x.shape
    values = torch.empty((M, K), dtype=torch.int8, device=x.device)
    scales = torch.empty((M,), dtype=torch.float32, device=x.device)
    _launch("reels_hip_i8_pack", x.device, _ptr(x), _DTYPE_CODE[dt], M, K, max(x.stride(0), K),
            _ptr(values), _ptr(scales), None, _stream(x.device))
    return QuantizedMatrix(values, scales, dt)


def quantized_linear(x: QuantizedMatrix, weight: QuantizedMatrix,
                     bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                     residual: Optional[torch.Tensor] = None,
                     dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """activation(deq(x) deq(weight)^T + bias) + residual, rounded once: x ``[M][K]`` from
    ``rms_norm_quantized`` or ``quantize_rows``, weight ``[N][K]``, bias ``[N]`` and residual
    ``[M][N]`` in the result's type (x's compute type unless dtype says otherwise), activation None
    or "gelu_tanh". The sum over K is exact (K < 131072)."""
    _check_codes(x)
    _check_codes(weight)
    M, K = x.values.shape
    N, Kw = weight.values.shape
    if Kw != K:
        raise ValueError("DimensionMismatch: input and weight dimensions differ")
    if K < 1 or K >= 1 << 17 or N < 1:
        raise ValueError(f"K must be between 1 and 131071 and N positive, got {K} and {N}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'gelu_tanh', got {activation!r}")
    dt = dtype or x.compute_dtype
    if dt not in _DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dt}")
    _check_shape(bias, (N,), "bias")
    _check_shape(residual, (M, N), "residual")
    _need_device(x.values, "x")
    dev = x.values.device
    x = _on_activation_device(x, dev)
    weight = _on_activation_device(weight, dev)
    for t, n in ((bias, "bias"), (residual, "residual")):
        if t is not None and t.device != dev:
            raise ValueError(f"{n} is on {t.device}, the rows on {dev}")
    bias, residual = _contig(bias, dt, "bias"), _contig(residual, dt, "residual")
    y = torch.empty((M, N), dtype=dt, device=dev)
    px, pw = x.values.data_ptr(), weight.values.data_ptr()
    ws, nbytes = None, 0
    if (K | px | pw) & 3:  # zero-padded copies of the codes
        nbytes = _lib.lib().reels_hip_i8i8_workspace_bytes(M, K, N)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    _launch("reels_hip_i8i8_linear", dev, px, _ptr(x.scales), pw, _ptr(weight.scales), _ptr(bias),
            _ptr(residual), _ACTIVATIONS[activation], _DTYPE_CODE[dt], M, K, N, _ptr(y), _ptr(ws),
            nbytes, _stream(dev))
    return y
