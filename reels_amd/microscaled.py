"""Rows in microscaled 4 bits and their product, over ``reels_hip_mx4_*``. For sampling, as the product
of int8 rows (``quantized_linear``) is, with half the bytes and on the 4-bit rate of the matrix cores:
blocks of 32 neighbours of a row share a power of two, an element is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
with a sign. It has no gradient.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .layers import _DTYPE_CODE, _act_dtype, _check_shape, _contig, _launch, _need_device, _ptr, _stream
from .quantized import _ACTIVATIONS

_BLOCK, _TILE = 32, 256


def _padded(K: int) -> int:
    return -(-K // _TILE) * _TILE


@functools.lru_cache(maxsize=4096)
def _layout(M: int, K: int):
    """Shapes of the codes and of the scales."""
    return (M, _padded(K) // 2), (-(-M // 64), _padded(K) // _TILE, 512)


@dataclass
class MicroscaledMatrix:
    """A matrix ``[M][K]`` in 4 bits. codes: uint8 ``[M][Kp / 2]``, K padded with zeros to a multiple of
    256, the even column in the low half of a byte. scales: uint8 ``[ceil(M / 64)][Kp / 256][512]``, the
    exponent + 127 of each block's power of two (255: the block held NaN or an infinity, its values are
    NaN), in the order in which the matrix cores take them (``block_scales`` gives them by rows; what stands
    in the places of rows past M is never used).
    compute_dtype: the type of what is made from it."""

    codes: torch.Tensor
    scales: torch.Tensor
    size: Tuple[int, int]
    compute_dtype: torch.dtype = torch.bfloat16

    @property
    def shape(self):
        return tuple(self.size)

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values ``[M][K]`` (exact in bfloat16 and float32)."""
        dt = dtype or self.compute_dtype
        if dt not in _DTYPE_CODE:
            raise TypeError(f"unsupported dtype {dt}")
        q = _checked(self, "the matrix")
        M, K = q.shape
        y = torch.empty((M, K), dtype=dt, device=q.device)
        _launch("reels_hip_mx4_unpack", q.device, _ptr(q.codes), _ptr(q.scales), _DTYPE_CODE[dt], M, K,
                _ptr(y), _stream(q.device))
        return y

    def block_scales(self) -> torch.Tensor:
        """The scales by rows, uint8 ``[M][ceil(K / 32)]``."""
        M, K = self.shape
        tiles = self.scales.reshape(-1, _padded(K) // _TILE, 2, 32, 4, 2).permute(0, 5, 3, 1, 4, 2)
        return tiles.reshape(-1, _padded(K) // _BLOCK)[:M, :-(-K // _BLOCK)].contiguous()

    @staticmethod
    def from_blocks(codes: torch.Tensor, scales: torch.Tensor, K: int,
                    compute_dtype: torch.dtype = torch.bfloat16) -> "MicroscaledMatrix":
        """From codes uint8 ``[M][ceil(K / 2)]`` and scales uint8 ``[M][ceil(K / 32)]`` by rows, as checkpoints
        hold them. The codes past an odd K have to be zero."""
        M = codes.shape[0] if codes.dim() == 2 else -1
        for t, n, w in ((codes, "codes", -(-K // 2)), (scales, "scales", -(-K // _BLOCK))):
            if K < 1 or t.dtype != torch.uint8 or tuple(t.shape) != (M, w):
                raise ValueError(f"{n} must be a uint8 matrix [M][{w}], got {t.dtype} {tuple(t.shape)}")
        pad, Kp = torch.nn.functional.pad, _padded(K)
        s = pad(scales, (0, Kp // _BLOCK - scales.shape[1], 0, -M % 64))
        s = s.view(-1, 2, 32, Kp // _TILE, 4, 2).permute(0, 3, 5, 2, 4, 1).reshape(-1, Kp // _TILE, 512)
        return MicroscaledMatrix(pad(codes, (0, Kp // 2 - codes.shape[1])).contiguous(), s.contiguous(), (M, K),
                                 compute_dtype)


def _checked(q: MicroscaledMatrix, name: str) -> MicroscaledMatrix:
    """Types, shapes, device and alignment of the operand, dense."""
    M, K = q.size
    if M < 0 or K < 1:
        raise ValueError(f"{name} must have rows of at least one element, got size {(M, K)}")
    _need_device(q.codes, name)
    codes, scales = q.codes, q.scales
    want = _layout(M, K)
    if (codes.dtype != torch.uint8 or codes.shape != want[0] or scales.dtype != torch.uint8 or scales.shape != want[1]
            or scales.device != codes.device):
        raise ValueError(f"{name} must have uint8 codes and scales of shapes {want} on one device, got {codes.dtype} "
                         f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        codes, scales = codes.contiguous(), scales.contiguous()
    if (codes.data_ptr() | scales.data_ptr()) & 15:
        codes, scales = codes.clone(), scales.clone()
    return q if codes is q.codes and scales is q.scales else MicroscaledMatrix(codes, scales, q.size, q.compute_dtype)


def _empty(M: int, K: int, dtype, device) -> MicroscaledMatrix:
    codes, scales = _layout(M, K)
    return MicroscaledMatrix(torch.empty(codes, dtype=torch.uint8, device=device),
                             torch.empty(scales, dtype=torch.uint8, device=device), (M, K), dtype)


def quantize_microscaled(x: torch.Tensor) -> MicroscaledMatrix:
    """The rows of a matrix ``[M][K]`` (activations or a weight; bfloat16, float16 or float32) in 4
    bits: every block's power of two puts its largest magnitude, rounded to 2 significant bits, at 4 or
    6; each element goes to the nearest value, ties to the even code."""
    dt = _act_dtype(x, "x")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be a [M][K] matrix, got shape {tuple(x.shape)}")
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    M, K = x.shape
    q = _empty(M, K, dt, x.device)
    _launch("reels_hip_mx4_pack", x.device, _ptr(x), max(x.stride(0), K), _DTYPE_CODE[dt], M, K,
            _ptr(q.codes), _ptr(q.scales), _stream(x.device))
    return q


def microscaled_linear(x: MicroscaledMatrix, weight: MicroscaledMatrix,
                       bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                       residual: Optional[torch.Tensor] = None,
                       dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """activation(deq(x) deq(weight)^T + bias) + residual, rounded once: x ``[M][K]`` from
    ``modulated_norm_quantized`` or ``quantize_microscaled``, weight ``[N][K]``, bias ``[N]`` and residual
    ``[M][N]`` in the result's type (x's compute type unless dtype says otherwise), activation None or
    "gelu_tanh". Sums in float32."""
    x, weight = _checked(x, "x"), _checked(weight, "weight")
    (M, K), (N, Kw) = x.shape, weight.shape
    if Kw != K:
        raise ValueError("DimensionMismatch: input and weight dimensions differ")
    if N < 1:
        raise ValueError("the weight must have at least one row")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'gelu_tanh', got {activation!r}")
    dt = dtype or x.compute_dtype
    if dt not in _DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dt}")
    _check_shape(bias, (N,), "bias")
    _check_shape(residual, (M, N), "residual")
    dev = x.device
    for t, n in ((weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is not None and t.device != dev:
            raise ValueError(f"{n} is on {t.device}, the rows on {dev}")
    bias, residual = _contig(bias, dt, "bias"), _contig(residual, dt, "residual")
    y = torch.empty((M, N), dtype=dt, device=dev)
    _launch("reels_hip_mx4_linear", dev, _ptr(x.codes), _ptr(x.scales), _ptr(weight.codes),
            _ptr(weight.scales), _ptr(bias), _ptr(residual), _ACTIVATIONS[activation], _DTYPE_CODE[dt],
            M, K, N, _ptr(y), _stream(dev))
    return y
