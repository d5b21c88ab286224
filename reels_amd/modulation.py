"""The norm between two sublayers of a transformer block, its output modulated by the conditioning, with
the gated residual before it (modulation, src/layers/modulation.jl:2-11; layernorm, src/layers/linear.jl;
rmsnorm, src/layers/normalization.jl:10-24), over ``reels_hip_modulated_norm*``.

Rows are the last dimension of ``[B, ..., C]`` or ``[M, C]``; bfloat16, float16 or float32, C up to 16384.
gate, scale and shift are in the rows' type or in float32 and all of one kind: one row for all rows
(``[C]``), one for each sample (``[B, C]`` or ``[B, 1, .., C]``, rows of three dimensions or more), or one
for each row (the rows' shape); slices of a larger tensor are taken as they lie where their rows are
whole. Every call runs the HIP kernels on the current stream of the rows' device; CPU tensors raise.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib, activations, microscaled
from .activations import CompressedActivations
from .layers import _DTYPE_CODE, _act_dtype, _contig, _launch, _ptr, _stream
from .microscaled import MicroscaledMatrix
from .normalization import _like, _rows, _same_device

_MOST = 16384


class KeptRows(NamedTuple):
    sum: CompressedActivations
    branch: Optional[CompressedActivations]


class ModulatedNormResult(NamedTuple):
    output: torch.Tensor         # [..., C]
    sum: torch.Tensor            # [..., C] x + gate * branch, what was normed (x itself without a branch)
    stats: torch.Tensor          # [..., 3] float32: the mean in two parts and 1 / the spread
    kept: Optional[KeptRows]     # the sum and the branch in 8 bits, with compress


class ModulatedNormQuantized(NamedTuple):
    output: MicroscaledMatrix    # [M][C]
    sum: torch.Tensor            # [..., C]


class ModulatedNormGradients(NamedTuple):
    x: torch.Tensor
    branch: torch.Tensor              # without a gate the same tensor as x
    gate: Optional[torch.Tensor]      # float32, of the modulations' shapes
    scale: Optional[torch.Tensor]
    shift: Optional[torch.Tensor]     # of scale's shape


def _groups(shape, mod, name):
    """How many rows a modulation of shape `mod` has for rows of `shape`: 1, one for each sample, or one each."""
    C = shape[-1]
    if mod == shape:
        return math.prod(shape[:-1])
    if mod == (C,) or (len(shape) == 2 and mod == (1, C)):
        return 1
    if len(shape) > 2 and mod in ((shape[0], C), (shape[0],) + (1,) * (len(shape) - 2) + (C,)):
        return shape[0]
    raise ValueError(f"{name} must have shape {(C,)}, one row for each sample or the rows' shape {tuple(shape)}, "
                     f"got {tuple(mod)}")


@functools.lru_cache(maxsize=4096)  # a function of shapes and types alone
def _kind(shape, dt, mods):
    """(type code, rows of a group) of modulations given as (name, shape, type) or None."""
    G, mt, first = None, dt, None
    for m in mods:
        if m is None:
            continue
        name, mod, t = m
        n = _groups(shape, mod, name)
        if t != dt and t != torch.float32:
            raise TypeError(f"{name} must be {dt} or float32, got {t}")
        if G is None:
            G, mt, first = n, t, name
        elif n != G or t != mt:
            raise ValueError(f"gate, scale and shift must be of one kind and type; {name} is {tuple(mod)} "
                             f"{t}, unlike {first}")
    M = math.prod(shape[:-1])
    return _DTYPE_CODE[mt], max(M // G, 1) if G else max(M, 1)


def _modulations(x, dt, mods):
    """([tensor or None, row stride] for each modulation one after the other, type code, rows of a group). mods:
    (tensor or None, name) pairs. The tensors hold the memory until the launch."""
    shape, dev = x.shape, x.device
    C = shape[-1]
    code, rpg = _kind(shape, dt, tuple([None if t is None else (name, t.shape, t.dtype) for t, name in mods]))
    out = []
    for t, name in mods:
        if t is None:
            out += (None, C)
            continue
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the rows on {dev}")
        ld = C
        if not t.is_contiguous():
            G = _groups(shape, t.shape, name)
            t = t.reshape(G, C)
            if C > 1 and t.stride(1) != 1:
                t = t.contiguous()
            ld = t.stride(0) if G > 1 else C
        out += (t, ld)
    return out, code, rpg


@functools.lru_cache(maxsize=4096)  # a function of the sizes alone
def _workspace_bytes(rows, cols, rows_per_group):
    return _lib.lib().reels_hip_modulated_norm_workspace_bytes(rows, cols, rows_per_group)


def _gradient_of(t):
    if t.dtype == torch.float32 and t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=torch.float32, device=t.device)


def _check_rows(x, name):
    dt = _act_dtype(x, name)
    if x.dim() < 2 or not 1 <= x.shape[-1] <= _MOST:
        raise ValueError(f"{name} must be [..., C] with C from 1 to {_MOST}, got shape {tuple(x.shape)}")
    return dt


def _beside(t, like, dt, name):
    if t is None:
        return
    if t.shape != like.shape:
        raise ValueError(f"{name} must have shape {tuple(like.shape)}, got {tuple(t.shape)}")
    if t.dtype != dt:
        raise TypeError(f"{name} must be {dt}, got {t.dtype}")
    _same_device(t, like, name)


def _operands(x, scale, shift, branch, gate, eps):
    """(type, the C arguments up to eps, the sum, x as it is read, the tensors that the arguments point into)."""
    dt = _check_rows(x, "x")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift must be given together")
    if gate is not None and branch is None:
        raise ValueError("a gate needs a branch")
    _beside(branch, x, dt, "branch")
    held, code, rpg = _modulations(x, dt, ((gate, "gate"), (scale, "scale"), (shift, "shift")))
    C = x.shape[-1]
    xr, ld_x = _rows(x, C)
    br, ld_b = (None, C) if branch is None else _rows(branch, C)
    gt, ld_g, sc, ld_sc, sh, ld_sh = held
    args = (xr.data_ptr(), ld_x, _ptr(br), ld_b, _ptr(gt), ld_g, _ptr(sc), ld_sc, _ptr(sh), ld_sh, code,
            _DTYPE_CODE[dt], x.numel() // C, C, rpg, eps)
    return dt, args, x if branch is None else _like(x, xr), xr, (br, held)


def modulated_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                   branch: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, center: bool = True, compress: bool = False) -> ModulatedNormResult:
    """s = x + gate * branch (rounded to the type; x + branch without a gate), output = (s - mean) /
    sqrt(mean((s - mean)^2) + eps) * (1 + scale) + shift, rounded once; mean = 0 with center=False (the
    root-mean-square norm). Without a branch ``sum`` is x itself. With compress the sum and the branch also
    come back in 8 bits, for a backward that does not keep the tensors themselves."""
    dt, args, s, xr, held = _operands(x, scale, shift, branch, gate, eps)
    dev = x.device
    y = _like(x, xr)
    stats = torch.empty((*x.shape[:-1], 3), dtype=torch.float32, device=dev)
    kept, ptrs = None, (None,) * 4
    if compress:
        a = activations._empty(x, dt)
        b = None if branch is None else activations._empty(x, dt)
        kept = KeptRows(a, b)
        ptrs = (a.values.data_ptr(), a.scales.data_ptr()) + (
            (None, None) if b is None else (b.values.data_ptr(), b.scales.data_ptr()))
    _launch("reels_hip_modulated_norm", dev, *args, int(center), None if branch is None else s.data_ptr(),
            y.data_ptr(), stats.data_ptr(), *ptrs, _stream(dev))
    del held
    return ModulatedNormResult(y, s, stats, kept)


def modulated_norm_quantized(x: torch.Tensor, scale: Optional[torch.Tensor] = None,
                             shift: Optional[torch.Tensor] = None, branch: Optional[torch.Tensor] = None,
                             gate: Optional[torch.Tensor] = None, eps: float = 1e-6,
                             center: bool = True) -> ModulatedNormQuantized:
    """The same norm with its rows ``[M][C]`` in microscaled 4 bits, tagged with x's type;
    ``microscaled_linear`` takes them. The values are formed in 64 bits before they are rounded."""
    dt, args, s, _, held = _operands(x, scale, shift, branch, gate, eps)
    dev, C = x.device, x.shape[-1]
    q = microscaled._empty(x.numel() // C, C, dt, dev)
    _launch("reels_hip_modulated_norm_mx4", dev, *args, int(center), None if branch is None else s.data_ptr(),
            q.codes.data_ptr(), q.scales.data_ptr(), _stream(dev))
    del held
    return ModulatedNormQuantized(q, s)


def modulated_norm_backward(dy: torch.Tensor, s: Union[torch.Tensor, CompressedActivations], stats: torch.Tensor,
                            scale: Optional[torch.Tensor] = None,
                            branch: Union[None, torch.Tensor, CompressedActivations] = None,
                            gate: Optional[torch.Tensor] = None, dsum: Optional[torch.Tensor] = None,
                            center: bool = True, want_modulation: bool = True) -> ModulatedNormGradients:
    """Gradients of ``modulated_norm`` from its ``sum`` (or the kept one) and ``stats``: of x, with ``dsum``,
    the gradient that reaches the sum from elsewhere, added before the one rounding; of the branch (x's times
    the gate); and, unless want_modulation is False, of scale, shift and (where the branch is given, kept
    like s) gate, summed in float32 over the rows that share them."""
    dt = _check_rows(dy, "dy")
    if s.shape != dy.shape:
        raise ValueError(f"s must have shape {tuple(dy.shape)}, got {tuple(s.shape)}")
    kept = isinstance(s, CompressedActivations)
    dev, C = dy.device, dy.shape[-1]
    want_gate = want_modulation and gate is not None and branch is not None
    if want_gate and isinstance(branch, CompressedActivations) != kept:
        raise ValueError("s and branch must both be kept in 8 bits or neither")
    scales = [None, None]
    if kept:
        s = activations._checked(s, "s")
        _same_device(s, dy, "s")
        s, scales[0] = s.values, s.scales
        if want_gate:
            if branch.shape != dy.shape:
                raise ValueError(f"branch must have shape {tuple(dy.shape)}, got {tuple(branch.shape)}")
            branch = activations._checked(branch, "branch")
            _same_device(branch, dy, "branch")
            branch, scales[1] = branch.values, branch.scales
    else:
        _beside(s, dy, dt, "s")
        if want_gate:
            _beside(branch, dy, dt, "branch")
            branch = branch.contiguous()
        s = s.contiguous()
    _beside(dsum, dy, dt, "dsum")
    if stats.shape[-1:] != (3,) or stats.shape[:-1] != dy.shape[:-1]:
        raise ValueError(f"stats must have shape {tuple(dy.shape[:-1]) + (3,)}, got {tuple(stats.shape)}")
    _same_device(stats, dy, "stats")
    held, code, rpg = _modulations(dy, dt, ((gate, "gate"), (scale, "scale")))
    gt, ld_g, sc, ld_sc = held
    dy, stats = dy.contiguous(), _contig(stats, torch.float32, "stats")
    dsum = None if dsum is None else dsum.contiguous()
    M = dy.numel() // C
    dx = torch.empty_like(dy)
    db = dx if gate is None else torch.empty_like(dy)

    dgate = _gradient_of(gate) if want_gate else None
    dscale = dshift = None
    if want_modulation and scale is not None:
        dscale, dshift = _gradient_of(scale), _gradient_of(scale)
    ws, nbytes = None, 0
    if dgate is not None or dscale is not None:
        if M == 0:
            for t in (dgate, dscale, dshift):
                if t is not None:
                    t.zero_()
        nbytes = _workspace_bytes(M, C, rpg)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
    _launch("reels_hip_modulated_norm_bwd", dev, _ptr(dy), _ptr(s), _ptr(scales[0]), _ptr(dsum),
            _ptr(branch) if want_gate else None, _ptr(scales[1]), _ptr(gt), ld_g, _ptr(sc), ld_sc, _ptr(stats), code, _DTYPE_CODE[dt], M, C, rpg,
            int(center), _ptr(dx), None if gate is None else _ptr(db), _ptr(dgate), _ptr(dscale), _ptr(dshift),
            _ptr(ws), nbytes, _stream(dev))
    return ModulatedNormGradients(dx, db, dgate, dscale, dshift)


class ModulatedNormFunction(torch.autograd.Function):
    """Autograd rule: ``y = ModulatedNormFunction.apply(x, scale, shift, None, None, eps, center, compress)``,
    or with a branch ``y, s = ...apply(x, scale, shift, branch, gate, ...)`` and s the sum. With compress the
    sum and the branch are kept in 8 bits. The modulations' gradients come back in their own type."""

    @staticmethod
    def forward(ctx, x, scale, shift, branch, gate, eps=1e-6, center=True, compress=False):
        ctx.set_materialize_grads(False)
        r = modulated_norm(x, scale, shift, branch, gate, eps, center, compress)
        ctx.dtype, ctx.center, ctx.compress = x.dtype, center, compress
        held = branch if gate is not None and ctx.needs_input_grad[4] else None
        if compress:
            k = r.kept
            b = (None, None) if held is None else (k.branch.values, k.branch.scales)
            ctx.save_for_backward(k.sum.values, k.sum.scales, *b, r.stats, scale, gate)
        else:
            ctx.save_for_backward(r.sum, None, held, None, r.stats, scale, gate)
        ctx.shift_dtype, ctx.shift_shape = (None, None) if shift is None else (shift.dtype, shift.shape)
        return r.output if branch is None else (r.output, r.sum)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        s, ss, b, bs, stats, scale, gate = ctx.saved_tensors
        if dy is None and dsum is None:
            return (None,) * 8
        if ctx.compress:
            s = CompressedActivations(s, ss, ctx.dtype)
            b = None if b is None else CompressedActivations(b, bs, ctx.dtype)
        need = ctx.needs_input_grad
        if dy is None:
            # Nothing reaches the norm: the sum's gradient alone, whatever the sum holds. With 1 / the spread at 0 and
            # finite rows in the sum's place the norm adds zeros.
            dy, s, stats = torch.zeros_like(dsum), dsum, torch.zeros_like(stats)
            b = b.restore() if isinstance(b, CompressedActivations) else b
        g = modulated_norm_backward(dy, s, stats, scale, b, gate, dsum, ctx.center,
                                    want_modulation=need[1] or need[2] or need[4])

        def of(t, like, want):
            return t.to(like) if want and t is not None else None
        # scale and shift of one kind can differ in shape ([B, C] beside [B, 1, C])
        dshift = None if g.shift is None else g.shift.view(ctx.shift_shape)
        return (g.x, of(g.scale, None if scale is None else scale.dtype, need[1]), of(dshift, ctx.shift_dtype, need[2]),
                g.branch if need[3] else None, of(g.gate, None if gate is None else gate.dtype, need[4]),
                None, None, None)
