"""Rotary positions against the rotation in 64 bits. The angle's fraction is rounded to f32 (an error
of pi 2^-24 at most), sine and cosine are within two steps, and a rotated element is two products and
a sum: 9 u (|u| + |v|) before the rounding to the type."""
import math

import pytest
import torch

from reels_amd import (RotaryFunction, grid_positions, memory_efficient_attention, rms_norm, rotary,
                       rotary_axes, rotary_backward, rotary_qk, rotary_qk_backward)
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def rotated(x, positions, axes, theta, interleaved, sign=1):
    """(the rotation in 64 bits, |u| + |v| of each element's pair)"""
    x = x.double()
    p = positions.double()
    p = p[None] if p.dim() == 2 else p
    freq = [torch.tensor([math.pow(theta, -j / n) for j in range(n)], dtype=torch.float64, device=x.device)
            for n in axes]
    ang = torch.cat([p[..., a:a + 1] * f for a, f in enumerate(freq)], -1)[:, :, None, :]
    c, s = torch.cos(ang), sign * torch.sin(ang)
    P = sum(axes)
    ui, vi = ((slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P)))
    u, v = x[..., ui], x[..., vi]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., ui], y[..., vi] = u * c - v * s, u * s + v * c
    size[..., ui] = size[..., vi] = u.abs() + v.abs()
    return y, size


# batch, tokens, q heads, k heads, head dim, axes
CASES = [(1, 1, 1, 1, 2, (1,)), (1, 7, 3, 1, 32, (6, 5, 5)), (2, 33, 5, 5, 128, (22, 21, 21)),
         (1, 50, 4, 2, 64, (32,)), (3, 10, 2, 2, 100, (18, 16, 16)), (1, 9, 3, 3, 72, (12, 12, 12)),
         (2, 5, 2, 1, 80, (8, 8, 8)), (1, 6, 2, 2, 96, (0, 24, 24)), (1, 4, 1, 3, 512, (64, 64, 64, 64)),
         (1, 3, 2, 2, 66, (11, 11, 11)), (1, 5, 40, 40, 128, (22, 21, 21)), (1, 2, 3, 3, 16, (0, 0))]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,S,Hq,Hk,D,axes", CASES)
def test_rotation_and_its_backward(dev, B, S, Hq, Hk, D, axes, interleaved, dtype):
    g = torch.Generator(device=dev).manual_seed(D + S)
    q, k = (torch.randn(B, S, h, D, generator=g, device=dev).to(DT[dtype]) for h in (Hq, Hk))
    for shared in (True, False):
        shape = (S, len(axes)) if shared else (B, S, len(axes))
        for pos in (torch.randint(-40, 900, shape, generator=g, device=dev, dtype=torch.int32),
                    torch.rand(shape, generator=g, device=dev) * 1e4 - 2e3):
            kw = dict(axes=axes, theta=1e4, interleaved=interleaved)
            yq, yk = rotary_qk(q, k, pos, **kw)
            for x, y in ((q, yq), (k, yk)):
                ref, size = rotated(x, pos, axes, 1e4, interleaved)
                assert_within(y, ref, 9 * U * size, "rotated")
                rest = 2 * sum(axes)
                assert torch.equal(y[..., rest:], x[..., rest:])
            assert torch.equal(rotary(k, pos, **kw), yk)
            dq, dk = rotary_qk_backward(q, k, pos, **kw)
            for x, y in ((q, dq), (k, dk)):
                ref, size = rotated(x, pos, axes, 1e4, interleaved, -1)
                assert_within(y, ref, 9 * U * size, "rotated back")
            assert torch.equal(rotary_backward(q, pos, **kw), dq)


def test_far_positions(dev):
    """Angles of many turns keep their fraction."""
    x = torch.randn(1, 6, 2, 128, device=dev)
    pos = torch.tensor([[0], [1], [2 ** 24 - 1], [2 ** 31 - 1], [-2 ** 31], [1234567891]], dtype=torch.int32, device=dev)
    ref, size = rotated(x, pos, (64,), 1e4, True)
    # 2^31 radians in 64 bits: the product and the reference's own reduction are 2^-21 apart at most
    assert_within(rotary(x, pos, (64,)), ref, 9 * U * size + 2.0 ** -20 * size, "far")
    posf = torch.tensor([[0.25], [-3.5], [2.0 ** 20 + 0.5], [7e6], [1e-3], [0.0]], device=dev)
    ref, size = rotated(x, posf, (64,), 5e5, False)
    assert_within(rotary(x, posf, (64,), theta=5e5, interleaved=False), ref, 9 * U * size, "fractions")


def test_other_strides(dev):
    """Thirds of one fused projection, a narrowed batch, heads apart (copied), odd offsets."""
    B, S, H, D = 2, 11, 3, 64
    pos = grid_positions(1, 1, 11, dev)
    qkv = torch.randn(B, S, 3 * H * D + 1, device=dev, dtype=torch.bfloat16)
    q = qkv[..., 1:1 + H * D].unflatten(-1, (H, D))
    k = qkv[..., 1 + H * D:1 + 2 * H * D].unflatten(-1, (H, D))
    a, b = rotary_qk(q, k, pos, (11, 11, 10))
    c, d = rotary_qk(q.contiguous(), k.contiguous(), pos, (11, 11, 10))
    assert torch.equal(a, c) and torch.equal(b, d)
    for t in (q.transpose(1, 2).contiguous().transpose(1, 2), q[:, :, ::2], q[:1].expand(3, -1, -1, -1),
              q[:, ::2], torch.randn(B, S, H, 2 * D, device=dev)[..., ::2]):
        p = pos[:t.shape[1]]
        assert torch.equal(rotary(t, p, (11, 11, 10)), rotary(t.contiguous(), p, (11, 11, 10)))
    one = torch.randn(5, 1, H, D, device=dev)[::2]
    assert torch.equal(rotary(one, pos[:1], (32,) + (0, 0)), rotary(one.contiguous(), pos[:1], (32, 0, 0)))


def test_empty_and_copied(dev):
    pos = grid_positions(1, 2, 2, dev)
    assert rotary(torch.empty(0, 4, 2, 32, device=dev), pos, rotary_axes(32)).shape == (0, 4, 2, 32)
    assert rotary(torch.empty(1, 0, 2, 32, device=dev), pos[:0], rotary_axes(32)).shape == (1, 0, 2, 32)
    x = torch.randn(1, 4, 2, 32, device=dev)
    x[0, 0, 0, 20] = float("inf")
    x[0, 1, 1, 31] = float("nan")
    y = rotary(x, pos, (0, 8, 2))
    assert torch.equal(y[..., 20:].nan_to_num(7.0), x[..., 20:].nan_to_num(7.0))
    none = torch.empty(1, 4, 0, 32, device=dev)
    assert rotary(none, pos, rotary_axes(32)).shape == none.shape


def test_autograd(dev):
    q = torch.randn(1, 6, 2, 32, device=dev, requires_grad=True)
    k = torch.randn(1, 6, 1, 32, device=dev, requires_grad=True)
    pos = grid_positions(1, 2, 3, dev)
    yq, yk = RotaryFunction.apply(q, k, pos, rotary_axes(32), 1e4, True)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    wq, wk = rotary_qk_backward(dq, dk, pos, rotary_axes(32))
    assert torch.equal(gq, wq) and torch.equal(gk, wk)
    # against differences of the linear map in 64 bits
    e = torch.zeros_like(q, dtype=torch.float64)
    e[0, 5, 1, 9] = 1.0
    d = (rotated(e, pos, rotary_axes(32), 1e4, True)[0] * dq.double()).sum()
    assert abs(float(d) - float(gq[0, 5, 1, 9])) <= 16 * U * float(dq.detach().abs().max())
    y, none = RotaryFunction.apply(q, None, pos, rotary_axes(32))
    assert none is None and torch.equal(y, yq)
    (g,) = torch.autograd.grad(y, q, dq)
    assert torch.equal(g, wq)


def test_captured(dev):
    q = torch.randn(1, 60, 3, 64, device=dev, dtype=torch.float16)
    pos = grid_positions(3, 4, 5, dev)
    rotary_qk(q, q, pos, rotary_axes(64))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_qk(q, q, pos, rotary_axes(64))
    for k in range(3):
        q.copy_(torch.randn_like(q))
        pos += 1
        want = rotary_qk(q, q, pos, rotary_axes(64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), k


def test_norm_rotary_attention(dev):
    """The queries' and keys' way into the attention of a block: scores depend on the differences of
    positions alone."""
    B, S, H, D = 1, 24, 2, 128
    x = torch.randn(B, S, H * D, device=dev)
    w = 1 + 0.1 * torch.randn(H * D, device=dev)
    q = rms_norm(x, w).output.view(B, S, H, D)
    pos = grid_positions(2, 3, 4, dev)
    outs = []
    for shift in (0, 100):
        a, b = rotary_qk(q, q, pos + shift, rotary_axes(D))
        outs.append(memory_efficient_attention(a, b, x.view(B, S, H, D)).output)
    # scores of size up to sqrt(D) |q|^2 / D, each off by 40 u or so
    assert (outs[0] - outs[1]).abs().max() <= 1e-4 * x.abs().max()
