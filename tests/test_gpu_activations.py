"""Activations in 8 bits against their definition in 64 bits (codes and scale bytes are equal), the GELU that
keeps its input and its pullback. gelu' is formed in f32: t = tanh within 6 u (2 u of tanh_f itself, the rest
from its argument, whose five roundings meet a slope times argument below 0.45); 0.5 (1 + t) takes 3 u of it (y = 0.5 x (1 + t) so
3 u |x|, and three roundings of its own),
0.5 x (1 - t^2) k (1 + 3 a x^2) 6 u |x| k (1 + 3 a x^2), and eight products and sums 8 u of the parts."""
import math

import pytest
import torch

import reels_amd as ra
from reels_amd import CompressedActivations, compress_activations, gelu_tanh_backward, gelu_tanh_compressed
from tests._blocks import blocks8, hard_rows
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = [(1, 1), (3, 7), (5, 31), (4, 32), (7, 33), (100, 101), (64, 256), (9, 1000), (33, 1536), (3, 5120), (2, 13825), (1, 70001)]


def grad_bound(x, dy):
    """(dy gelu'(x), its f32 error)."""
    k, a = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(k * (x + a * x ** 3))
    part = 0.5 * x * k * (1 + 3 * a * x * x)
    grad = 0.5 * (1 + t) + part * (1 - t * t)
    return dy * grad, dy.abs() * U * (3 + 12 * part.abs() + 8 * (1 + (part * (1 - t * t)).abs()) + grad.abs())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,C", SIZES)
def test_codes_and_values(dev, M, C, dtype):
    x = hard_rows(M, C, DT[dtype], dev)
    k = compress_activations(x)
    q, s, v = blocks8(x.double())
    assert torch.equal(k.scales, s)
    assert torch.equal(k.values, q)
    assert k.compute_dtype == DT[dtype] and k.shape == x.shape
    for d in DT.values():
        r = v.to(d)
        if d == torch.float16:  # saturates
            r = torch.where(torch.isinf(r), torch.sign(r) * 65504, r)
        got = k.restore(d)
        assert torch.equal(torch.isnan(got), torch.isnan(r))
        assert torch.equal(got.nan_to_num(7.0), r.nan_to_num(7.0)), d
    # the values are as near as 7 bits come: half a step of the largest
    ok = torch.isfinite(v) & torch.isfinite(x.double())
    top = x.double().abs().nan_to_num(0.0, 0.0, 0.0)
    top = torch.nn.functional.pad(top, (0, -C % 32)).view(M, -1, 32).amax(2).repeat_interleave(32, 1)[:, :C]
    inside = top < torch.finfo(DT[dtype]).max * 0.99
    assert bool(((v - x.double()).abs() <= top / 127 + 2.0 ** -133)[ok & inside].all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,C", SIZES)
def test_gelu_forward_and_backward(dev, M, C, dtype):
    g = torch.Generator(device=dev).manual_seed(M + C)
    x = (torch.randn(M, C, generator=g, device=dev) * 2).to(DT[dtype])
    dy = torch.randn(M, C, generator=g, device=dev).to(DT[dtype])
    y, k = gelu_tanh_compressed(x)
    xd = x.double()
    yd = torch.nn.functional.gelu(xd, approximate="tanh")
    assert_within(y, yd, U * (3 * xd.abs() + 3 * yd.abs()), "y")
    both = compress_activations(x)
    assert torch.equal(k.values, both.values) and torch.equal(k.scales, both.scales)
    dx = gelu_tanh_backward(k, dy)
    ref, slack = grad_bound(blocks8(x.double())[2], dy.double())
    assert_within(dx, ref, slack, "dx")
    in_place = dy.clone()
    L = ra._lib.lib()
    assert L.reels_hip_act8_gelu_tanh_bwd(k.values.data_ptr(), k.scales.data_ptr(), in_place.data_ptr(),
                                          {"f32": 0, "bf16": 1, "f16": 2}[dtype], M, C, in_place.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(in_place, dx)


def test_nan_blocks(dev):
    x = torch.randn(3, 100, device=dev)
    x[1, 40] = float("nan")
    x[2, 99] = float("inf")
    k = compress_activations(x)
    v, dx = k.restore(), gelu_tanh_backward(k, torch.ones_like(x))
    for t in (v, dx):
        bad = torch.isnan(t)
        assert not bad[0].any() and bad[1, 32:64].all() and bad[1].sum() == 32 and bad[2, 96:].all() and bad[2].sum() == 4


def test_shapes_strides_and_empty(dev):
    x = torch.randn(2, 3, 5, 40, device=dev, dtype=torch.bfloat16)
    k = compress_activations(x.transpose(1, 2))
    assert k.shape == (2, 5, 3, 40) and k.scales.shape == (2, 5, 3, 2)
    assert torch.equal(k.restore(), compress_activations(x.transpose(1, 2).contiguous()).restore())
    r = k.reshape(-1, 40)
    assert r.shape == (30, 40) and torch.equal(r.restore(), k.restore().reshape(30, 40))
    cut = CompressedActivations(r.values[::2], r.scales[::2], torch.bfloat16)  # not dense
    assert torch.equal(cut.restore(), r.restore()[::2])
    odd = torch.randn(1 + 7 * 33, device=dev, dtype=torch.float16)[1:].view(7, 33)  # off its alignment
    assert torch.equal(compress_activations(odd).values, compress_activations(odd.clone()).values)
    e = compress_activations(x[:0])
    assert e.restore().shape == (0, 3, 5, 40) and gelu_tanh_backward(e, x[:0]).shape == (0, 3, 5, 40)
    v = compress_activations(x[0, 0, 0])
    assert v.shape == (40,) and v.scales.shape == (2,)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K,N,r", [(70, 64, 96, 4), (300, 257, 130, 3), (1000, 1536, 512, 32)])
def test_linear_backward(dev, M, K, N, r, dtype):
    """The linear's backward from kept rows is the backward of the rows that they stand for."""
    dt = DT[dtype]
    g = torch.Generator(device=dev).manual_seed(M)

    def rnd(*s):
        return torch.randn(s, generator=g, device=dev).to(dt)
    W = ra.quantize_frozen_matrix(rnd(N, K))
    x, dy, A, B, gx = rnd(M, K), rnd(M, N), rnd(K, r), rnd(r, N), rnd(M, K)
    k = compress_activations(x)
    h = ra.i8lora_forward(x, W, A, B, save_h=True)[1]
    for kw in (dict(h=h), dict(), dict(want_dA=False, h=h), dict(want_dbias=True)):
        for a, b in zip(ra.i8lora_backward(dy, k, W, A, B, 0.5, **kw), ra.i8lora_backward(dy, k.restore(), W, A, B, 0.5, **kw)):
            assert (a is None and b is None) or torch.equal(a, b)
    layer = ra.LoRALinear(W, r, A=A, B=B)
    a, b = ra.lora_backward(layer, k.reshape(2, M // 2, K), dy.view(2, M // 2, N)), ra.lora_backward(layer, k.restore(), dy)
    assert torch.equal(a["dx"].view(M, K), b["dx"]) and torch.equal(a["A"], b["A"]) and torch.equal(a["B"], b["B"])
    kg = compress_activations(gx)
    two = ra.i8lora_backward(dy, k.restore(), W, A, B, 0.5, h=h)
    for a, b in zip(ra.i8lora_backward_gelu(dy, k, kg, W, A, B, 0.5, h=h), (gelu_tanh_backward(kg, two[0]),) + two[1:]):
        assert torch.equal(a, b)


def test_autograd(dev):
    g = torch.Generator(device=dev).manual_seed(4)
    W = ra.quantize_frozen_matrix(torch.randn(96, 64, generator=g, device=dev).bfloat16())
    x = torch.randn(50, 64, generator=g, device=dev).bfloat16().requires_grad_()
    A = (torch.randn(64, 8, generator=g, device=dev) / 8).requires_grad_()
    B = (torch.randn(8, 96, generator=g, device=dev) / 8).requires_grad_()
    dy = torch.randn(50, 96, generator=g, device=dev).bfloat16()
    k = compress_activations(x.detach())

    def step(kept):
        z = ra.GeluTanhCompressedFunction.apply(ra.I8LoRALinearFunction.apply(x, A, B, W.values, W.scales, None, 1.0, kept))
        return torch.autograd.grad(z, (x, A, B), dy)
    z = ra.i8lora_forward(x.detach(), W, A.detach().bfloat16(), B.detach().bfloat16(), None, 1.0)[0]
    dz = gelu_tanh_backward(compress_activations(z), dy)
    kept, whole = step(k), step(None)
    assert torch.equal(kept[0], whole[0]) and torch.equal(kept[2], whole[2])  # dx and dB do not read x
    want = ra.i8lora_backward(dz, k.restore(), W, A.detach().bfloat16(), B.detach().bfloat16(), 1.0)
    assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1])
    with pytest.raises(ValueError, match="kept"):
        ra.I8LoRALinearFunction.apply(x, A, B, W.values, W.scales, None, 1.0, compress_activations(x.detach()[:3]))


def test_other_stream_and_graph(dev):
    x = torch.randn(300, 1000, device=dev, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    y0, k0 = gelu_tanh_compressed(x)
    d0 = gelu_tanh_backward(k0, dy)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y1, k1 = gelu_tanh_compressed(x)
        d1 = gelu_tanh_backward(k1, dy)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y0, y1) and torch.equal(k0.values, k1.values) and torch.equal(d0, d1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, k2 = gelu_tanh_compressed(x)
        d2, r2 = gelu_tanh_backward(k2, dy), k2.restore()
    for i in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        y, k = gelu_tanh_compressed(x)
        assert torch.equal(y, y2) and torch.equal(k.restore(), r2) and torch.equal(gelu_tanh_backward(k, dy), d2)


def test_offsets_past_32_bits(dev):
    """A matrix of more than 2^32 bytes: its last rows are those of a small one."""
    C, M = 13824, 170000
    x = torch.zeros(M, C, device=dev, dtype=torch.bfloat16)
    tail = torch.randn(5, C, device=dev).bfloat16()
    x[-5:] = tail
    y, k = gelu_tanh_compressed(x)
    ys, ks = gelu_tanh_compressed(tail)
    assert torch.equal(y[-5:], ys) and torch.equal(k.values[-5:], ks.values) and torch.equal(k.scales[-5:], ks.scales)
    assert torch.equal(k.restore()[-5:], ks.restore()) and not bool(k.values[:-5].any())
    dx = gelu_tanh_backward(k, x)
    assert torch.equal(dx[-5:], gelu_tanh_backward(ks, tail))


@pytest.mark.parametrize("dtype", list(DT))
def test_gelu_pullback_at_the_ends_of_the_range(dev, dtype):
    """Past 16 the slope is 1 or 0 to the last bit, up to the type's largest value: from kept values, from the
    values themselves and behind the linear's dX."""
    dt = DT[dtype]
    top = torch.finfo(dt).max
    sizes = [v for v in (17.0, 1e3, 3e4, 1e10, 9e18, 1.3e19, 6e19, 1e25, top / 3, top) if v <= top]
    x = torch.tensor(sizes + [-v for v in sizes], device=dev, dtype=torch.float64).to(dt)[:, None].repeat(1, 96)
    g = torch.Generator(device=dev).manual_seed(2)
    dy = torch.randn(x.shape, generator=g, device=dev).to(dt)
    k = compress_activations(x)
    assert torch.isfinite(k.restore(torch.float32)).all()
    for dx in (gelu_tanh_backward(k, dy), gelu_tanh_backward(x, dy)):
        assert torch.equal(dx, torch.where(x > 0, dy, torch.zeros_like(dy)))
    W = ra.quantize_frozen_matrix(torch.randn(64, 96, generator=g, device=dev).to(dt))
    dz = torch.randn(len(x), 64, generator=g, device=dev).to(dt)
    dx = ra.i8lora_backward(dz, None, W, want_dA=False, want_dB=False)[0]
    want = torch.where(x > 0, dx, torch.zeros_like(dx))
    for gx in (x, k):
        assert torch.equal(ra.i8lora_backward_gelu(dz, None, gx, W, want_dA=False, want_dB=False)[0], want)
