"""The operators around the linears as a program uses them together: a block's run forward and
backward, other streams, two streams at once, tensors whose offsets pass 32 bits,
outputs in the place of inputs."""
import ctypes
import math

import pytest
import torch

import reels_amd as ra
from reels_amd import _lib
from reels_amd.layers import _DTYPE_CODE, _launch, _stream
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu


def test_self_attention_of_a_block_trains(dev):
    """norm -> projections -> norms of q and k -> rotary -> attention, and back down to the gradients of
    the norms' weights, clipped: against the same in 64 bits. Float32 compute: the operators' errors
    are a few u of the sizes involved, the attention's and the linears' 1e-5 of them."""
    B, S, H, D = 1, 36, 2, 32
    K = H * D
    g = torch.Generator(device=dev).manual_seed(4)

    def rnd(*s, scale=1.0):
        return torch.randn(*s, generator=g, device=dev) * scale
    x, res, dout = rnd(B, S, K), rnd(B, S, K), rnd(B, S, H, D)
    w0, wq, wk = 1 + rnd(K, scale=0.1), 1 + rnd(K, scale=0.1), 1 + rnd(K, scale=0.1)
    mats = [ra.quantize_frozen_matrix(rnd(K, K, scale=K ** -0.5)) for _ in range(3)]
    pos, axes = ra.grid_positions(2, 3, 6, dev), ra.rotary_axes(D)

    n = ra.rms_norm(x, w0, 1e-6, res)
    flat = n.output.reshape(S, K)
    q, k, v = (ra.i8lora_forward(flat, m)[0] for m in mats)
    nq, nk = ra.rms_norm(q, wq), ra.rms_norm(k, wk)
    rq, rk = ra.rotary_qk(nq.output.view(B, S, H, D), nk.output.view(B, S, H, D), pos, axes)
    out, cache = ra.memory_efficient_attention(rq, rk, v.view(B, S, H, D))
    ga = ra.memory_efficient_attention_backward(rq, rk, v.view(B, S, H, D), dout, cache)
    dq, dk = ra.rotary_qk_backward(ga.q, ga.k, pos, axes)
    gq = ra.rms_norm_backward(dq.reshape(S, K), q, wq, nq.rstd)
    gk = ra.rms_norm_backward(dk.reshape(S, K), k, wk, nk.rstd)
    dflat = sum(ra.i8lora_backward(d, None, m)[0]
                for d, m in zip((gq.x, gk.x, ga.v.reshape(S, K)), mats))
    g0 = ra.rms_norm_backward(dflat.view(B, S, K), n.sum, w0, n.rstd, dsum=res)
    grads = [g0.weight, gq.weight, gk.weight]

    # the same in 64 bits by autograd
    xs, ws = [t.double().requires_grad_(True) for t in (x, res)], [t.double().requires_grad_(True) for t in (w0, wq, wk)]
    deq = [m.values.double() * m.scales.double()[:, None] for m in mats]

    def norm(t, w):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + float(torch.tensor(1e-6))) * w

    def rot(t):
        ang = torch.cat([pos[:, a:a + 1].double() * torch.tensor([1e4 ** (-j / p) for j in range(p)], dtype=torch.float64,
                                                                 device=dev) for a, p in enumerate(axes)], -1)
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    sm = xs[0] + xs[1]
    f = norm(sm, ws[0]).reshape(S, K)
    Q, Kk, V = (f @ m.t() for m in deq)
    rQ, rK = rot(norm(Q, ws[1]).view(B, S, H, D)), rot(norm(Kk, ws[2]).view(B, S, H, D))
    p = torch.softmax((rQ.transpose(1, 2) @ rK.transpose(1, 2).transpose(-1, -2)) / math.sqrt(D), -1)
    O = (p @ V.view(B, S, H, D).transpose(1, 2)).transpose(1, 2)
    want = torch.autograd.grad((O, sm), xs + ws, (dout.double(), res.double()))
    for got, ref in [(out, O), (g0.x, want[0]), (g0.x, want[1])] + list(zip(grads, want[2:])):
        assert_within(got, ref, 1e-4 * ref.detach().abs().max(), "block")
    before = [t.clone() for t in grads]
    total = math.sqrt(sum(float(t.double().square().sum()) for t in before))
    norm_dev = ra.clip_gradients(grads, total / 3)
    assert abs(float(norm_dev) - total) <= 2 * U * total
    for t, b in zip(grads, before):
        assert_within(t, b.double() / 3, 1e-6 * b.abs(), "clipped")


def calls(seed):
    """Every operator once on inputs of its own; returns what they give."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, r = (torch.randn(200, 1000, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.rand(1000, generator=g, device="cuda")
    n = ra.rms_norm(x, w, 1e-6, r)
    b = ra.rms_norm_backward(x, n.sum, w, n.rstd, r)
    q = ra.rms_norm_quantized(x, w, 1e-6, r).output
    m = ra.quantize_rows(torch.randn(700, 1000, generator=g, device="cuda").bfloat16())
    y = ra.quantized_linear(q, m, activation="gelu_tanh")
    z = ra.quantized_linear(ra.QuantizedMatrix(q.values[:3], q.scales[:3], q.compute_dtype), m)
    o = ra.quantized_linear(ra.quantize_rows(x[:, :999]), ra.quantize_rows(x[:50, 1:]))
    h = x[:, :960].reshape(1, 200, 15, 64)
    a, c = ra.rotary_qk(h, h[:, :, :5], ra.grid_positions(1, 10, 20, "cuda"), (12, 10, 10))
    gs = [t.float() for t in (x, r)]
    norm = ra.clip_gradients(gs, 1.0)
    return [n.output, n.sum, n.rstd, b.x, b.weight, q.values, q.scales, y, z, o, a, c, norm, *gs]


def test_other_streams_and_two_at_once(dev):
    want = [[t.clone() for t in calls(s)] for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for turn in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = calls(i + 1)
        torch.cuda.synchronize()
        for i in range(2):
            assert all(map(torch.equal, got[i], want[i])), (turn, i)


def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the last rows are those of a call on them alone."""
    M, C = 420_000, 5120  # 2.15e9 elements
    x = torch.empty(M, C, dtype=torch.bfloat16, device=dev).normal_()
    w = torch.rand(C, device=dev)
    last = x[-3:].clone()
    n = ra.rms_norm(x, w)
    assert torch.equal(n.output[-3:], ra.rms_norm(last, w).output)
    gx = ra.rms_norm_backward(x, x, w, n.rstd, want_dweight=False).x
    assert torch.equal(gx[-3:], ra.rms_norm_backward(last, last, w, n.rstd[-3:], want_dweight=False).x)
    del n, gx
    q = ra.rms_norm_quantized(x, w).output
    assert torch.equal(q.values[-3:], ra.rms_norm_quantized(last, w).output.values)
    del q
    pos = torch.arange(M, dtype=torch.int32, device=dev)[:, None]
    y = ra.rotary(x.view(1, M, 40, 128), pos, (64,))
    assert torch.equal(y[:, -3:], ra.rotary(last.view(1, 3, 40, 128), pos[-3:], (64,)))
    del y
    out = torch.empty_like(x)
    norm = ra.clip_gradients([x], 1.0, out=[out])
    assert abs(float(norm) / math.sqrt(M * C) - 1) < 1e-3
    f = float(torch.tensor(1.0 / (float(norm) + 1e-6)))
    assert_within(out[-3:], last.double() * f, 4 * U * last.double().abs() * f, "clipped")
    del out
    xq, m = ra.quantize_rows(x[:, :64]), ra.quantize_rows(x[:C, 64:128])
    y = ra.quantized_linear(xq, m)
    part = ra.quantized_linear(ra.QuantizedMatrix(xq.values[-3:], xq.scales[-3:], xq.compute_dtype), m)
    assert torch.equal(y[-3:], part)


def test_rows_that_are_not_finite_are_seen_after_quantising(dev):
    x = torch.randn(4, 300, device=dev).bfloat16()
    x[1, 7], x[2, 299] = float("nan"), float("inf")
    q = ra.quantize_rows(x)
    v = q.values.double() * q.scales.double()[:, None]
    assert torch.isfinite(v[[0, 3]]).all() and not torch.isfinite(v[1]).all() and not torch.isfinite(v[2]).all()


@pytest.mark.parametrize("C,dtype", [(101, torch.float32), (2049, torch.bfloat16), (5121, torch.float16),
                                     (8191, torch.float32), (20001, torch.bfloat16)])
def test_sum_in_place(dev, C, dtype):
    """The sum may take the place of x or of the residual: the same bits as into a buffer of its own,
    where a row ends inside a chunk and where the row is read twice (20001)."""
    x, r = (torch.randn(9, C, device=dev).to(dtype) for _ in range(2))
    w = torch.randn(C, device=dev)
    want, wantq = ra.rms_norm(x, w, 1e-6, r), ra.rms_norm_quantized(x, w, 1e-6, r)
    code = _DTYPE_CODE[dtype]
    for into in (0, 1):
        for quantized in (False, True):
            ops = [x.clone(), r.clone()]
            s = ops[into]
            out = torch.empty(9, C, dtype=torch.int8 if quantized else dtype, device=dev)
            row = torch.empty(9, device=dev)
            _launch("reels_hip_rms_norm_i8" if quantized else "reels_hip_rms_norm", dev, ops[0].data_ptr(), C,
                    ops[1].data_ptr(), C, w.data_ptr(), _lib.F32, code, 9, C, 1e-6, s.data_ptr(), out.data_ptr(),
                    row.data_ptr(), _stream(dev))
            assert torch.equal(s, want.sum)
            if quantized:
                assert torch.equal(out, wantq.output.values) and torch.equal(row, wantq.output.scales)
            else:
                assert torch.equal(out, want.output) and torch.equal(row, want.rstd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 77), (5, 100, 130), (65, 63, 70), (300, 256, 131), (1100, 1796, 1025),
                                   (4099, 1028, 2311)])
def test_product_over_its_residual(dev, M, K, N, dtype):
    """y may be the residual itself, in every form of the product."""
    x, w = (ra.quantize_rows(torch.randn(n, K, device=dev).to(dtype)) for n in (M, N))
    res = torch.randn(M, N, device=dev).to(dtype)
    want = ra.quantized_linear(x, w, None, "gelu_tanh", res)
    nbytes = _lib.lib().reels_hip_i8i8_workspace_bytes(M, K, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch("reels_hip_i8i8_linear", dev, x.values.data_ptr(), x.scales.data_ptr(), w.values.data_ptr(),
            w.scales.data_ptr(), None, res.data_ptr(), _lib.ACT_GELU_TANH, _DTYPE_CODE[dtype], M, K, N,
            res.data_ptr(), ws.data_ptr(), nbytes, _stream(dev))
    assert torch.equal(res, want)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,axes", [(128, (22, 21, 21)), (64, (8, 8)), (10, (1, 2))])
def test_rotary_in_place(dev, D, axes, interleaved):
    q, k = (torch.randn(2, 37, h, D, device=dev).bfloat16() for h in (3, 2))
    pos = torch.randint(0, 50, (37, len(axes)), device=dev, dtype=torch.int32)
    want = ra.rotary_qk(q, k, pos, axes, 1e4, interleaved)
    pairs = (ctypes.c_int32 * len(axes))(*axes)
    _launch("reels_hip_rotary", dev, q.data_ptr(), 3 * D, k.data_ptr(), 2 * D, pos.data_ptr(), _lib.I32, 1, _lib.BF16,
            2, 37, 3, 2, D, pairs, len(axes), 1e4, int(interleaved), 0, q.data_ptr(), k.data_ptr(), _stream(dev))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_second_derivatives_raise(dev):
    """The backward kernels have no derivative of their own: asking for it is an error, not a term left out."""
    x, r = (torch.randn(4, 64, device=dev, requires_grad=True) for _ in range(2))
    w = torch.ones(64, device=dev, requires_grad=True)
    pos = torch.arange(4, dtype=torch.int32, device=dev)[:, None]
    for y in (ra.RMSNormFunction.apply(x, w, None, 1e-6), ra.RMSNormFunction.apply(x, w, r, 1e-6)[1],
              ra.RotaryFunction.apply(x.view(1, 4, 2, 32), None, pos, (16,), 1e4, True)[0]):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.square().sum().backward()


@pytest.mark.parametrize("dtype,tiny", [(torch.float32, 3e-41), (torch.bfloat16, 4e-39), (torch.float16, 2e-6)])
def test_subnormal_values_are_kept(dev, dtype, tiny):
    """Inputs, sums and results below the type's normal range are rounded to its steps there, not to zero."""
    g = torch.Generator(device=dev).manual_seed(9)
    x, r = ((torch.randn(6, 517, generator=g, device=dev, dtype=torch.float64) * tiny).to(dtype) for _ in range(2))
    w = torch.full((517,), 2.0 ** -6, device=dev)
    n = ra.rms_norm(x, w, 1e-6, r)
    want = (x.double() + r.double()).cpu().to(dtype).to(dev)
    assert torch.equal(n.sum, want) and n.sum.count_nonzero() > 2000
    s = want.double()
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + float(torch.tensor(1e-6))) * w.double()
    assert_within(n.output, y, 4 * U * y.abs(), "y")
    big = torch.full((5,), 3.0, device=dev, dtype=dtype)
    grads = [x.clone(), big.clone()]
    norm = ra.clip_gradients(grads, 1.0)
    f = 1.0 / (math.sqrt(float(big.double().square().sum() + x.double().square().sum())) + 1e-6)
    assert_within(grads[0], x.double() * f, 2 * U * x.double().abs() * f, "clipped")
    assert float(norm) > 3
    q = x[:, :512].reshape(1, 6, 8, 64)
    pos = torch.arange(6, device=dev, dtype=torch.int32)[:, None]
    back = ra.rotary_backward(ra.rotary(q, pos, (32,)), pos, (32,))
    # two rotations of a pair: two roundings of each to the type's step there, and 18 u of sizes
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    size = q.double().unflatten(-1, (32, 2)).abs().sum(-1, keepdim=True).expand(1, 6, 8, 32, 2).flatten(-2)
    assert ((back.double() - q.double()).abs() <= 2 * step + (18 * U + 3 * torch.finfo(dtype).eps) * size).all()
    codes = ra.QuantizedMatrix(torch.randint(-127, 128, (6, 300), generator=g, device=dev, dtype=torch.int8),
                               torch.full((6,), 3e-42, device=dev), dtype)
    m = ra.QuantizedMatrix(torch.randint(-127, 128, (70, 300), generator=g, device=dev, dtype=torch.int8),
                           torch.full((70,), 1.5, device=dev) if dtype != torch.float16 else
                           torch.full((70,), 1e31, device=dev))
    v = torch.matmul(codes.values.double(), m.values.double().t().contiguous()) * codes.scales.double()[:, None] * m.scales.double()
    assert_within(ra.quantized_linear(codes, m), v, 4 * U * v.abs(), "product")
