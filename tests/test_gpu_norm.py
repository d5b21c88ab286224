"""RMS norm, its int8 output and its backward against the formulas in 64 bits. Bounds count the f32
roundings of the kernels (u = 2^-24): y has two products and rstd's rounding (3 u); dx forms g = dy w
(u), k = rstd^2 mean(g s) from rounded g and rstd (4 u on the mean of |g s|), their difference and its
product with rstd (3 u); dw adds rows / 256 + 100 terms at most one after the other."""
import math

import pytest
import torch

from reels_amd import (QuantizedMatrix, RMSNormFunction, memory_efficient_attention, quantized_linear,
                       rms_norm, rms_norm_backward, rms_norm_quantized)
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# rows, columns: one element, below and past a vector, a wave's and a workgroup's forms, the loop form
SIZES = [(1, 1), (3, 2), (5, 7), (33, 8), (100, 101), (17, 128), (40, 256), (9, 517), (64, 1536),
         (7, 2049), (3, 5120), (5, 8193), (2, 16385), (3, 32768), (2, 32777), (1, 70001)]


def make(M, C, dtype, residual, wtype, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed + M * 131 + C)
    dt = DT[dtype]

    def rnd(*s):
        return torch.randn(s, generator=g, device=dev)
    x = (rnd(M, C) * 1.5).to(dt)
    r = rnd(M, C).to(dt) if residual else None
    w = None if wtype is None else (1 + 0.3 * rnd(C)).to(DT[wtype])
    return x, r, w, rnd(M, C).to(dt), rnd(M, C).to(dt)


def formula(x, r, w, eps):
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    sd = s.double()
    rstd = 1.0 / torch.sqrt(sd.square().mean(-1) + eps)
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    return s, sd, rstd, wd


def check_sum(got, x, r):
    # x + r rounded once: equal, or apart where the f32 sum is a tie of the 16-bit type
    if r is None:
        assert got is x
    else:
        assert torch.equal(got, (x.float() + r.float()).to(x.dtype))


@pytest.mark.parametrize("dtype,wtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                         ("f16", None), ("f32", "f32"), ("f32", None)])
@pytest.mark.parametrize("M,C", SIZES)
def test_forward_and_backward(dev, M, C, dtype, wtype):
    for residual in (False, True):
        x, r, w, dy, dsum = make(M, C, dtype, residual, wtype)
        res = rms_norm(x, w, 1e-6, r)
        check_sum(res.sum, x, r)
        _, sd, rstd, wd = formula(x, r, w, 1e-6)
        sd = res.sum.double()
        rstd = 1.0 / torch.sqrt(sd.square().mean(-1) + float(torch.tensor(1e-6)))
        y = sd * rstd[:, None] * wd
        assert_within(res.output, y, 4 * U * y.abs(), "y")
        assert_within(res.rstd, rstd, U * rstd, "rstd")
        ds = dsum if residual else None
        g = rms_norm_backward(dy, res.sum, w, res.rstd, ds, want_dweight=True)
        gd = dy.double() * wd
        mean = (gd * sd).mean(-1, keepdim=True)
        mean_abs = (gd * sd).abs().mean(-1, keepdim=True)
        rs = rstd[:, None]
        dx = rs * (gd - sd * rs * rs * mean)
        slack = 8 * U * rs * (gd.abs() + sd.abs() * rs * rs * mean_abs)
        if residual:
            dx = dx + ds.double()
            slack = slack + 2 * U * (ds.double().abs() + dx.abs())
        assert_within(g.x, dx, slack, "dx")
        if w is None:
            assert g.weight is None
        else:
            t = dy.double() * sd * rs
            assert_within(g.weight, t.sum(0), (100 + M / 256) * U * t.abs().sum(0), "dw")


def test_many_rows_weight_gradient(dev):
    """More rows than partial sums: every form of the row walk, and the same bits again."""
    for C, dtype in ((100, "f32"), (1000, "bf16"), (5120, "bf16"), (9000, "f16"), (33000, "bf16")):
        M = 4999 if C < 9000 else 700
        x, _, w, dy, _ = make(M, C, dtype, False, dtype)
        res = rms_norm(x, w)
        a, b = (rms_norm_backward(dy, x, w, res.rstd) for _ in range(2))
        t = dy.double() * x.double() * res.rstd.double()[:, None]
        assert_within(a.weight, t.sum(0), (100 + M / 64) * U * t.abs().sum(0), f"dw C={C}")
        assert torch.equal(a.weight, b.weight) and torch.equal(a.x, b.x)
        c = rms_norm_backward(dy, x, w, res.rstd, want_dweight=False)
        assert c.weight is None and torch.equal(a.x, c.x)


@pytest.mark.parametrize("dtype,wtype", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32"), ("bf16", None)])
@pytest.mark.parametrize("M,C", SIZES)
def test_quantized_rows(dev, M, C, dtype, wtype):
    for residual in (False, True):
        x, r, w, _, _ = make(M, C, dtype, residual, wtype)
        if M > 2:
            x[1] = 0
            if residual:
                r[1] = 0
        res = rms_norm_quantized(x, w, 1e-6, r)
        check_sum(res.sum, x, r)
        p = res.sum.double() * (1.0 if w is None else w.double())
        top = p.abs().amax(-1)
        rstd = 1.0 / torch.sqrt(res.sum.double().square().mean(-1) + float(torch.tensor(1e-6)))
        codes = torch.where(top[:, None] > 0, torch.round(127.0 * p / top[:, None].clamp_min(1e-300)),
                            torch.zeros_like(p))
        assert res.output.values.dtype == torch.int8
        assert torch.equal(res.output.values, codes.to(torch.int8))
        scale = torch.where(top > 0, top * rstd / 127.0, torch.ones_like(top))
        assert_within(res.output.scales, scale, U * scale, "scales")
        assert res.output.compute_dtype == x.dtype


def test_row_strides_and_offsets(dev):
    """Rows inside a wider matrix, starting at any element."""
    for dtype in DT:
        big = torch.randn(37, 900, device=dev).to(DT[dtype])
        res_big = torch.randn(37, 771, device=dev).to(DT[dtype])
        x, r = big[:, 3:304], res_big[:, 1:302]
        w = torch.randn(303, device=dev).to(DT[dtype])[2:]
        a, b = rms_norm(x, w, 1e-5, r), rms_norm(x.contiguous(), w.clone(), 1e-5, r.contiguous())
        assert torch.equal(a.output, b.output) and torch.equal(a.sum, b.sum) and torch.equal(a.rstd, b.rstd)
        qa, qb = rms_norm_quantized(x, w, 1e-5, r), rms_norm_quantized(x.contiguous(), w.clone(), 1e-5, r.contiguous())
        assert torch.equal(qa.output.values, qb.output.values) and torch.equal(qa.output.scales, qb.output.scales)
        t = big[:, ::2]  # columns apart: copied
        assert torch.equal(rms_norm(t).output, rms_norm(t.contiguous()).output)


def test_leading_dimensions_and_empty(dev):
    x = torch.randn(2, 3, 5, 64, device=dev, dtype=torch.bfloat16)
    a = rms_norm(x)
    assert a.output.shape == x.shape and a.rstd.shape == (2, 3, 5) and a.sum is x
    assert torch.equal(a.output.reshape(-1, 64), rms_norm(x.reshape(-1, 64)).output)
    v = torch.randn(64, device=dev)
    assert rms_norm(v).rstd.shape == ()
    e = torch.empty(0, 64, device=dev)
    r = rms_norm(e, torch.ones(64, device=dev))
    assert r.output.shape == (0, 64)
    g = rms_norm_backward(e, e, torch.ones(64, device=dev), r.rstd)
    assert torch.equal(g.weight, torch.zeros(64, device=dev)) and g.x.shape == (0, 64)
    q = rms_norm_quantized(e)
    assert q.output.values.shape == (0, 64)


@pytest.mark.parametrize("C", [96, 5120, 40000])
def test_values_outside_the_ordinary(dev, C):
    """Rows near the ends of the f32 range, zero rows, NaN and infinities."""
    x = torch.randn(7, C, device=dev)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, C // 2] = float("nan")
    x[4, C - 1] = float("inf")
    eps = 0.0
    r = rms_norm(x, None, eps)
    sd = x.double()
    rstd = 1.0 / torch.sqrt(sd.square().mean(-1))
    y = sd * rstd[:, None]
    assert_within(r.output[[0, 1, 5, 6]], y[[0, 1, 5, 6]], 4 * U * y[[0, 1, 5, 6]].abs(), "y")
    assert torch.isnan(r.output[2]).all() and torch.isnan(r.output[3]).all()
    assert torch.isnan(r.output[4, C - 1]) and not r.output[4, :C - 1].any()
    q = rms_norm_quantized(x, None, eps)
    assert torch.isnan(q.output.scales[[2, 3, 4]]).all() and not q.output.values[[2, 3, 4]].any()
    assert torch.isfinite(q.output.scales[[0, 1, 5, 6]]).all()
    top = x.double().abs().amax(-1, keepdim=True)
    want = torch.round(127.0 * x.double() / top)
    assert torch.equal(q.output.values[[0, 1, 5, 6]].double(), want[[0, 1, 5, 6]])
    w = torch.ones(C, device=dev)
    w[1] = float("nan")
    q = rms_norm_quantized(torch.ones(2, C, device=dev), w)
    assert torch.isnan(q.output.scales).all()


@pytest.mark.parametrize("C", [40, 3000, 40000])
def test_quantized_with_wide_weights(dev, C):
    """Weights and rows whose products pass the f32 range on either side still give the codes of the
    64-bit quotients."""
    g = torch.Generator(device=dev).manual_seed(C)
    x = torch.randn(6, C, generator=g, device=dev)
    x[1] *= 1e-36
    x[2] *= 1e30
    x[3] *= 10.0 ** torch.randint(-30, 1, (C,), generator=g, device=dev).float()
    for w in (torch.full((C,), 3e25, device=dev), 10.0 ** torch.randint(-30, 31, (C,), generator=g, device=dev).float(),
              torch.full((C,), 1e-25, device=dev)):
        for eps in (0.0, 1e-6):
            q = rms_norm_quantized(x, w, eps).output
            p = x.double() * w.double()
            top = p.abs().amax(-1, keepdim=True)
            rstd = 1.0 / torch.sqrt(x.double().square().mean(-1) + float(torch.tensor(eps)))
            fits = (top[:, 0] * rstd / 127).float().isfinite()
            assert torch.equal(q.values[fits].double(), torch.round(127.0 * p / top)[fits])
            assert torch.isnan(q.scales[~fits]).all() and torch.isfinite(q.scales[fits]).all()


def test_ties_go_to_even(dev):
    # 127 p / top is a half exactly where p is half the row's largest
    x = torch.tensor([[2.0, 1.0, -1.0, 0.5, 2.0, -2.0, 0.0, 0.0]], device=dev, dtype=torch.bfloat16)
    assert rms_norm_quantized(x).output.values.tolist() == [[127, 64, -64, 32, 127, -127, 0, 0]]


def test_autograd_matches_the_calls_and_differences(dev):
    for residual in (False, True):
        x, r, w, dy, dsum = (t if t is None else t.detach() for t in make(4, 24, "f32", residual, "f32"))
        leaves = [t.clone().requires_grad_(True) for t in ((x, w, r) if residual else (x, w))]
        if residual:
            y, s = RMSNormFunction.apply(leaves[0], leaves[1], leaves[2], 1e-6)
            got = torch.autograd.grad((y, s), leaves, (dy, dsum))
            assert torch.equal(got[0], got[2])
        else:
            y = RMSNormFunction.apply(leaves[0], leaves[1], None, 1e-6)
            got = torch.autograd.grad(y, leaves, dy)
        res = rms_norm(x, w, 1e-6, r)
        want = rms_norm_backward(dy, res.sum, w, res.rstd, dsum if residual else None)
        assert torch.equal(got[0], want.x) and torch.equal(got[1], want.weight)

        # central differences of the formula in 64 bits: step h, error h^2 of third derivatives
        def loss(xd, wd):
            sd = xd if r is None else xd + r.double()
            v = (sd / torch.sqrt(sd.square().mean(-1, keepdim=True) + 1e-6) * wd * dy.double()).sum()
            return v if r is None else v + (sd * dsum.double()).sum()
        h = 1e-5
        for i, j in ((0, 0), (2, 7), (3, 23)):
            e = torch.zeros_like(x, dtype=torch.float64)
            e[i, j] = h
            d = (loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * h)
            assert abs(float(d) - float(want.x[i, j])) < 1e-5 * (1 + abs(float(d)))
        e = torch.zeros(24, dtype=torch.float64, device=dev)
        e[5] = h
        d = (loss(x.double(), w.double() + e) - loss(x.double(), w.double() - e)) / (2 * h)
        assert abs(float(d) - float(want.weight[5])) < 1e-5 * (1 + abs(float(d)))
    # the sum alone, or the norm alone, reaches the loss
    x = torch.randn(3, 16, device=dev, requires_grad=True)
    r = torch.randn(3, 16, device=dev, requires_grad=True)
    y, s = RMSNormFunction.apply(x, None, r)
    gx, gr = torch.autograd.grad(s.sum(), (x, r), retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx)
    (gy,) = torch.autograd.grad(y.sum(), x)
    assert gy.shape == x.shape


def test_captured_calls_replay(dev):
    """Forward, int8 form and backward in one graph, replayed between eager calls."""
    x, r, w, dy, dsum = make(300, 1536, "bf16", True, "bf16")

    def step():
        n = rms_norm(x, w, 1e-6, r)
        g = rms_norm_backward(dy, n.sum, w, n.rstd, dsum)
        q = rms_norm_quantized(x, w, 1e-6, r)
        return n.output, n.sum, g.x, g.weight, q.output.values, q.output.scales
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_block_in_8_bits(dev):
    """Norm with residual, int8 product with GELU, second product with the residual: what each hands
    on is what the next takes."""
    M, K, N = 70, 256, 640
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn(M, K, generator=g, device=dev).bfloat16() for _ in range(2))
    w1 = QuantizedMatrix(torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8),
                         torch.full((N,), 5e-4, device=dev))
    n = rms_norm_quantized(x, None, 1e-6, r)
    y = quantized_linear(n.output, w1, activation="gelu_tanh")
    ref = n.output.values.double() * n.output.scales.double()[:, None]
    z = ref @ (w1.values.double() * w1.scales.double()[:, None]).t()
    want = torch.nn.functional.gelu(z, approximate="tanh")
    assert_within(y, want, 12 * U * z.abs(), "product of the norm's codes")


def test_norm_feeds_attention(dev):
    B, S, H, D = 1, 50, 2, 64
    x = torch.randn(B, S, H * D, device=dev, dtype=torch.bfloat16)
    q = rms_norm(x, torch.ones(H * D, device=dev)).output.view(B, S, H, D)
    out = memory_efficient_attention(q, q, x.view(B, S, H, D)).output
    p = torch.softmax(torch.matmul(q.double().transpose(1, 2), q.double().transpose(1, 2).mT.contiguous())
                      / D ** 0.5, -1)
    ref = torch.matmul(p, x.view(B, S, H, D).double().transpose(1, 2).contiguous()).transpose(1, 2)
    # P is rounded to bf16 and the result once more
    assert (out.double() - ref).abs().max() <= 2.0 ** -7 * x.double().abs().max()


@pytest.mark.parametrize("dtype,wtype", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("C", [5, 96, 5120, 16384, 40000])
def test_infinities_under_zero_weights_reach_the_quantized_rows(dev, C, dtype, wtype):
    """An infinity times a zero weight is NaN in the norm's row, whatever the other products are: its
    scale is NaN and its codes are 0."""
    at = C // 2
    x = (torch.randn(6, C, device=dev) + 3).to(DT[dtype])
    x[1, at], x[2, at], x[3, at] = math.inf, -math.inf, math.nan
    r = torch.zeros_like(x)
    if dtype == "f16":  # the sum overflows
        x[4, at] = r[4, at] = 60000.0
    else:
        r[4, at] = math.inf
    one = torch.ones(C, device=dev, dtype=DT[wtype])
    one[at] = 0
    for w, ordinary in ((one, None), (torch.zeros_like(one), 1.0)):
        for residual in (None, r):
            bad = [1, 2, 3] if residual is None else [1, 2, 3, 4]
            good = [i for i in range(6) if i not in bad]
            y = rms_norm(x, w, 1e-6, residual).output
            assert torch.isnan(y[bad, at]).all() and torch.isfinite(y[good]).all()
            q = rms_norm_quantized(x, w, 1e-6, residual).output
            assert torch.isnan(q.scales[bad]).all() and not q.values[bad].any()
            assert torch.isfinite(q.scales[good]).all()
            if ordinary is not None:
                assert (q.scales[good] == ordinary).all() and not q.values[good].any()
            else:
                assert (q.values[good].abs().amax(1) == 127).all()
