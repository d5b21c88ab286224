"""The product of int8 rows with an int8 weight against 64 bits. The sum is exact; it is rounded to
f32, multiplied by two scales and joined with the bias (4 u of the product, u of the bias), the GELU
has a slope below 1.13 and its tanh is within 2^-23 (x 0.5, with the rounding of its argument 4 u
|x|), and the residual adds one rounding."""
import pytest
import torch

from reels_amd import (QuantizedMatrix, _weight_mul, quantize_frozen_matrix, quantize_rows, quantized_linear,
                       rms_norm, rms_norm_quantized)
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gelu(x):
    return torch.nn.functional.gelu(x, approximate="tanh")


def make(M, K, N, dtype, seed=0, full=False):
    g = torch.Generator(device="cuda").manual_seed(seed + M + 7 * K + 13 * N)

    def codes(r, c):
        lo = -127 if not full else 127
        return torch.randint(lo, 128, (r, c), generator=g, device="cuda", dtype=torch.int8)
    x = QuantizedMatrix(codes(M, K), torch.rand(M, generator=g, device="cuda") * 0.02 + 1e-3, DT[dtype])
    w = QuantizedMatrix(codes(N, K), torch.rand(N, generator=g, device="cuda") * 1e-3 / K ** 0.5 + 1e-5, DT[dtype])
    bias = torch.randn(N, generator=g, device="cuda").to(DT[dtype])
    res = torch.randn(M, N, generator=g, device="cuda").to(DT[dtype])
    return x, w, bias, res


def check(y, x, w, bias, res, act, what=""):
    acc = torch.matmul(x.values.double(), w.values.double().t().contiguous())
    v = acc * x.scales.double()[:, None] * w.scales.double()
    slack = 4 * U * v.abs()
    if bias is not None:
        v = v + bias.double()
        slack = slack + U * (bias.double().abs() + v.abs())
    if act:
        slack = 1.13 * slack + 6 * U * v.abs()
        v = gelu(v)
    if res is not None:
        v = v + res.double()
        slack = slack + U * v.abs()
    assert_within(y, v, slack, f"y {what}")


# tokens, inputs, outputs: single tokens, edges of the tiles of every form, odd widths
SIZES = [(1, 1, 1), (1, 64, 16), (1, 5120, 1000), (2, 100, 77), (3, 17, 5), (7, 1536, 1537), (16, 256, 64),
         (17, 130, 33), (31, 512, 130), (33, 1000, 300), (64, 64, 64), (65, 65, 65), (100, 2048, 513),
         (128, 384, 256), (129, 1024, 257), (200, 4096, 640), (255, 640, 255), (300, 131071, 20),
         (513, 128, 769), (300, 4, 70), (300, 100, 130), (70, 252, 65), (1100, 1796, 1024), (2050, 1300, 2049), (777, 1000, 3001), (4100, 1024, 2304), (4099, 1028, 2310), (40000, 100, 2048), (20001, 256, 2049), (1025, 896, 1024), (2100, 1537, 130), (5000, 256, 512)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(dev, M, K, N, dtype):
    x, w, bias, res = make(M, K, N, dtype)
    y = quantized_linear(x, w)
    assert y.dtype == DT[dtype] and y.shape == (M, N)
    check(y, x, w, None, None, False, "plain")
    check(quantized_linear(x, w, bias, "gelu_tanh", res), x, w, bias, res, True, "bias, gelu, residual")
    check(quantized_linear(x, w, None, None, res), x, w, None, res, False, "residual")
    check(quantized_linear(x, w, bias), x, w, bias, None, False, "bias")


def test_largest_sums(dev):
    """All codes 127 over the longest reduction: no whole number is lost."""
    x, w, _, _ = make(5, 131071, 70, "f32", full=True)
    x.values[1], x.values[2] = -127, -128
    w.values[3] = -128
    check(quantized_linear(x, w), x, w, None, None, False)


def test_rows_do_not_depend_on_their_place(dev):
    for K, N in ((256, 300), (1024, 2048), (1000, 99)):
        x, w, bias, res = make(1500, K, N, "bf16")
        whole = quantized_linear(x, w, bias, "gelu_tanh", res)
        for a, b in ((0, 1), (3, 20), (700, 1000), (1499, 1500), (1, 1500)):
            part = quantized_linear(QuantizedMatrix(x.values[a:b], x.scales[a:b], x.compute_dtype), w, bias,
                                    "gelu_tanh", res[a:b])
            assert torch.equal(part, whole[a:b]), (K, N, a, b)


def test_offsets_and_strides(dev):
    """Operands at odd places of wider buffers."""
    x, w, bias, res = make(90, 256, 130, "bf16")
    flat = torch.zeros(90 * 256 + 64, dtype=torch.int8, device=dev)
    for off in (1, 4, 8):
        xv = flat[off:off + 90 * 256].view(90, 256)
        xv.copy_(x.values)
        wf = torch.zeros(130 * 256 + 64, dtype=torch.int8, device=dev)[off:off + 130 * 256].view(130, 256)
        wf.copy_(w.values)
        b = torch.cat([bias[:1], bias])[1:]
        r = torch.cat([res.reshape(-1)[:1], res.reshape(-1)])[1:].view(90, 130)
        y = quantized_linear(QuantizedMatrix(xv, x.scales, x.compute_dtype),
                             QuantizedMatrix(wf, w.scales, w.compute_dtype), b, None, r)
        assert torch.equal(y, quantized_linear(x, w, bias, None, res))
    wide = QuantizedMatrix(torch.cat([x.values, x.values], 1)[:, :256], x.scales, x.compute_dtype)
    assert torch.equal(quantized_linear(wide, w), quantized_linear(x, w))


def test_dtype_and_empty(dev):
    x, w, bias, _ = make(9, 64, 33, "bf16")
    check(quantized_linear(x, w, dtype=torch.float32), x, w, None, None, False)
    check(quantized_linear(x, w, bias.half(), dtype=torch.float16), x, w, bias.half(), None, False)
    e = QuantizedMatrix(x.values[:0], x.scales[:0])
    assert quantized_linear(e, w).shape == (0, 33)


def test_scales_of_nan_rows_reach_the_result(dev):
    h = torch.randn(4, 128, device=dev).bfloat16()
    h[2, 5] = float("nan")
    _, w, _, _ = make(1, 128, 40, "bf16")
    y = quantized_linear(rms_norm_quantized(h).output, w)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()


def test_quantize_rows_is_the_packing(dev):
    x = torch.randn(37, 129, device=dev).bfloat16()
    a, b = quantize_rows(x), quantize_frozen_matrix(x)
    assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)
    assert a.compute_dtype == torch.bfloat16
    c = quantize_rows(torch.cat([x, x], 1)[:, 129:])
    assert torch.equal(c.values, a.values)
    assert quantize_rows(x[:0]).values.shape == (0, 129)


def test_captured(dev):
    x, w, bias, res = make(300, 1024, 768, "bf16")
    few = QuantizedMatrix(x.values[:3], x.scales[:3], x.compute_dtype)
    odd, wodd, _, _ = make(200, 1000, 99, "bf16")

    def step():
        return quantized_linear(x, w, bias, "gelu_tanh", res), quantized_linear(few, w, bias), quantized_linear(odd, wodd)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        x.values.copy_(torch.randint(-127, 128, x.values.shape, device=dev, dtype=torch.int8))
        odd.values.copy_(torch.randint(-127, 128, odd.values.shape, device=dev, dtype=torch.int8))
        want = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(map(torch.equal, out, want)), k


def test_feed_forward_in_8_bits_is_near_the_linear_one(dev):
    """norm -> int8 product + GELU -> rows in 8 bits -> int8 product + residual, against the framework's
    16-bit activations. Rounding a row to 127 steps of its largest value is off by at most top / 254 an
    element; over a sum of K such errors times the weights their root sum of squares counts."""
    M, K, N = 130, 512, 1024
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(M, K, generator=g, device=dev).bfloat16()
    w1 = quantize_frozen_matrix((torch.randn(N, K, generator=g, device=dev) * 0.04).bfloat16())
    w2 = quantize_frozen_matrix((torch.randn(K, N, generator=g, device=dev) * 0.03).bfloat16())
    h = quantized_linear(rms_norm_quantized(x).output, w1, activation="gelu_tanh")
    y = quantized_linear(quantize_rows(h), w2, residual=x)
    ref_h = gelu(_weight_mul(w1, rms_norm(x).output).float()).bfloat16()
    ref = _weight_mul(w2, ref_h).float() + x.float()
    # codes: rms error top / (254 sqrt 3) = 0.0092 of a row's rms for a top of 4 rms; two products
    # and bf16 roundings: below 3% of the update's rms
    err = (y.float() - ref).square().mean().sqrt()
    assert float(err) < 0.03 * float((ref - x.float()).square().mean().sqrt()) + 2.0 ** -9 * float(ref.abs().max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 4111, 33), (5, 300, 70), (70, 260, 100), (1100, 1796, 1024), (4100, 1024, 2304)])
def test_sums_past_the_f32_range_before_the_weight_scale(dev, M, K, N, dtype):
    """Rows of 1e30 and more under a weight of small scales: the sum times the row's scale alone passes
    the f32 range, the result does not."""
    x, w, bias, res = make(M, K, N, dtype)
    x.scales[::2] = torch.rand(x.scales[::2].shape, device=dev) * 3e36 + 1e32
    w.scales.copy_(torch.rand(N, device=dev) * 1e-12 + 1e-14)
    for kw in (dict(), dict(bias=bias), dict(bias=bias, residual=res)):
        check(quantized_linear(x, w, **kw), x, w, kw.get("bias"), kw.get("residual"), False, str(list(kw)))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("K,N", [(4097, 9), (4111, 33), (5135, 64), (7501, 17), (8190, 40), (131071, 5)])
def test_one_token_of_any_length(dev, K, N, dtype):
    """One long token: lanes with fewer turns than others, pieces of 16 codes that end in the row's
    end, codes at odd addresses."""
    x, w, bias, res = make(1, K, N, dtype)
    check(quantized_linear(x, w), x, w, None, None, False, "plain")
    want = quantized_linear(x, w, bias, "gelu_tanh", res)
    check(want, x, w, bias, res, True, "bias, gelu, residual")
    for off in (1, 2, 7):
        flat = torch.zeros(off + K + N * K, dtype=torch.int8, device=dev)
        xv, wv = flat[off:off + K].view(1, K), flat[off + K:].view(N, K)
        xv.copy_(x.values)
        wv.copy_(w.values)
        y = quantized_linear(QuantizedMatrix(xv, x.scales, x.compute_dtype),
                             QuantizedMatrix(wv, w.scales, w.compute_dtype), bias, "gelu_tanh", res)
        assert torch.equal(y, want), off


@pytest.mark.parametrize("dtype", list(DT))
def test_long_rows_do_not_depend_on_their_place(dev, dtype):
    """One token, a few, hundreds and thousands take different kernels; a row has the same bits in all."""
    for M, K, N in ((300, 4111, 99), (1500, 4111, 260), (1500, 5120, 300), (4200, 5120, 1100)):
        x, w, bias, res = make(M, K, N, dtype)
        for act in (None, "gelu_tanh"):
            whole = quantized_linear(x, w, bias, act, res)
            for a, b in ((0, 1), (M - 1, M), (3, 19), (1, 70), (M // 2, M)):
                part = quantized_linear(QuantizedMatrix(x.values[a:b], x.scales[a:b], x.compute_dtype), w, bias,
                                        act, res[a:b])
                assert torch.equal(part, whole[a:b]), (K, N, act, a, b)
