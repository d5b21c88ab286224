"""Rows in microscaled 4 bits against their definition in 64 bits (codes and scale bytes are equal), and
their product. Products of two values and two powers of two are exact; one matrix instruction adds 64 or 128
of them, in any order at most 128 roundings, K / 64 instructions follow each other and up to eight waves'
sums are joined: (128 + K / 64 + 8) u of the sum of magnitudes, doubled for sums that are cut and not
rounded. The bias adds u, the GELU 1.13 times its argument's error and 6 u, the residual u."""
import pytest
import torch

import reels_amd as ra
from reels_amd import MicroscaledMatrix, microscaled_linear, quantize_microscaled
from tests._blocks import blocks4, hard_rows, nibbles
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ROWS = [(1, 1), (3, 7), (5, 31), (64, 32), (65, 33), (100, 101), (70, 256), (9, 257), (130, 1000), (200, 1536), (3, 13825)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K", ROWS)
def test_rows(dev, M, K, dtype):
    x = hard_rows(M, K, DT[dtype], dev)
    q = quantize_microscaled(x)
    c, s, v = blocks4(x.double())
    assert q.shape == (M, K) and q.compute_dtype == DT[dtype]
    assert torch.equal(q.block_scales(), s)
    assert torch.equal(nibbles(q), c)
    whole = torch.stack((q.codes & 15, q.codes >> 4), dim=-1).flatten(1)
    assert not bool(whole[:, K:].any())  # zeros up to the tile's end
    for d in DT.values():
        r = v.to(d)
        if d == torch.float16:  # saturates
            r = torch.where(torch.isinf(r), torch.sign(r) * 65504, r)
        got = q.dequantize(d)
        assert torch.equal(torch.isnan(got), torch.isnan(r))
        assert torch.equal(got.nan_to_num(7.0), r.nan_to_num(7.0)), d
    packed = torch.nn.functional.pad(c, (0, K % 2))
    again = MicroscaledMatrix.from_blocks(packed[:, 0::2] + 16 * packed[:, 1::2], s, K, DT[dtype])
    assert torch.equal(again.codes, q.codes) and torch.equal(again.block_scales(), s)
    assert torch.equal(again.dequantize(torch.float32).nan_to_num(7.0), v.float().nan_to_num(7.0))


def test_row_strides(dev):
    x = torch.randn(90, 300, device=dev, dtype=torch.bfloat16)
    for v in (x[:, 3:203], x[::2, :100], x.t()[:100], x.reshape(-1)[1:1 + 60 * 40].view(60, 40)):
        a, b = quantize_microscaled(v), quantize_microscaled(v.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a.codes, b.codes) and torch.equal(a.block_scales(), b.block_scales())


def make(M, K, N, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M + 7 * K + 13 * N)

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda")
    # rows and columns of different sizes, so that a scale in the wrong place shows
    x = quantize_microscaled((rnd(M, K) * torch.exp2(torch.round(3 * rnd(M, 1))) * torch.exp2(torch.round(2 * rnd(1, K)))).to(DT[dtype]))
    w = quantize_microscaled((rnd(N, K) * torch.exp2(torch.round(3 * rnd(N, 1))) * torch.exp2(torch.round(2 * rnd(1, K))) / K ** 0.5).bfloat16())
    return x, w, rnd(N).to(DT[dtype]), rnd(M, N).to(DT[dtype])


def check(y, x, w, bias=None, res=None, act=False, what=""):
    xv, wv = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    v = torch.matmul(xv, wv.t().contiguous())
    slack = 2 * (136 + x.shape[1] / 64) * U * torch.matmul(xv.abs(), wv.abs().t().contiguous())
    if bias is not None:
        v = v + bias.double()
        slack = slack + U * v.abs()
    if act:
        slack = 1.13 * slack + 6 * U * v.abs()
        v = torch.nn.functional.gelu(v, approximate="tanh")
    if res is not None:
        v = v + res.double()
        slack = slack + U * v.abs()
    if y.dtype == torch.float16:  # past its range: half a step over the largest value
        v = torch.where(v.abs() >= 65520, torch.sign(v) * float("inf"), v)
    assert_within(y, v, slack, f"y {what}")


# tokens, inputs, outputs: single tokens, edges of the tiles of every form, odd widths
SIZES = [(1, 1, 1), (1, 64, 16), (1, 5120, 1000), (2, 100, 77), (3, 17, 5), (7, 1536, 1537), (16, 256, 64), (15, 6000, 65),
         (17, 130, 33), (31, 512, 130), (33, 1000, 300), (64, 64, 64), (65, 65, 65), (100, 2048, 513),
         (128, 384, 256), (129, 1024, 257), (200, 4096, 640), (255, 640, 255), (300, 20000, 20),
         (513, 128, 769), (777, 1000, 3001), (4100, 1024, 2304), (4099, 1028, 2310), (40000, 100, 2048),
         (20001, 256, 2049), (20001, 300, 2049), (1025, 896, 1024), (2100, 1537, 130), (5000, 256, 512)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(dev, M, K, N, dtype):
    x, w, bias, res = make(M, K, N, dtype)
    y = microscaled_linear(x, w)
    assert y.dtype == DT[dtype] and y.shape == (M, N)
    check(y, x, w, what="plain")
    check(microscaled_linear(x, w, bias, "gelu_tanh", res), x, w, bias, res, True, "bias, gelu, residual")
    check(microscaled_linear(x, w, None, None, res), x, w, None, res, False, "residual")
    check(microscaled_linear(x, w, bias), x, w, bias, None, False, "bias")
    bits = torch.int32 if dtype == "f32" else torch.int16  # an f16 operand holds infinities where the sizes meet
    assert torch.equal(y.view(bits), microscaled_linear(x, w).view(bits))


@pytest.mark.parametrize("M", [5, 40, 300, 3000])
def test_not_finite(dev, M):
    """A block that held NaN makes its row NaN and no other, in every form; so does a weight's its column."""
    g = torch.Generator(device=dev).manual_seed(M)
    a = torch.randn(M, 700, generator=g, device=dev).bfloat16()
    b = torch.randn(2050, 700, generator=g, device=dev).bfloat16()
    a[M - 1, 699], b[2049, 3], b[1000, 300] = float("nan"), float("inf"), float("nan")
    y = microscaled_linear(quantize_microscaled(a), quantize_microscaled(b))
    bad = torch.isnan(y)
    assert bad[M - 1].all() and bad[:, 2049].all() and bad[:, 1000].all()
    bad[M - 1] = False
    bad[:, 2049] = bad[:, 1000] = False
    assert not bad.any() and not torch.isinf(y).any()


def test_dtype_empty_and_in_place(dev):
    x, w, bias, _ = make(40, 64, 33, "bf16")
    check(microscaled_linear(x, w, dtype=torch.float32), x, w)
    check(microscaled_linear(x, w, bias.half(), dtype=torch.float16), x, w, bias.half())
    e = quantize_microscaled(torch.empty(0, 64, device=dev, dtype=torch.bfloat16))
    assert microscaled_linear(e, w).shape == (0, 33) and e.dequantize().shape == (0, 64)
    for M in (9, 100, 3000):  # y over the residual
        x, w, bias, res = make(M, 300, 1030, "bf16")
        y = microscaled_linear(x, w, bias, None, res)
        L = ra._lib.lib()
        assert L.reels_hip_mx4_linear(x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
                                      bias.data_ptr(), res.data_ptr(), 0, 1, M, 300, 1030, res.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(res, y)


def test_slices_and_offsets(dev):
    """Rows of a larger operand in whole tiles, bias and residual at odd places, strided codes."""
    x, w, bias, res = make(300, 520, 130, "bf16")
    part = MicroscaledMatrix(x.codes[64:200], x.scales[1:4], (136, 520), torch.bfloat16)
    check(microscaled_linear(part, w, bias, None, res[64:200]), part, w, bias, res[64:200])
    b = torch.cat([bias[:1], bias])[1:]
    r = torch.cat([res.reshape(-1)[:1], res.reshape(-1)])[1:].view(300, 130)
    assert torch.equal(microscaled_linear(x, w, b, None, r), microscaled_linear(x, w, bias, None, res))
    wide = MicroscaledMatrix(torch.cat([x.codes, x.codes], 1)[:, :384], x.scales, (300, 520), torch.bfloat16)
    assert torch.equal(microscaled_linear(wide, w), microscaled_linear(x, w))
    off = torch.empty(x.codes.numel() + 4, dtype=torch.uint8, device=dev)[4:].view_as(x.codes).copy_(x.codes)
    assert torch.equal(microscaled_linear(MicroscaledMatrix(off, x.scales, (300, 520)), w), microscaled_linear(x, w))


def test_other_stream_and_graph(dev):
    for M in (1, 50, 2000):
        x, w, bias, res = make(M, 1000, 1030, "bf16")
        a = torch.randn(M, 1000, device=dev, dtype=torch.bfloat16)
        y0 = microscaled_linear(x, w, bias, "gelu_tanh", res)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            y1 = microscaled_linear(x, w, bias, "gelu_tanh", res)
        torch.cuda.current_stream().wait_stream(st)
        assert torch.equal(y0, y1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y2 = microscaled_linear(quantize_microscaled(a), w, bias, "gelu_tanh", res)
        for _ in range(3):
            a.copy_(torch.randn_like(a))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y2, microscaled_linear(quantize_microscaled(a), w, bias, "gelu_tanh", res))


def test_offsets_past_32_bits(dev):
    """Codes of more than 2^32 bytes and outputs past 2^32 elements: the last rows are those of a small call."""
    K, N = 13824, 7001
    x = quantize_microscaled(torch.randn(128, K, device=dev).bfloat16())
    w = quantize_microscaled(torch.randn(N, K, device=dev).bfloat16())
    times = 5000  # 640000 rows: 4.4 GB of codes
    big = MicroscaledMatrix(x.codes.repeat(times, 1), x.scales.repeat(times, 1, 1), (128 * times, K), torch.bfloat16)
    y = microscaled_linear(big, w)
    ref = y[:128]
    check(ref, x, w)
    assert torch.equal(y[-128:], ref) and torch.equal(y[128 * 4999 - 128 * 2000:128 * 4999 - 128 * 1999], ref)
    del y
    v = big.dequantize()
    assert torch.equal(v[-128:], x.dequantize())
    q = quantize_microscaled(v)
    assert torch.equal(q.codes[-128:], big.codes[-128:]) and torch.equal(q.scales[-2:], big.scales[-2:])
