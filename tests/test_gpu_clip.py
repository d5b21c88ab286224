"""Global gradient norm and clipping against sums in 64 bits: the norm is rounded once to f32 (2^-24,
and 2^-45 of the sum's own), a clipped value has the factor's rounding and one product's (2 u) before
the rounding to its type."""
import math

import pytest
import torch

from reels_amd import QuantizedMatrix, clip_gradients, gradient_norm, i8lora_backward
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def make(sizes, dtypes, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(DT[d]) for s, d in zip(sizes, dtypes)]


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


LISTS = [([1], ["f32"]), ([0, 5, 0], ["f32"] * 3), ([16384, 16385, 16383], ["f32", "bf16", "f16"]),
         ([(33, 7), (3, 1537), (100001,)], ["bf16", "f32", "f16"]), ([(3,)] * 97, ["f32"] * 97),
         ([(64, 33)] * 300, ["f32", "bf16", "f16"] * 100), ([40_000_000], ["bf16"])]


@pytest.mark.parametrize("sizes,dtypes", LISTS)
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9, math.inf])
def test_norm_and_clipped(dev, sizes, dtypes, max_norm):
    grads = make(sizes, dtypes)
    want = norm64(grads)
    n = gradient_norm(grads)
    assert n.shape == () and n.dtype == torch.float32
    assert abs(float(n) - want) <= 1.01 * U * want
    out = [torch.full_like(g, 7) for g in grads]
    m = clip_gradients(grads, max_norm, out=out)
    assert torch.equal(m, n)
    f = min(1.0, max_norm / (want + 1e-6))
    for g, o in zip(grads, out):
        assert_within(o, g.double() * f, 2 * U * g.double().abs() * f, "clipped")
        if f == 1.0:
            assert torch.equal(o, g)
    keep = [g.clone() for g in grads]
    k = clip_gradients(keep, max_norm)
    assert torch.equal(k, n) and all(torch.equal(a, b) for a, b in zip(keep, out))


def test_pieces_of_buffers_at_any_offset(dev):
    """Gradients and outputs that lie one after the other at odd places: nothing beside them moves."""
    for dt in DT.values():
        src, dst = (torch.randn(5000, device=dev).to(dt) for _ in range(2))
        before = dst.clone()
        cuts = [(1, 1000), (1003, 17), (1021, 3000)]
        clip_gradients([src[a:a + n] for a, n in cuts], 0.25, out=[dst[a + 3:a + 3 + n] for a, n in cuts])
        f = 0.25 / (norm64([src[a:a + n] for a, n in cuts]) + 1e-6)
        mask = torch.ones(5000, dtype=torch.bool, device=dev)
        for a, n in cuts:
            mask[a + 3:a + 3 + n] = False
            s = src[a:a + n].double()
            assert_within(dst[a + 3:a + 3 + n], s * f, 2 * U * s.abs() * f, "piece")
        assert torch.equal(dst[mask], before[mask])


def test_not_finite_stays(dev):
    for bad in (math.nan, math.inf, -math.inf):
        g = [torch.randn(1000, device=dev), torch.randn(50, device=dev).bfloat16()]
        g[0][17] = bad
        want = [t.clone() for t in g]
        n = clip_gradients(g, 1.0)
        assert not math.isfinite(float(n))
        assert all(torch.equal(a.nan_to_num(5.0, 6.0, 7.0), b.nan_to_num(5.0, 6.0, 7.0)) for a, b in zip(g, want))
    # large finite values whose squares pass the f32 range
    g = [torch.full((1000,), 1e30, device=dev)]
    n = clip_gradients(g, 1.0)
    assert abs(float(n) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert_within(g[0], torch.full((1000,), 1 / math.sqrt(1000), dtype=torch.float64), 1e-8, "large")


def test_dense_orders_and_none(dev):
    a = torch.randn(30, 70, device=dev)
    g = [a.t(), None, torch.randn(2, 3, 4, 5, device=dev).contiguous(memory_format=torch.channels_last)]
    want = norm64([g[0], g[2]])
    before = [t if t is None else t.clone() for t in g]
    n = clip_gradients(g, 1.0)
    assert abs(float(n) - want) <= 1.01 * U * want
    for t, b in zip(g, before):
        if t is not None:
            assert_within(t, b.double() / (want + 1e-6), 2 * U * b.abs() / want, "in place")


def test_same_bits_again(dev):
    grads = make([(64, 333)] * 50 + [3_000_001], ["f32"] * 50 + ["f16"])
    assert torch.equal(gradient_norm(grads), gradient_norm([g.clone() for g in grads]))


def test_captured(dev):
    grads = make([(700, 16)] * 120, ["f32"] * 120)
    out = [torch.empty_like(g) for g in grads]
    clip_gradients(grads, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(grads, 1.0, out=out)
    for k in range(3):
        for g in grads:
            g.copy_(torch.randn_like(g))
        want_out = [torch.empty_like(g) for g in grads]
        want = clip_gradients(grads, 1.0, out=want_out)
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(map(torch.equal, out, want_out)), k


def test_adapter_gradients_are_clipped_together(dev):
    """What i8lora_backward returns for several layers goes straight in."""
    g = torch.Generator(device=dev).manual_seed(5)
    grads = []
    for K, N in ((64, 96), (96, 64)):
        w = QuantizedMatrix(torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8),
                            torch.full((N,), 1e-3, device=dev))
        x, dy, A, B = (torch.randn(s, generator=g, device=dev).bfloat16()
                       for s in ((40, K), (40, N), (K, 4), (4, N)))
        grads += list(i8lora_backward(dy, x, w, A, B, 1.0)[1:])
    before = [t.clone() for t in grads]
    n = clip_gradients(grads, 1.0)
    want = norm64(before)
    assert want > 1 and abs(float(n) - want) <= 1.01 * U * want
    for t, b in zip(grads, before):
        assert_within(t, b.double() / (want + 1e-6), 2 * U * b.abs() / want, "clipped")


def test_what_is_clipped_counts_as_changed(dev):
    """A graph that has saved a tensor notices that it was clipped in place, or written as an output."""
    g, h, out = (torch.randn(40, device=dev) for _ in range(3))
    p = torch.randn(40, device=dev, requires_grad=True)
    for write in (lambda: clip_gradients([g, None, h], 0.1), lambda: clip_gradients([h], 0.1, out=[g])):
        loss = (p * g).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # what is only read does not count as changed
    loss = (p * g).sum()
    clip_gradients([g], 0.1, out=[out])
    gradient_norm([g])
    loss.backward()
    assert torch.equal(p.grad, g)


def test_clipping_a_tensor_of_inference_mode(dev):
    """Tensors of inference mode have no count of changes; they are clipped like others."""
    with torch.inference_mode():
        g = torch.randn(100, device=dev)
        want = norm64([g])
        b = g.clone()
        clip_gradients([g], 0.5)
        assert_within(g, b.double() * (0.5 / (want + 1e-6)), 2 * U * b.double().abs() * (0.5 / want), "clipped")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norms_past_the_f32_range_leave_the_gradients(dev, dtype):
    """The norm that is returned decides: where it is infinite, the gradients stay."""
    for n in (2, 1000, 40001):
        g = [torch.full((n,), 3e38, device=dev).to(DT[dtype]), torch.randn(5, device=dev)]
        want = [t.clone() for t in g]
        out = [torch.empty_like(t) for t in g]
        assert float(gradient_norm(g)) == math.inf
        assert float(clip_gradients(g, 1.0, out=out)) == math.inf and all(map(torch.equal, out, want))
        assert float(clip_gradients(g, 1.0)) == math.inf and all(map(torch.equal, g, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_factors_below_the_f32_range(dev, dtype):
    """A factor that f32 holds with fewer bits, or not at all: the products keep theirs."""
    for size, max_norm in ((1e36, 1e-6), (1e36, 1e-3), (1.2e36, 2e-9), (1e30, 1e-15), (1e36, 0.01)):
        g = [torch.randn(70001, device=dev).mul_(size).to(DT[dtype])]
        want = norm64(g)
        f = float(torch.tensor(max_norm)) / want
        b = g[0].double()
        n = clip_gradients(g, max_norm)
        assert abs(float(n) - want) <= 1.01 * U * want
        assert_within(g[0], b * f, 2 * U * b.abs() * f, f"{size} {max_norm}")


def test_none_in_both_lists(dev):
    g = make([5, 7, 9], ["f32"] * 3)
    want = [t.clone() for t in g]
    clip_gradients(want, 0.25)
    out = [torch.zeros_like(t) for t in g]
    clip_gradients([None, g[0], None, g[1], g[2]], 0.25, out=[None, out[0], None, out[1], out[2]])
    assert all(map(torch.equal, out, want))
    for bad in ([None, *out, None], [out[0], None, None, out[1], out[2]], out):
        with pytest.raises(ValueError, match="one by one"):
            clip_gradients([None, g[0], None, g[1], g[2]], 0.25, out=bad)
