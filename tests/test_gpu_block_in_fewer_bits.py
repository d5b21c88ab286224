"""The operators of a block in fewer bits as they are used together: one feed-forward sublayer between two
modulated norms, sampled in 4 bits, and trained with its activations kept in 8 bits."""
import pytest
import torch

import reels_amd as ra
from tests._blocks import blocks4, blocks8
from tests._util import assert_parity

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make(dev, B=2, S=150, C=320, H=900, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, generator=g, device=dev)
    six = 0.3 * rnd(B, 6, C)
    return dict(x=rnd(B, S, C).to(BF), attn=rnd(B, S, C).to(BF), six=six, w1=(rnd(H, C) / C ** 0.5).to(BF), b1=(0.1 * rnd(H)).to(BF),
                w2=(rnd(C, H) / H ** 0.5).to(BF), b2=(0.1 * rnd(C)).to(BF), B=B, S=S, C=C, H=H, rnd=rnd)


def test_sampling_in_4_bits(dev):
    t = make(dev)
    B, S, C, H = t["B"], t["S"], t["C"], t["H"]
    shift, scale, gate, gate2, shift2, scale2 = (t["six"][:, i:i + 1] for i in range(6))
    w1, w2 = ra.quantize_microscaled(t["w1"]), ra.quantize_microscaled(t["w2"])

    def block():
        n = ra.modulated_norm_quantized(t["x"], scale, shift, branch=t["attn"], gate=gate)
        h = ra.microscaled_linear(n.output, w1, t["b1"], "gelu_tanh")
        y = ra.microscaled_linear(ra.quantize_microscaled(h), w2, t["b2"])
        return n, h, y, ra.modulated_norm(n.sum, scale2, shift2, branch=y.view(B, S, C), gate=gate2)
    n, h, y, out = block()
    # each step against 64 bits from what the step before it stored
    s = (t["x"].float() + gate * t["attn"].float()).to(BF)
    assert torch.equal(n.sum, s)
    sd = s.double()
    c = sd - sd.mean(-1, keepdim=True)
    v = (c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + scale.double()) + shift.double()).view(-1, C)
    q = blocks4(v.float().double())[2]
    assert float((n.output.dequantize(torch.float32) != q.float()).float().mean()) < 1e-4
    w1d, w2d = (blocks4(w.double())[2].t().contiguous() for w in (t["w1"], t["w2"]))
    hd = torch.nn.functional.gelu(n.output.dequantize(torch.float32).double() @ w1d + t["b1"].double(), approximate="tanh")
    assert_parity(h.float().cpu().numpy(), hd.cpu().numpy(), "h")
    yd = blocks4(h.double())[2] @ w2d + t["b2"].double()
    assert_parity(y.float().cpu().numpy(), yd.cpu().numpy(), "y")
    sd = out.sum.double()
    assert torch.equal(out.sum, (s.float() + gate2 * y.view(B, S, C).float()).to(BF))
    c = sd - sd.mean(-1, keepdim=True)
    od = c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + scale2.double()) + shift2.double()
    assert_parity(out.output.float().cpu().numpy(), od.cpu().numpy(), "output")
    graph = torch.cuda.CUDAGraph()
    block()
    with torch.cuda.graph(graph):
        rec = block()
    for _ in range(3):
        t["x"].copy_(torch.randn_like(t["x"]))
        graph.replay()
        torch.cuda.synchronize()
        now = block()
        assert torch.equal(rec[3].output, now[3].output) and torch.equal(rec[3].sum, now[3].sum) and torch.equal(rec[2], now[2])


def step(t, leaves, kept, dy, ds):
    """Forward and backward of the sublayer; kept: its activations in 8 bits."""
    x, attn, six, A1, B1, A2, B2, W1, W2 = leaves
    shift, scale, gate, gate2, shift2, scale2 = (six[:, i:i + 1] for i in range(6))
    B, S, C, H = t["B"], t["S"], t["C"], t["H"]
    n, s = ra.ModulatedNormFunction.apply(x, scale, shift, attn, gate, 1e-6, True, kept)
    keep = ra.compress_activations if kept else (lambda v: None)
    flat = n.reshape(-1, C)
    z = ra.I8LoRALinearFunction.apply(flat, A1, B1, W1.values, W1.scales, t["b1"], 2.0, keep(flat.detach()))
    if kept:
        h = ra.GeluTanhCompressedFunction.apply(z)
    else:
        h = torch.nn.functional.gelu(z.float(), approximate="tanh").to(BF)
    y = ra.I8LoRALinearFunction.apply(h, A2, B2, W2.values, W2.scales, t["b2"], 2.0, keep(h.detach()))
    o, s2 = ra.ModulatedNormFunction.apply(s, scale2, shift2, y.view(B, S, C), gate2, 1e-6, True, kept)
    grads = torch.autograd.grad((o, s2), leaves[:7], (dy, ds))
    return o.detach(), s2.detach(), grads


def test_training_with_activations_in_8_bits(dev):
    t = make(dev, seed=5)
    C, H, rnd = t["C"], t["H"], t["rnd"]
    W1, W2 = ra.quantize_frozen_matrix(t["w1"]), ra.quantize_frozen_matrix(t["w2"])
    leaves = [t["x"], t["attn"], t["six"], rnd(C, 8) / C ** 0.5, rnd(8, H) / 8, rnd(H, 8) / H ** 0.5, rnd(8, C) / 8]
    leaves = [v.clone().requires_grad_() for v in leaves] + [W1, W2]
    dy, ds = rnd(*t["x"].shape).to(BF), rnd(*t["x"].shape).to(BF)
    kept, whole = step(t, leaves, True, dy, ds), step(t, leaves, False, dy, ds)
    assert torch.equal(kept[1], step(t, leaves, True, dy, ds)[1])
    # the forwards differ by the GELU's bits alone, the gradients by activations rounded to 7 bits (2^-7 of a
    # block's largest at most, near 1% of its size for ordinary values): a few of those along the chain
    for a, b, tol in [(kept[0], whole[0], 0.01), (kept[1], whole[1], 0.01)] + [(a, b, 0.05) for a, b in zip(kept[2], whole[2])]:
        assert float((a.double() - b.double()).norm() / b.double().norm()) < tol
    for a, b in zip(kept[2], step(t, leaves, True, dy, ds)[2]):
        assert torch.equal(a, b)  # bitwise reproducible
    # 33 bytes for 32 elements are kept of each activation
    k = ra.compress_activations(t["x"])
    assert k.values.nbytes + k.scales.nbytes == t["x"].numel() * 33 // 32
    assert torch.equal(k.restore().view(-1, C).double(), blocks8(t["x"].double().view(-1, C))[2])


def test_two_threads_on_two_streams(dev):
    """Calls of two threads at once, each on its own stream, with operands of its own."""
    import threading
    from reels_amd import _lib
    cases = []
    for seed, size in ((1, dict(S=150, C=320, H=900)), (2, dict(S=77, C=1000, H=260))):
        t = make(dev, seed=seed, **size)
        w1 = ra.quantize_microscaled(t["w1"])
        shift, scale, gate = (t["six"][:, i:i + 1] for i in range(3))
        dy = t["rnd"](t["B"], t["S"], t["C"]).to(BF)

        def work(t=t, w1=w1, shift=shift, scale=scale, gate=gate, dy=dy):
            n = ra.modulated_norm_quantized(t["x"], scale, shift, branch=t["attn"], gate=gate)
            h, kept = ra.gelu_tanh_compressed(ra.microscaled_linear(n.output, w1, t["b1"]))
            r = ra.modulated_norm(t["x"], scale, shift, branch=t["attn"], gate=gate, compress=True)
            g = ra.modulated_norm_backward(dy, r.kept.sum, r.stats, scale, branch=r.kept.branch, gate=gate)
            return [h, kept.restore(), ra.gelu_tanh_backward(kept, h), r.output] + list(g)
        cases.append(work)
    want = [f() for f in cases]
    torch.cuda.synchronize()
    errors = []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = cases[i]()
                torch.cuda.current_stream().synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
            # a refused call's message belongs to the thread that made it
            assert _lib.lib().reels_hip_act8_keep(None, 1, 1 if i else -1, 8, None, None, None) != 0
            assert ("NULL" in _lib.lib().reels_hip_last_error().decode()) == bool(i)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
