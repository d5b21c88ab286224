"""The modulated norm, its rows in 8 and 4 bits and its backward against the formulas in 64 bits. Bounds
count f32 roundings (u = 2^-24). y: s - mean has 2 u, rstd and its product 2 u, 1 + scale u, the sum u. d:
g = dy (1 + scale) 2 u, n 4 u; mean g and mean g n add chunks of at most eight terms in f32 (8 u) before
they go on in 64 bits, and are rounded: 12 u and 18 u of the means of magnitudes; then three differences and
products. Sums over rows follow each other in a thread, then over at most 16 groups, 32 slices and
parts / 32 partial rows: 100 + rows / 64 roundings at most."""
import pytest
import torch

from reels_amd import (CompressedActivations, ModulatedNormFunction, modulated_norm, modulated_norm_backward,
                       modulated_norm_quantized, rms_norm)
from tests._blocks import blocks4, blocks8, nibbles
from tests._util import U, assert_within

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6

# samples, tokens, columns: one element, below and past a chunk, the forms of a wave and of a workgroup
SIZES = [(1, 1, 1), (2, 3, 2), (1, 5, 7), (3, 11, 8), (2, 50, 101), (1, 17, 128), (2, 20, 256), (3, 3, 517), (2, 33, 1000),
         (1, 64, 1536), (2, 7, 2049), (1, 5, 4096), (2, 3, 5120), (1, 5, 8193), (1, 3, 13824), (2, 2, 16384)]


def make(B, S, C, dtype, mtype, kind, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed + B * 7 + S * 131 + C)
    dt = DT[dtype]

    def rnd(*s):
        return torch.randn(s, generator=g, device=dev)
    m = {"all": (C,), "sample": (B, C), "token": (B, S, C)}[kind]
    t = dict(x=(rnd(B, S, C) * 1.5 + 2 * rnd(C)).to(dt), branch=rnd(B, S, C).to(dt), dy=rnd(B, S, C).to(dt),
             dsum=rnd(B, S, C).to(dt))
    return t, dict(gate=rnd(*m).to(DT[mtype]), scale=(0.3 * rnd(*m)).to(DT[mtype]), shift=rnd(*m).to(DT[mtype]))


def rows(m, B):
    return m[:, None, :] if m.dim() == 2 else m


def unit(s, center, eps=EPS):
    sd = s.double()
    mean = sd.mean(-1, keepdim=True) if center else torch.zeros_like(sd[..., :1])
    rstd = 1.0 / torch.sqrt((sd - mean).square().mean(-1, keepdim=True) + float(torch.tensor(eps)))
    return sd, mean, rstd


def check_forward(res, x, branch, gate, scale, shift, center, B):
    if branch is None:
        assert res.sum is x
    else:
        p = branch.float() if gate is None else rows(gate, B).float() * branch.float()
        assert torch.equal(res.sum, (x.float() + p).to(x.dtype))
    sd, mean, rstd = unit(res.sum, center)
    st = res.stats.double()
    mag = sd.abs().mean(-1)
    assert bool(((st[..., 0] + st[..., 1] - mean[..., 0]).abs() <= 2.0 ** -40 * mag).all())
    assert_within(res.stats[..., 2], rstd[..., 0], U * rstd[..., 0], "rstd")
    n = (sd - mean) * rstd
    up = 1.0 if scale is None else 1.0 + rows(scale, B).double()
    y = n * up + (0.0 if shift is None else rows(shift, B).double())
    assert_within(res.output, y, 7 * U * (n * up).abs() + U * y.abs(), "y")


def check_backward(g, t, s, branch, stats, gate, scale, dsum, center, B, S):
    C = t["dy"].shape[-1]
    st = stats.double()
    n = (s - (st[..., 0] + st[..., 1])[..., None]) * st[..., 2:]
    rs = st[..., 2:]
    up = torch.ones(C, dtype=torch.float64, device=s.device) if scale is None else 1.0 + rows(scale, B).double()
    dy = t["dy"].double()
    gd = dy * up
    m0 = gd.mean(-1, keepdim=True) if center else 0.0
    m1 = (gd * n).mean(-1, keepdim=True)
    a0 = gd.abs().mean(-1, keepdim=True) if center else 0.0
    a1 = (gd * n).abs().mean(-1, keepdim=True)
    d = rs * (gd - m0 - n * m1)
    slack = rs * U * (8 * gd.abs() + 16 * a0 + 28 * n.abs() * a1)
    if dsum is not None:
        d = d + dsum.double()
        slack = slack + 2 * U * (dsum.double().abs() + d.abs())
    assert_within(g.x, d, slack, "dx")
    if gate is None:
        assert g.branch is g.x
    else:
        gt = rows(gate, B).double()
        assert_within(g.branch, d * gt, slack * gt.abs() + U * (d * gt).abs(), "dbranch")

    def total(v, like):
        return v if like.dim() == 3 else v.sum(1) if like.dim() == 2 else v.sum((0, 1))
    deep = (100 + B * S / 64) * U
    if scale is not None:
        assert_within(g.scale, total(dy * n, scale), total(deep * (dy * n).abs(), scale), "dscale")
        assert_within(g.shift, total(dy, scale), total(deep * dy.abs(), scale), "dshift")
        assert g.scale.shape == scale.shape
    if gate is not None and branch is not None:
        assert_within(g.gate, total(d * branch, gate), total(slack * branch.abs() + deep * (d * branch).abs(), gate), "dgate")


@pytest.mark.parametrize("dtype,mtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("B,S,C", SIZES)
def test_forward_and_backward(dev, B, S, C, dtype, mtype):
    for kind, center, compress in (("sample", True, False), ("token", False, False), ("all", True, True), ("sample", False, True),
                                   ("token", True, True)):
        t, m = make(B, S, C, dtype, mtype, kind)
        r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], EPS, center, compress)
        check_forward(r, t["x"], t["branch"], m["gate"], m["scale"], m["shift"], center, B)
        s, b, sd, bd = r.sum, t["branch"], r.sum.double(), t["branch"].double()
        if compress:
            s, b = r.kept.sum, r.kept.branch
            for k, of in ((s, r.sum), (b, t["branch"])):
                q, sc, v = blocks8(of.double().reshape(-1, C))
                assert torch.equal(k.values.reshape(-1, C), q) and torch.equal(k.scales.reshape(B * S, -1), sc)
            sd, bd = (blocks8(v.reshape(-1, C))[2].reshape(B, S, C) for v in (sd, bd))
        else:
            assert r.kept is None
        g = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], b, m["gate"], t["dsum"], center)
        check_backward(g, t, sd, bd, r.stats, m["gate"], m["scale"], t["dsum"], center, B, S)
        again = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], b, m["gate"], t["dsum"], center)
        for u, v in zip(g, again):
            assert torch.equal(u, v)
        few = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], None, m["gate"], t["dsum"], center, want_modulation=False)
        assert few.gate is None and few.scale is None and torch.equal(few.x, g.x) and torch.equal(few.branch, g.branch)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,S,C", [(1, 5, 7), (2, 9, 300), (1, 3, 5120)])
def test_parts_left_out(dev, B, S, C, dtype):
    """No modulation, no gate, no branch, no other gradient."""
    t, m = make(B, S, C, dtype, "f32", "sample")
    for branch, gate, scale, dsum in ((None, None, None, None), ("branch", None, None, None), (None, None, "scale", "dsum"),
                                      ("branch", "gate", None, "dsum"), ("branch", None, "scale", None)):
        b, gt, sc, ds = (t.get(n, m.get(n)) if n else None for n in (branch, gate, scale, dsum))
        sh = None if sc is None else m["shift"]
        for compress in (False, True):
            r = modulated_norm(t["x"], sc, sh, b, gt, EPS, True, compress)
            check_forward(r, t["x"], b, gt, sc, sh, True, B)
            s = r.kept.sum if compress else r.sum
            sd = s.restore(torch.float32).double() if compress else s.double()
            kb = b if b is None or not compress else r.kept.branch
            bd = None if b is None else kb.restore(torch.float32).double() if compress else b.double()
            g = modulated_norm_backward(t["dy"], s, r.stats, sc, kb, gt, ds, True)
            check_backward(g, t, sd, bd, r.stats, gt, sc, ds, True, B, S)
            assert (g.gate is None) == (gt is None) and (g.scale is None) == (sc is None)
    if dtype != "f32" or C < 5000:
        # without a mean and a modulation it is the root-mean-square norm
        r, want = modulated_norm(t["x"], eps=EPS, center=False), rms_norm(t["x"], None, EPS)
        assert_within(r.output, want.output.double(), 4 * U * want.output.double().abs()
                      + torch.finfo(DT[dtype]).eps * want.output.double().abs(), "rms")


@pytest.mark.parametrize("dtype,mtype", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("B,S,C", SIZES)
def test_rows_in_4_bits(dev, B, S, C, dtype, mtype):
    """Values in 64 bits rounded to f32, then their codes; a value whose 64-bit sum falls within 2^-45 of a
    border may take either side, and a block whose largest does."""
    for kind, center in (("sample", True), ("token", False)):
        t, m = make(B, S, C, dtype, mtype, kind)
        r = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], EPS, center)
        s = (t["x"].float() + rows(m["gate"], B).float() * t["branch"].float()).to(DT[dtype])
        assert torch.equal(r.sum, s)
        sd, mean, rstd = unit(s, center)
        part, shift = (sd - mean) * rstd * (1.0 + rows(m["scale"], B).double()), rows(m["shift"], B).double()
        y, mag = (part + shift).reshape(-1, C), (part.abs() + shift.abs()).reshape(-1, C)
        c, sc, _ = blocks4(y.float().double())
        near = torch.zeros_like(c, dtype=torch.bool)
        for f in (-2.0 ** -45, 2.0 ** -45):  # codes that another sum of these values may give
            cf, sf, _ = blocks4((y + f * mag).float().double())
            near |= (cf != c) | (sf != sc).repeat_interleave(32, 1)[:, :C]
        assert r.output.shape == (B * S, C) and r.output.compute_dtype == DT[dtype]
        differ = nibbles(r.output) != c
        assert not bool((differ & ~near).any()), int((differ & ~near).sum())
        assert float(near.float().mean()) < 0.01 or C < 64
        whole = torch.stack((r.output.codes & 15, r.output.codes >> 4), dim=-1).flatten(1)
        assert not bool(whole[:, C:].any())


def test_far_mean(dev):
    """Rows whose mean is many times their spread keep their digits."""
    g = torch.Generator(device=dev).manual_seed(5)
    for far in (1e3, 1e5):
        x = (torch.randn(4, 1536, generator=g, device=dev).double() + far).float()
        r = modulated_norm(x, eps=EPS)
        sd, mean, rstd = unit(x, True)
        n = (sd - mean) * rstd
        assert_within(r.output, n, 6 * U * n.abs() + 2.0 ** -40 * far, "y")


def test_large_and_small_values(dev):
    """Squares past the f32 range and below it."""
    for size in (1e30, 1e-25):
        x = (torch.randn(3, 300, device=dev) * size)
        r = modulated_norm(x, eps=0.0)
        sd, mean, rstd = unit(x, True, 0.0)
        n = (sd - mean) * rstd
        assert_within(r.output, n, 8 * U * n.abs() + 2.0 ** -40, "y")


def test_not_finite(dev):
    """A row that holds NaN or an infinity is NaN, and so are its blocks; the others are as without it.
    An infinite gate or scale stays in its own sample."""
    t, m = make(2, 9, 300, "bf16", "f32", "sample")
    x = t["x"].clone()
    x[0, 3, 7], x[1, 5, 299] = float("nan"), float("inf")
    a = modulated_norm(x, m["scale"], m["shift"], t["branch"], m["gate"])
    b = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
    bad = torch.zeros(2, 9, dtype=torch.bool, device=dev)
    bad[0, 3] = bad[1, 5] = True
    assert torch.isnan(a.output[bad]).all() and torch.equal(a.output[~bad], b.output[~bad])
    q = modulated_norm_quantized(x, m["scale"], m["shift"], t["branch"], m["gate"]).output.dequantize().view(2, 9, 300)
    p = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"]).output.dequantize().view(2, 9, 300)
    assert torch.isnan(q[bad]).all() and torch.equal(q[~bad], p[~bad])
    g = modulated_norm_backward(t["dy"], a.sum, a.stats, m["scale"], t["branch"], m["gate"], t["dsum"])
    w = modulated_norm_backward(t["dy"], b.sum, b.stats, m["scale"], t["branch"], m["gate"], t["dsum"])
    assert torch.isnan(g.x[bad]).all() and torch.equal(g.x[~bad], w.x[~bad])
    gate = m["gate"].clone()
    gate[1, 0] = float("inf")
    c = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], gate)
    assert torch.equal(c.output[0], b.output[0]) and torch.isnan(c.output[1]).all()
    scale = m["scale"].clone()
    scale[1, 0] = float("inf")
    c = modulated_norm(t["x"], scale, m["shift"], t["branch"], m["gate"])
    assert torch.equal(c.output[0], b.output[0]) and torch.equal(c.output[1, :, 1:], b.output[1, :, 1:])


def test_strides_and_slices(dev):
    """The modulations as slices of one projection, rows of wider buffers, odd addresses, expanded rows."""
    B, S, C = 3, 20, 258
    g = torch.Generator(device=dev).manual_seed(9)
    six = torch.randn(B, 6, C, generator=g, device=dev)
    x, br, dy = (torch.randn(B, S, C, generator=g, device=dev).bfloat16() for _ in range(3))
    sh, sc, gt = (six[:, i:i + 1] for i in (0, 1, 5))

    def both(*mods, x=x, br=br):
        a = modulated_norm(x, mods[0], mods[1], br, mods[2])
        d = modulated_norm_backward(dy.view_as(a.output), a.sum, a.stats, mods[0], br, mods[2])
        return [t.reshape(-1) for t in (a.output, a.sum) + tuple(d)]
    want = both(sc.reshape(B, C).clone(), sh.reshape(B, C).clone(), gt.reshape(B, C).clone())
    for u, v in zip(both(sc, sh, gt), want):
        assert torch.equal(u, v)
    each = [t.expand(B, S, C) for t in (sc, sh, gt)]
    for u, v in zip(both(*each)[:4], want):
        assert torch.equal(u, v)
    tokens = torch.randn(B, S, 6, C, generator=g, device=dev)
    mods = [tokens[:, :, i] for i in range(3)]
    for u, v in zip(both(*mods), both(*[t.clone() for t in mods])):
        assert torch.equal(u, v)
    wide = torch.randn(B * S, C + 6, generator=g, device=dev).bfloat16()
    wide[:, 3:3 + C] = x.view(-1, C)
    flat = torch.cat([br.reshape(-1)[:1], br.reshape(-1)])[1:].view(B * S, C)
    one = [t[0].reshape(C) for t in (sc, sh, gt)]
    for u, v in zip(both(*one, x=wide[:, 3:3 + C], br=flat), both(*one, x=x.reshape(-1, C), br=br.reshape(-1, C))):
        assert torch.equal(u, v)
    mixed = modulated_norm(x.transpose(0, 1), one[0], one[1], br.transpose(0, 1), one[2])
    assert torch.equal(mixed.output, modulated_norm(x.transpose(0, 1).contiguous(), one[0], one[1],
                                                    br.transpose(0, 1).contiguous(), one[2]).output)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("S,C", [(300, 6), (300, 100), (300, 200), (300, 512), (2100, 1000), (50, 1500), (50, 5120), (20, 9001)])
def test_odd_addresses_of_each_form(dev, S, C, dtype):
    """Operands that start between two vectors, and modulations inside a wider tensor, give the same bits."""
    t, m = make(2, S, C, dtype, "f32", "token")

    def odd(v):
        return torch.cat([v.reshape(-1)[:1], v.reshape(-1)])[1:].view(v.shape)
    wide = torch.stack([odd(m[n]) for n in ("gate", "scale", "shift")], 2)
    inside = dict(zip(("gate", "scale", "shift"), wide.unbind(2)))

    def both(t, m):
        r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], compress=True)
        q = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"]).output
        g = modulated_norm_backward(t["dy"], r.sum, r.stats, m["scale"], t["branch"], m["gate"], t["dsum"])
        k = modulated_norm_backward(t["dy"], r.kept.sum, r.stats, m["scale"], r.kept.branch, m["gate"], t["dsum"])
        return [r.output, r.sum, r.stats, r.kept.sum.values, r.kept.branch.scales, q.codes, q.block_scales()] + list(g) + list(k)
    for u, v in zip(both({n: odd(v) for n, v in t.items()}, inside), both(t, m)):
        assert torch.equal(u, v)


def test_over_the_inputs(dev):
    """The sum over x or the branch, dx over dy or the other gradient: what the C entries allow."""
    from reels_amd import _lib
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for B, S, C in ((2, 9, 300), (1, 7, 5125)):
        t, m = make(B, S, C, "bf16", "f32", "sample")
        r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
        want = modulated_norm_backward(t["dy"], r.sum, r.stats, m["scale"], None, m["gate"], t["dsum"], want_modulation=False)
        p = {n: v.data_ptr() for n, v in m.items()}
        for over in ("x", "branch"):
            c = {n: v.clone() for n, v in t.items()}
            y, stats = torch.empty_like(r.output), torch.empty_like(r.stats)
            assert L.reels_hip_modulated_norm(c["x"].data_ptr(), C, c["branch"].data_ptr(), C, p["gate"], C, p["scale"], C, p["shift"],
                                              C, 0, 1, B * S, C, S, EPS, 1, c[over].data_ptr(), y.data_ptr(), stats.data_ptr(),
                                              None, None, None, None, st) == 0
            assert torch.equal(c[over], r.sum) and torch.equal(y, r.output) and torch.equal(stats, r.stats)
        for over in ("dy", "dsum"):
            c = {n: v.clone() for n, v in t.items()}
            db = torch.empty_like(r.output)
            assert L.reels_hip_modulated_norm_bwd(c["dy"].data_ptr(), r.sum.data_ptr(), None, c["dsum"].data_ptr(), None, None,
                                                  p["gate"], C, p["scale"], C, r.stats.data_ptr(), 0, 1, B * S, C, S, 1,
                                                  c[over].data_ptr(), db.data_ptr(), None, None, None, None, 0, st) == 0
            assert torch.equal(c[over], want.x) and torch.equal(db, want.branch)


def test_many_rows(dev):
    """Groups whose sums run over many workgroups, and many small groups."""
    for B, S, C, kind in [(1, 5000, 130, "sample"), (3, 1111, 515, "sample"),
                          (700, 3, 64, "sample"), (700, 2, 64, "all")]:
        t, m = make(B, S, C, "f32", "f32", kind)
        r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
        g = modulated_norm_backward(t["dy"], r.sum, r.stats, m["scale"], t["branch"], m["gate"], t["dsum"])
        check_backward(g, t, r.sum.double(), t["branch"].double(), r.stats, m["gate"], m["scale"], t["dsum"], True, B, S)


@pytest.mark.parametrize("compress", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [6, 24, 96, 128, 130, 256, 300, 515, 1000, 1536, 5120, 5125, 8200, 16384])
def test_many_rows_of_each_form(dev, C, dtype, compress):
    """Several rows one after the other in every wave or workgroup, in two groups."""
    B, S = 2, 2500 if C < 5000 else 1100
    t, m = make(B, S, C, dtype, "f32", "sample")
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], EPS, True, compress)
    check_forward(r, t["x"], t["branch"], m["gate"], m["scale"], m["shift"], True, B)
    s, b = (r.kept.sum, r.kept.branch) if compress else (r.sum, t["branch"])
    sd, bd = (v.restore(torch.float32).double() if compress else v.double() for v in (s, b))
    g = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], b, m["gate"], t["dsum"])
    check_backward(g, t, sd, bd, r.stats, m["gate"], m["scale"], t["dsum"], True, B, S)


def test_empty(dev):
    for shape in ((0, 5, 40), (3, 0, 40), (0, 40)):
        x = torch.empty(shape, device=dev)
        mod = [torch.randn(40, device=dev) for _ in range(3)]
        r = modulated_norm(x, mod[0], mod[1], x, mod[2], compress=True)
        assert r.output.shape == shape and r.kept.sum.shape == shape
        assert modulated_norm_quantized(x, mod[0], mod[1]).output.shape == (0, 40)
        g = modulated_norm_backward(x, r.sum, r.stats, mod[0], x, mod[2])
        assert g.x.shape == shape and not g.scale.any() and not g.shift.any() and not g.gate.any()
    x = torch.empty(3, 0, 40, device=dev)
    g = modulated_norm_backward(x, x, torch.empty(3, 0, 3, device=dev), torch.randn(3, 40, device=dev))
    assert g.scale.shape == (3, 40) and not g.scale.any() and not g.shift.any()


def test_autograd(dev):
    """Against torch's own gradients of the formula in 64 bits."""
    for kind, compress in (("sample", False), ("token", False), ("all", True)):
        t, m = make(2, 6, 100, "f32", "f32", kind, seed=3)
        leaves = [t["x"], m["scale"], m["shift"], t["branch"], m["gate"]]
        leaves = [v.clone().requires_grad_() for v in leaves]
        y, s = ModulatedNormFunction.apply(*leaves, EPS, True, compress)
        grads = torch.autograd.grad((y, s), leaves, (t["dy"], t["dsum"]))
        wide = [v.detach().double().requires_grad_() for v in leaves]
        sd = wide[0] + rows(wide[4], 2) * wide[3]
        c = sd - sd.mean(-1, keepdim=True)
        yd = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * (1 + rows(wide[1], 2)) + rows(wide[2], 2)
        want = torch.autograd.grad((yd, sd), wide, (t["dy"].double(), t["dsum"].double()))
        # f32, or a backward from 7 bits: a step of the block's largest is 2^-6 of it at most
        tol = 2.0 ** -5 if compress else 1e-5
        for a, b in zip(grads, want):
            assert a.shape == b.shape
            assert float((a.double() - b).norm() / b.norm()) < tol
        only = torch.autograd.grad(ModulatedNormFunction.apply(*leaves, EPS, True, compress)[1], leaves, t["dsum"])
        assert torch.equal(only[0], t["dsum"]) and not only[1].any() and not only[2].any()
    x = t["x"].clone().requires_grad_()
    y = ModulatedNormFunction.apply(x, None, None, None, None)
    torch.autograd.grad(y.sum(), x)
    with pytest.raises(RuntimeError):
        (d,) = torch.autograd.grad(ModulatedNormFunction.apply(x, None, None, None, None).sum(), x, create_graph=True)
        torch.autograd.grad(d.sum(), x)


def test_differences(dev):
    """The gradient along a direction against differences of the forward."""
    t, m = make(2, 5, 70, "f32", "f32", "sample", seed=8)
    names = ("x", "scale", "shift", "branch", "gate")
    at = {**t, **m}
    g = torch.Generator(device=dev).manual_seed(1)
    dirs = {n: torch.randn(at[n].shape, generator=g, device=dev) for n in names}

    def value(h):
        v = {n: at[n] + h * dirs[n] for n in names}
        r = modulated_norm(v["x"], v["scale"], v["shift"], v["branch"], v["gate"])
        return float((r.output.double() * t["dy"].double()).sum() + (r.sum.double() * t["dsum"].double()).sum())
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
    d = modulated_norm_backward(t["dy"], r.sum, r.stats, m["scale"], t["branch"], m["gate"], t["dsum"])
    got = sum(float((getattr(d, n).double() * dirs[n].double()).sum()) for n in names)
    h = 1e-2
    # the error of the fourth-order difference is h^4 times a fifth derivative of order one per term
    want = (8 * (value(h) - value(-h)) - (value(2 * h) - value(-2 * h))) / (12 * h)
    assert abs(got - want) < 2e-3 * max(1.0, abs(want)), (got, want)


def test_other_stream_and_graph(dev):
    t, m = make(2, 300, 1000, "bf16", "f32", "sample")

    def step():
        r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], compress=True)
        g = modulated_norm_backward(t["dy"], r.kept.sum, r.stats, m["scale"], r.kept.branch, m["gate"], t["dsum"])
        q = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
        return [r.output, r.sum, q.output.dequantize()] + list(g)
    want = step()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for i in range(3):
        for v in t.values():
            v.copy_(torch.randn_like(v))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_kept_rows_of_another_shape(dev):
    t, m = make(2, 6, 64, "bf16", "f32", "sample")
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], compress=True)
    with pytest.raises(ValueError, match="both"):
        modulated_norm_backward(t["dy"], r.kept.sum, r.stats, m["scale"], t["branch"], m["gate"])
    with pytest.raises(ValueError, match="shape"):
        modulated_norm_backward(t["dy"], CompressedActivations(r.kept.sum.values[:1], r.kept.sum.scales[:1]), r.stats)


def test_gradients_of_an_ungated_branch_are_two_tensors(dev):
    """x and the branch have one gradient; what is done to one leaf's does not reach the other's."""
    t, m = make(2, 6, 64, "bf16", "f32", "sample")
    x, b = t["x"].clone().requires_grad_(), t["branch"].clone().requires_grad_()
    y, s = ModulatedNormFunction.apply(x, m["scale"], m["shift"], b, None)
    torch.autograd.backward((y, s), (t["dy"], t["dsum"]))
    assert torch.equal(x.grad, b.grad)
    keep = b.grad.clone()
    x.grad.zero_()
    assert torch.equal(b.grad, keep)
    both = t["x"].clone().requires_grad_()  # one tensor as x and as the branch
    y, s = ModulatedNormFunction.apply(both, m["scale"], m["shift"], both, m["gate"])
    (d,) = torch.autograd.grad((y, s), both, (t["dy"], t["dsum"]))
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["x"], m["gate"])
    g = modulated_norm_backward(t["dy"], r.sum, r.stats, m["scale"], t["x"], m["gate"], t["dsum"])
    assert torch.equal(d, g.x + g.branch)


def test_rows_without_spread(dev):
    """Equal elements: the shift with a positive eps; 0 / 0 without one."""
    x = torch.full((4, 96), 3.25, device=dev)
    x[2:, 1] = 4.0
    shift = torch.randn(96, device=dev)
    y = modulated_norm(x, torch.zeros(96, device=dev), shift).output
    assert torch.equal(y[0], shift) and torch.isfinite(y).all()
    r = modulated_norm(x, eps=0.0)
    assert torch.isnan(r.output[:2]).all() and torch.isfinite(r.output[2:]).all()
    c = x[2:].double() - x[2:].double().mean(-1, keepdim=True)
    want = c / c.square().mean(-1, keepdim=True).sqrt()
    assert_within(r.output[2:], want, 7 * U * want.abs(), "without eps")


def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the last rows are those of a small call, and so are the sums where all other
    rows' gradients are zero (bound: the roundings of 64 additions in another order)."""
    M, C, tail = 140000, 16384, 40
    assert M * C > 2 ** 31
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(M, C, generator=g, device=dev, dtype=torch.bfloat16)
    b = torch.randn(M, C, generator=g, device=dev, dtype=torch.bfloat16)
    dy = torch.zeros_like(x)
    dy[-tail:] = torch.randn(tail, C, generator=g, device=dev).bfloat16()
    gate, scale, shift = (torch.randn(C, generator=g, device=dev) for _ in range(3))

    def ends(t):
        return t[-tail:]
    r = modulated_norm(x, scale, shift, b, gate, compress=True)
    w = modulated_norm(ends(x), scale, shift, ends(b), gate, compress=True)
    for u, v in ((r.output, w.output), (r.sum, w.sum), (r.stats, w.stats), (r.kept.sum.values, w.kept.sum.values),
                 (r.kept.sum.scales, w.kept.sum.scales), (r.kept.branch.values, w.kept.branch.values)):
        assert torch.equal(ends(u), v)
    for s, sb, ws, wb in ((r.sum, b, w.sum, ends(b)), (r.kept.sum, r.kept.branch, w.kept.sum, w.kept.branch)):
        d = modulated_norm_backward(dy, s, r.stats, scale, sb, gate)
        e = modulated_norm_backward(ends(dy), ws, w.stats, scale, wb, gate)
        assert torch.equal(ends(d.x), e.x) and torch.equal(ends(d.branch), e.branch) and not d.x[:-tail].any()
        n = (w.sum.double() - (w.stats[:, :1] + w.stats[:, 1:2]).double()) * w.stats[:, 2:].double()
        for name, mag in (("shift", ends(dy).double().abs()), ("scale", ends(dy).double().abs() * (n.abs() + 0.1)),
                          ("gate", (e.x.double().abs() + 1e-2) * (ends(b).double().abs() + 0.1))):
            assert_within(getattr(d, name), getattr(e, name).double(), 128 * U * mag.sum(0), name)
    q = modulated_norm_quantized(x, scale, shift, b, gate)
    p = modulated_norm_quantized(ends(x), scale, shift, ends(b), gate)
    assert torch.equal(ends(q.output.codes), p.output.codes) and torch.equal(ends(q.output.block_scales()), p.output.block_scales())


@pytest.mark.parametrize("dtype,B,S,C", [("bf16", 2, 40, 24), ("f32", 2, 40, 200), ("f16", 2, 40, 512), ("f32", 2, 300, 700),
                                         ("bf16", 2, 300, 700), ("f32", 2, 1400, 700), ("bf16", 2, 1500, 1536), ("f16", 2, 700, 5125),
                                         ("bf16", 2, 400, 9001), ("f32", 2, 400, 9001), ("f32", 2, 300, 16384)])
def test_sum_over_the_inputs_of_each_form(dev, dtype, B, S, C):
    """The sum over x or the branch where a row has 16 lanes, a wave or a workgroup, in every row that a workgroup
    takes one after the other: the bits of a call with a sum of its own."""
    from reels_amd import _lib
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    t, m = make(B, S, C, dtype, "f32", "sample")
    t["x"][..., 0] += 40  # an element far from the others: its row's pivot
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], compress=True)
    q = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"]).output
    p = {n: v.data_ptr() for n, v in m.items()}
    for over in ("x", "branch"):
        for mode in ("rows", "kept", "4 bits"):
            c = {n: t[n].clone() for n in ("x", "branch")}
            args = (c["x"].data_ptr(), C, c["branch"].data_ptr(), C, p["gate"], C, p["scale"], C, p["shift"], C, 0, code, B * S, C,
                    S, EPS, 1, c[over].data_ptr())
            if mode == "4 bits":
                codes, scales = torch.empty_like(q.codes), torch.empty_like(q.scales)
                assert L.reels_hip_modulated_norm_mx4(*args, codes.data_ptr(), scales.data_ptr(), st) == 0
                got, want = (codes,), (q.codes,)
            else:
                y, stats = torch.empty_like(r.output), torch.empty_like(r.stats)
                k = [torch.empty_like(v) for v in (r.kept.sum.values, r.kept.sum.scales, r.kept.branch.values, r.kept.branch.scales)]
                kept = [v.data_ptr() if mode == "kept" else None for v in k]
                assert L.reels_hip_modulated_norm(*args, y.data_ptr(), stats.data_ptr(), *kept, st) == 0
                got, want = (y, stats), (r.output, r.stats)
                if mode == "kept":
                    got, want = got + tuple(k), want + (r.kept.sum.values, r.kept.sum.scales, r.kept.branch.values, r.kept.branch.scales)
            assert torch.equal(c[over], r.sum), (over, mode)
            assert all(torch.equal(u, v) for u, v in zip(got, want)), (over, mode)


def test_modulations_of_one_kind_in_two_shapes(dev):
    """scale [B, C] beside shift and gate [B, 1, C], and [1, C] beside [C]: each gradient has its own leaf's shape."""
    for shape, a, b in (((2, 6, 64), (2, 64), (2, 1, 64)), ((2, 6, 64), (2, 1, 64), (2, 64)), ((7, 64), (64,), (1, 64)),
                        ((7, 64), (1, 64), (64,))):
        x, br, dy = (torch.randn(shape, device=dev) for _ in range(3))
        scale, shift, gate = torch.randn(a, device=dev), torch.randn(b, device=dev), torch.randn(b, device=dev)

        def grads(*mods):
            leaves = [t.clone().requires_grad_() for t in mods]
            y, _ = ModulatedNormFunction.apply(x, leaves[0], leaves[1], br, leaves[2])
            return torch.autograd.grad(y, leaves, dy)
        got, want = grads(scale, shift, gate), grads(scale, shift.view(a), gate.view(a))
        for u, v, like in zip(got, want, (scale, shift, gate)):
            assert u.shape == like.shape and torch.equal(u.flatten(), v.flatten())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,C", [(5, 100), (5, 200), (3, 300), (2100, 700), (4, 700), (3, 1536), (3, 5125), (3, 9001)])
def test_rows_at_the_ends_of_the_range(dev, S, C, dtype):
    """Elements whose difference from the mean passes the f32 range: n stays at most sqrt(C), and so do y and the
    gradients. rstd is subnormal here: its half step is up to 2^-22 of it."""
    t, m = make(1, S, C, dtype, "f32", "sample")
    top = torch.finfo(DT[dtype]).max
    x = torch.where(torch.rand(1, S, C, device=dev) < 0.7, -0.98 * top, 0.98 * top).to(DT[dtype])
    x[..., 0], x[..., C - 1] = top, -top
    assert bool(((x.double() - x.double().mean(-1, keepdim=True)).abs().amax(-1) > 2.0 ** 128).all())
    for compress in (False, True):
        r = modulated_norm(x, m["scale"], m["shift"], compress=compress)
        sd, mean, rstd = unit(x, True)
        st = r.stats.double()
        assert bool(((st[..., 0] + st[..., 1] - mean[..., 0]).abs() <= 2.0 ** -40 * top).all())
        assert_within(r.stats[..., 2], rstd[..., 0], U * rstd[..., 0], "rstd")
        n, up = (sd - mean) * rstd, 1.0 + m["scale"][:, None].double()
        y = n * up + m["shift"][:, None].double()
        assert_within(r.output, y, 7 * U * (n * up).abs() + U * y.abs(), "y")
        s = r.kept.sum if compress else r.sum
        sd = blocks8(x.double().reshape(-1, C))[2].reshape(1, S, C) if compress else sd
        g = modulated_norm_backward(t["dy"], s, r.stats, m["scale"])
        check_backward(g, t, sd, None, r.stats, None, m["scale"], None, True, 1, S)
        few = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], want_modulation=False)
        assert torch.equal(few.x, g.x)
    q = modulated_norm_quantized(x, m["scale"], m["shift"]).output
    assert torch.isfinite(q.dequantize(torch.float32)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,C", [(5, 6), (5, 100), (5, 200), (3, 300), (2100, 700), (4, 700), (3, 1536), (3, 5125), (3, 9001)])
def test_rows_at_the_ends_of_the_range(dev, S, C, dtype):
    """Elements whose difference from the mean passes the f32 range: n stays at most sqrt(C). Bounds (u = 2^-24, m =
    |mean| rstd): rstd is subnormal, so off by e = 2^-150 / rstd of it, which n takes over; the mean is taken off as a
    product with one rounding, m u; the rest of y as above. In d that error of n enters the mean of g n and n times
    that mean; the backward starts from the stored rstd, so e drops out. dscale: m u of the sum of |dy|."""
    t, m = make(1, S, C, dtype, "f32", "sample")
    top = torch.finfo(DT[dtype]).max
    g = torch.Generator(device=dev).manual_seed(C)
    x = torch.where(torch.rand(1, S, C, generator=g, device=dev) < 0.7, -0.98 * top, 0.98 * top).to(DT[dtype])
    x[..., 0], x[..., 1:5], x[..., C - 1] = top, -0.98 * top, -top
    assert bool(((x.double() - x.double().mean(-1, keepdim=True)).abs().amax(-1) > 2.0 ** 128).all())
    up, dy = 1.0 + m["scale"][:, None].double(), t["dy"].double()
    for compress in (False, True):
        r = modulated_norm(x, m["scale"], m["shift"], compress=compress)
        sd, mean, rstd = unit(x, True)
        st = r.stats.double()
        assert bool(((st[..., 0] + st[..., 1] - mean[..., 0]).abs() <= 2.0 ** -40 * top).all())
        assert_within(r.stats[..., 2], rstd[..., 0], U * rstd[..., 0], "rstd")
        n, far = (sd - mean) * rstd, U * (mean * rstd).abs()
        y = n * up + m["shift"][:, None].double()
        assert_within(r.output, y, ((7 * U + 2.0 ** -150 / rstd) * n.abs() + far) * up.abs() + U * y.abs(), "y")
        s = r.kept.sum if compress else r.sum
        sd = blocks8(x.double().reshape(-1, C))[2].reshape(1, S, C) if compress else sd
        d = modulated_norm_backward(t["dy"], s, r.stats, m["scale"])
        rs, n = st[..., 2:], (sd - (st[..., 0] + st[..., 1])[..., None]) * st[..., 2:]
        gd = dy * up
        m1, a0, a1 = ((v).mean(-1, keepdim=True) for v in (gd * n, gd.abs(), (gd * n).abs()))
        slack = rs * U * (8 * gd.abs() + 16 * a0 + 28 * n.abs() * a1) + 1.1 * rs * far * (n.abs() * a0 + m1.abs())
        assert_within(d.x, rs * (gd - gd.mean(-1, keepdim=True) - n * m1), slack, "dx")
        deep = (100 + S / 64) * U
        assert_within(d.scale, (dy * n).sum(1), (deep * (dy * n).abs() + 1.1 * far * dy.abs()).sum(1), "dscale")
        assert_within(d.shift, dy.sum(1), (deep * dy.abs()).sum(1), "dshift")
        few = modulated_norm_backward(t["dy"], s, r.stats, m["scale"], want_modulation=False)
        assert torch.equal(few.x, d.x)
    q = modulated_norm_quantized(x, m["scale"], m["shift"]).output
    assert torch.isfinite(q.dequantize(torch.float32)).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("S,C", [(14000, 24), (14000, 130), (14000, 256), (3001, 300), (3001, 700), (1001, 1536), (401, 5125),
                                 (301, 9001), (201, 16384)])
def test_rows_one_after_the_other(dev, S, C, dtype):
    """More rows than the forward's 16-lane groups, waves or workgroups, in three groups of rows: every one walks on
    into another group's modulations, with its rows as they are, kept and in 4 bits."""
    B = 3
    t, m = make(B, S, C, dtype, "f32", "sample")
    r = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
    check_forward(r, t["x"], t["branch"], m["gate"], m["scale"], m["shift"], True, B)
    k = modulated_norm(t["x"], m["scale"], m["shift"], t["branch"], m["gate"], compress=True)
    assert torch.equal(k.output, r.output) and torch.equal(k.sum, r.sum) and torch.equal(k.stats, r.stats)
    for kept, of in ((k.kept.sum, r.sum), (k.kept.branch, t["branch"])):
        q, sc, _ = blocks8(of.double().reshape(-1, C))
        assert torch.equal(kept.values.reshape(-1, C), q) and torch.equal(kept.scales.reshape(B * S, -1), sc)
    q = modulated_norm_quantized(t["x"], m["scale"], m["shift"], t["branch"], m["gate"])
    assert torch.equal(q.sum, r.sum)
    codes, scales = nibbles(q.output).view(B, S, C), q.output.block_scales().view(B, S, -1)
    for b in range(B):
        # each sample by the definition, 1000 rows at a time; a value within 2^-45 of a border may take either side
        for i in range(0, S, 1000):
            sd, mean, rstd = unit(r.sum[b, i:i + 1000], True)
            part, shift = (sd - mean) * rstd * (1.0 + m["scale"][b].double()), m["shift"][b].double()
            y, mag = part + shift, part.abs() + shift.abs()
            c, sc, _ = blocks4(y.float().double())
            near, far = torch.zeros_like(c, dtype=torch.bool), torch.zeros_like(sc, dtype=torch.bool)
            for f in (-2.0 ** -45, 2.0 ** -45):
                cf, sf, _ = blocks4((y + f * mag).float().double())
                far |= sf != sc
                near |= (cf != c) | far.repeat_interleave(32, 1)[:, :C]
            assert not bool(((codes[b, i:i + 1000] != c) & ~near).any())
            assert not bool(((scales[b, i:i + 1000] != sc) & ~far).any())
            assert float(near.float().mean()) < 0.01


@pytest.mark.parametrize("compress", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [7, 300, 1536, 9001])
def test_gradient_of_the_sum_alone(dev, C, dtype, compress):
    """Where only the sum is used its gradient reaches x, the branch and the gate as it is, also in rows whose sum or
    spread is not finite."""
    t, m = make(2, 9, C, dtype, "f32", "sample")
    t["x"][0, 3, 2], t["x"][1, 5, C - 1], t["x"][1, 7] = float("nan"), float("inf"), 2.0
    t["branch"][1, 7] = 0.0
    leaves = [v.clone().requires_grad_() for v in (t["x"], m["scale"], m["shift"], t["branch"], m["gate"])]
    _, s = ModulatedNormFunction.apply(*leaves, 0.0, True, compress)
    dx, dscale, dshift, db, dgate = torch.autograd.grad(s, leaves, t["dsum"])
    assert torch.equal(dx, t["dsum"]) and not dscale.any() and not dshift.any()
    # one product: rounded once to the type, or to f32 before that (binary16 has an instruction that does it at once)
    want = t["dsum"].double() * m["gate"][:, None].double()
    assert_within(db, want, U * want.abs(), "dbranch")
    b = blocks8(t["branch"].double().reshape(-1, C))[2].view(2, 9, C).to(DT[dtype]) if compress else t["branch"]
    each = t["dsum"].double() * b.double()
    assert_within(dgate, each.sum(1), (100 * U * each.abs()).sum(1), "dgate")
