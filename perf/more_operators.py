"""Performance cases of a transformer block in fewer bits: the modulated norm with the gated residual
before it and its backward, the same norm with its rows in 4 bits, rows in microscaled 4 bits and
their product, and the GELU that keeps its input in 8 bits for its backward.

``listed()`` names the work that a block of the video transformer hands to them, ``draw(rng)`` gives
more cases over the same ranges. A case is a dict of plain values; ``prepare`` makes what a program
holds before the call, ``run`` is one pass (with ``own`` the framework's calls, otherwise the same in
elementary torch operations) and ``exact`` the result in 64 bits from the definitions.

Microscaled blocks are 32 neighbours of a row with one power of two as their scale: the exponent of
the block's largest magnitude after it is rounded to the format's significand (2 bits for the 4-bit
values 0, 0.5, 1, 1.5, 2, 3, 4, 6; 7 bits for the 8-bit codes), so that nothing saturates.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda"
_EPS = 1e-6
_BLOCK = 32


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    return [
        # one short clip whose tokens each have a noise level, so a modulation of their own, in
        # Float32 compute at an odd width, root-mean-square norm: forward and backward
        dict(name="norm_tokens_f32", op="norm", B=1, S=257, C=1001, dtype="f32", mtype="f32",
             per_token=True, center=False, kept=False),
        # two samples of one latent frame in the reference's compute precision, the backward from
        # 8-bit activations: forward and backward
        dict(name="norm_frame_kept", op="norm", B=2, S=1560, C=1536, dtype="f16", mtype="f32",
             per_token=False, center=True, kept=True),
        # between two sublayers of the large video model at full clip length: forward and backward
        dict(name="norm_video", op="norm", B=1, S=32760, C=5120, dtype="bf16", mtype="f32",
             per_token=False, center=True, kept=False),
        # one conditioning row on its way into a 4-bit product: the smallest call
        dict(name="norm_i4_row", op="norm_i4", B=1, S=1, C=5120, dtype="bf16", mtype="bf16",
             per_token=False, center=True),
        # the same norm before a 4-bit product of the large video model at full clip length
        dict(name="norm_i4_video", op="norm_i4", B=1, S=32760, C=5120, dtype="bf16", mtype="f32",
             per_token=False, center=True),
        # an odd weight matrix packed into 4 bits
        dict(name="rows_ragged", op="rows", M=3001, K=1001, dtype="f32"),
        # the hidden rows of the large model's feed-forward at full clip length
        dict(name="rows_video", op="rows", M=32760, K=13824, dtype="bf16"),
        # one row through the first feed-forward projection with its GELU
        dict(name="product_row", op="product", M=1, K=5120, N=13824, dtype="bf16", bias=True,
             activation=True, residual=False),
        # a layer whose widths are no multiples of the tiles, a few hundred tokens, f32 output
        dict(name="product_ragged", op="product", M=777, K=1000, N=3001, dtype="f32", bias=True,
             activation=False, residual=True),
        # the second feed-forward projection of the large video model at full clip length, bias and
        # residual added: the largest call
        dict(name="product_video", op="product", M=32760, K=13824, N=5120, dtype="bf16", bias=True,
             activation=False, residual=True),
        # the text encoder's feed-forward activation for a short prompt, forward and backward
        dict(name="gelu_prompt", op="gelu", M=77, C=10240, dtype="f16"),
        # the large video model's feed-forward activation at full clip length, forward and backward
        dict(name="gelu_video", op="gelu", M=32760, C=13824, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_WIDTHS = [256, 512, 768, 1024, 1536, 2048, 2560, 4096, 5120, 8960, 10240, 13824]


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "norm_i4", "rows", "product", "product", "gelu"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_i4"):
        C = rng.choice(_WIDTHS) if rng.random() < 0.5 else _log(rng, 8, 13824)
        B = rng.choice([1, 1, 2, 3])
        per_token = rng.random() < 0.25
        # at most the elements of the large listed case; modulations of each token are as many again
        most = 32760 * 5120 * 2 // (C * B * _SIZE[dtype] * (4 if per_token else 1))
        case = dict(op=op, B=B, S=_log(rng, 1, max(1, min(65520, most))), C=C, dtype=dtype,
                    mtype=rng.choice([dtype, "f32"]), per_token=per_token,
                    center=rng.random() < 0.7)
        return dict(case, kept=rng.random() < 0.5) if op == "norm" else case
    if op == "product":
        K = rng.choice(_WIDTHS) if rng.random() < 0.6 else _log(rng, 1, 5120)
        N = rng.choice(_WIDTHS) if rng.random() < 0.6 else _log(rng, 1, 5120)
        most = min(32760, int(2e12 / (K * N)))
        return dict(op="product", M=_log(rng, 1, most), K=K, N=N, dtype=dtype,
                    bias=rng.random() < 0.6, activation=rng.random() < 0.4,
                    residual=rng.random() < 0.4)
    C = rng.choice(_WIDTHS) if rng.random() < 0.5 else _log(rng, 1, 13824)
    most = max(1, min(65520, 32760 * 13824 * 2 // (C * _SIZE[dtype])))
    if op == "rows":
        return dict(op="rows", M=_log(rng, 1, most), K=C, dtype=dtype)
    return dict(op="gelu", M=_log(rng, 1, most), C=C, dtype=dtype)


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _randn(g, shape, sigma, dtype):
    return (torch.randn(shape, generator=g, device=_DEV) * sigma).to(dtype)


def _rows_of(g, M, K, dtype, sigma):
    """Rows as they reach a linear: normal values, with a few channels that are much larger."""
    x = torch.randn((M, K), generator=g, device=_DEV) * sigma
    x *= 1.0 + 15.0 * (torch.rand((K,), generator=g, device=_DEV) < 0.005)
    return x.to(dtype)


def _packed(x):
    """Rows in microscaled 4 bits as a program keeps them: codes [M][K / 2] of K padded to a multiple
    of 256, the even column in the low half of a byte; a scale's exponent + 127 for each block; and
    those bytes again in the order in which the matrix cores take them, tiles of 64 rows x 8 blocks:
    [tile of rows][tile of blocks][block % 2][row % 32][block / 2][row / 32]."""
    M, K = x.shape
    Kp = -(-K // 256) * 256
    values, e = _round4(torch.nn.functional.pad(x.float(), (0, Kp - K)))
    at = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=_DEV)
    codes = torch.bucketize(values.abs(), at).to(torch.uint8) + 8 * torch.signbit(values).to(torch.uint8)
    codes = codes[:, 0::2] + 16 * codes[:, 1::2]
    scales = (e + 127).to(torch.uint8)
    tiles = torch.nn.functional.pad(scales, (0, 0, 0, -M % 64))
    tiles = tiles.view(-1, 2, 32, Kp // 256, 4, 2).permute(0, 3, 5, 2, 4, 1).contiguous()
    return codes.contiguous(), scales, tiles.view(-1, Kp // 256, 512)


def _inputs(case, seed):
    g = _gen(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    st = dict(case=case)
    if op in ("norm", "norm_i4"):
        B, S, C = case["B"], case["S"], case["C"]
        mods = (B, S, C) if case["per_token"] else (B, C)
        # residual stream with a mean of its own in each channel
        st["x"] = (torch.randn((B, S, C), generator=g, device=_DEV) * 1.5
                   + torch.randn((C,), generator=g, device=_DEV)).to(dt)
        st["branch"] = _randn(g, (B, S, C), 1.0, dt)
        for name, sigma in (("gate", 0.5), ("scale", 0.3), ("shift", 0.3)):
            st[name] = _randn(g, mods, sigma, _DT[case["mtype"]])
        if op == "norm":
            st["dy"] = _randn(g, (B, S, C), 1.0, dt)
            st["dsum"] = _randn(g, (B, S, C), 1.0, dt)
    elif op == "rows":
        st["x"] = _rows_of(g, case["M"], case["K"], dt, 1.0)
    elif op == "product":
        st["x"] = _packed(_rows_of(g, case["M"], case["K"], torch.bfloat16, 1.0))
        st["w"] = _packed(_randn(g, (case["N"], case["K"]), 0.02, torch.bfloat16))
        st["bias"] = _randn(g, (case["N"],), 0.1, dt) if case["bias"] else None
        st["residual"] = _randn(g, (case["M"], case["N"]), 1.0, dt) if case["residual"] else None
    else:
        st["x"] = _rows_of(g, case["M"], case["C"], dt, 1.0)
        st["dy"] = _randn(g, (case["M"], case["C"]), 1.0, dt)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---- microscaled blocks in elementary operations ---------------------------------------------------
def _blocks(x):
    M, K = x.shape
    return torch.nn.functional.pad(x, (0, -K % _BLOCK)).view(M, -1, _BLOCK)


def _exponent(x, bits):
    """The exponent of each block's largest magnitude, rounded to so many significant bits."""
    m, e = torch.frexp(x.abs().amax(dim=2))  # magnitude = m 2^e, m in [0.5, 1)
    return e - 1 + (m >= 1.0 - 2.0 ** -(bits + 1)).int()


def _round4(x):
    """(values, exponents) of rows in 4 bits: whole multiples of a step that grows with the value."""
    v = _blocks(x)
    e = (_exponent(v, 2) - 2).clamp_min(-127)
    unit = torch.exp2(e[..., None].float())
    a = v / unit
    size = a.abs()
    step = 0.5 * (1.0 + (size >= 2.0) + 2.0 * (size >= 4.0))
    return (torch.round(a / step) * step).flatten(1)[:, :x.shape[1]], e


def _values4(x):
    """The values that rows stand for in 4 bits."""
    v, e = _round4(x)
    return (_blocks(v) * torch.exp2(e[..., None].float())).flatten(1)[:, :x.shape[1]]


def _values8(x):
    """The values that rows stand for in 8 bits."""
    v = _blocks(x.float())
    e = _exponent(v, 7).clamp_min(-127)
    unit = torch.exp2((e[..., None] - 6).float())
    return (torch.round(v / unit) * unit).flatten(1)[:, :x.shape[1]]


def _unpacked(rows, K):
    """f32 values of a packed operand."""
    codes, scales, _ = rows
    at = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=_DEV)
    at = torch.cat((at, -at))
    v = at[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1).int()]
    unit = torch.exp2(scales.float() - 127.0)
    return (v.view(v.shape[0], -1, _BLOCK) * unit[..., None]).flatten(1)[:, :K]


# ---- one pass ------------------------------------------------------------------------------------
def _each(st, name):
    """A modulation against rows: one for each token, or one for each sample."""
    m = st[name].float()
    return m if st["case"]["per_token"] else m[:, None, :]


def _plain_normed(st, dt):
    """The stored sum, its normed rows and 1 / their size."""
    x = st["x"]
    s = (x.float() + _each(st, "gate") * st["branch"].float()).to(x.dtype)
    return (s,) + _plain_unit(s, dt, st["case"]["center"])


def _plain_unit(s, dt, center):
    n = s.to(dt)
    if center:
        n = n - n.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((n * n).mean(dim=-1, keepdim=True) + _EPS)
    return n * rstd, rstd


def _plain_norm(st):
    case, dt = st["case"], st["x"].dtype
    s, n, rstd = _plain_normed(st, torch.float32)
    up = 1.0 + _each(st, "scale")
    y = n * up + _each(st, "shift")
    dy, branch = st["dy"].float(), st["branch"].float()
    if case["kept"]:  # the backward has the sum and the branch in 8 bits
        C = case["C"]
        kept = _values8(s.view(-1, C)).view(s.shape)
        branch = _values8(st["branch"].view(-1, C)).view(s.shape)
        mean = s.float().mean(dim=-1, keepdim=True) if case["center"] else 0.0
        n = (kept - mean) * rstd
    g = dy * up
    d = g - n * (g * n).mean(dim=-1, keepdim=True)
    if case["center"]:
        d = d - g.mean(dim=-1, keepdim=True)
    d = rstd * d + st["dsum"].float()
    grads = (d * branch, dy * n, dy)
    if not case["per_token"]:
        grads = tuple(t.sum(dim=1) for t in grads)
    return (y.to(dt), s, d.to(dt), (d * _each(st, "gate")).to(dt)) + grads


def _plain_norm_i4(st):
    # in 64 bits: a code next to the border of two values
    s, n, _ = _plain_normed(st, torch.float64)
    y = n * (1.0 + _each(st, "scale").double()) + _each(st, "shift").double()
    return _values4(y.float().view(-1, y.shape[-1])).to(s.dtype), s


def _gelu(x):
    k = math.sqrt(2.0 / math.pi)
    return 0.5 * x * (1.0 + torch.tanh(k * (x + 0.044715 * x * x * x)))


def _plain_product(st):
    case = st["case"]
    y = torch.matmul(_unpacked(st["x"], case["K"]), _unpacked(st["w"], case["K"]).t())
    if case["bias"]:
        y = y + st["bias"].float()
    if case["activation"]:
        y = _gelu(y)
    if case["residual"]:
        y = y + st["residual"].float()
    return y.to(_DT[case["dtype"]])


def _plain_gelu(st):
    x, dt = st["x"].float(), st["x"].dtype
    kept = _values8(x)
    k, a = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(k * (kept + a * kept * kept * kept))
    slope = 0.5 * (1.0 + t) + 0.5 * kept * (1.0 - t * t) * k * (1.0 + 3.0 * a * kept * kept)
    return _gelu(x).to(dt), kept.to(dt), (st["dy"].float() * slope).to(dt)


def _own_norm(ra, st):
    case = st["case"]
    r = ra.modulated_norm(st["x"], st["scale"], st["shift"], branch=st["branch"], gate=st["gate"],
                          eps=_EPS, center=case["center"], compress=case["kept"])
    s, branch = (r.kept.sum, r.kept.branch) if case["kept"] else (r.sum, st["branch"])
    g = ra.modulated_norm_backward(st["dy"], s, r.stats, st["scale"], branch=branch,
                                   gate=st["gate"], dsum=st["dsum"], center=case["center"])
    return r.output, r.sum, g.x, g.branch, g.gate, g.scale, g.shift


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        import reels_amd as ra
        dt = _DT[case["dtype"]]
        if op == "norm":
            return _own_norm(ra, st)
        if op == "norm_i4":
            r = ra.modulated_norm_quantized(st["x"], st["scale"], st["shift"], branch=st["branch"],
                                            gate=st["gate"], eps=_EPS, center=case["center"])
            return r.output.dequantize(), r.sum
        if op == "rows":
            return ra.quantize_microscaled(st["x"]).dequantize()
        if op == "product":
            x, w = (ra.MicroscaledMatrix(st[n][0], st[n][2], (case[d], case["K"]), dt)
                    for n, d in (("x", "M"), ("w", "N")))
            return ra.microscaled_linear(x, w, bias=st["bias"], residual=st["residual"],
                                         activation="gelu_tanh" if case["activation"] else None)
        y, kept = ra.gelu_tanh_compressed(st["x"])
        return y, kept.restore(), ra.gelu_tanh_backward(kept, st["dy"])
    if op == "rows":
        return _values4(st["x"].float()).to(st["x"].dtype)
    return {"norm": _plain_norm, "norm_i4": _plain_norm_i4, "product": _plain_product,
            "gelu": _plain_gelu}[op](st)


# ---- the work of one pass ------------------------------------------------------------------------
def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op in ("norm", "norm_i4"):
        rows = case["B"] * case["S"]
        n, groups = rows * case["C"], rows if case["per_token"] else case["B"]
        me = _SIZE[case["mtype"]] * groups * case["C"]
        # forward: x and the branch -> the sum (and y)
        if op == "norm_i4":  # the codes and their scales are written and read back as values
            return {"bytes": n * 4 * e + 3 * me + 17 * n // 16, "flops": 12 * n}
        # backward: dy, the sum, the stream's gradient and the branch -> dx and the branch's
        nbytes = 4 * n * e + 3 * me + 4 * n * e + 2 * me + 3 * 4 * groups * case["C"] + 12 * rows
        # the sum and the branch in 8 bits are written once and read once
        nbytes += 4 * 33 * n // 32 if case["kept"] else 2 * n * e
        return {"bytes": nbytes, "flops": 30 * n}
    if op == "product":
        M, K, N = case["M"], case["K"], case["N"]
        out = M * N * e * (2 if case["residual"] else 1) + (N * e if case["bias"] else 0)
        return {"bytes": (M + N) * K * 17 // 32 + out, "flops": 2 * M * N * K}
    if op == "rows":  # the codes and their scales are written and read back as values
        n = case["M"] * case["K"]
        return {"bytes": 2 * n * e + 17 * n // 16, "flops": 4 * n}
    n = case["M"] * case["C"]
    # x -> y and the codes; the codes -> their values; dy and the codes -> dx
    return {"bytes": 5 * n * e + 3 * 33 * n // 32, "flops": 40 * n}


# ---- the same in 64 bits -------------------------------------------------------------------------
def _exact_power(x, nearly_two):
    """2^floor(log2(largest of each block)), doubled where that is at least nearly_two times it."""
    top = x.abs().max(dim=2, keepdim=True).values
    p = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -140))))
    return torch.where(top >= nearly_two * p, 2.0 * p, p)


def _exact_values(x, bits):
    """Rows in 4 or 8 bits in 64-bit arithmetic: by the borders of neighbouring values, or by rounding."""
    v = _blocks(x)
    if bits == 8:
        unit = _exact_power(v, 127.5 / 64.0).clamp_min(2.0 ** -127) / 64.0
        q = v.div_(unit).round_().mul_(unit)
    else:
        unit = (_exact_power(v, 1.75) / 4.0).clamp_min(2.0 ** -127)
        v /= unit
        size, q = v.abs(), torch.zeros_like(v)
        # at a border the value with an even code
        for border, up, step in ((0.25, False, 0.5), (0.75, True, 0.5), (1.25, False, 0.5), (1.75, True, 0.5),
                                 (2.5, False, 1.0), (3.5, True, 1.0), (5.0, False, 2.0)):
            q += step * ((size >= border) if up else (size > border))
        q = torch.copysign(q, v).mul_(unit)
    return q.flatten(1)[:, :x.shape[1]]


def _exact_norm(case, st):
    f64, C = torch.float64, case["C"]
    x, branch = st["x"].to(f64), st["branch"].to(f64)
    shape = (case["B"], case["S"] if case["per_token"] else 1, C)
    gate, scale, shift = (st[n].to(f64).reshape(shape) for n in ("gate", "scale", "shift"))
    # the sum is rounded where it is stored, and the norm is that of the stored values
    s = (x + gate * branch).to(st["x"].dtype).to(f64)
    del x
    mean = s.sum(dim=-1, keepdim=True) / C if case["center"] else torch.zeros_like(s[..., :1])
    size = (((s - mean) ** 2).sum(dim=-1, keepdim=True) / C + _EPS).sqrt()
    unit = (s - mean) / size
    y = torch.addcmul(shift, unit, scale + 1.0)
    if case["op"] == "norm_i4":
        return _exact_values(y.reshape(-1, C), 4), s
    dy = st["dy"].to(f64)
    if case["kept"]:
        unit = (_exact_values(s.reshape(-1, C), 8).reshape(s.shape) - mean) / size
        branch = _exact_values(branch.reshape(-1, C), 8).reshape(s.shape)
    dunit = dy * (scale + 1.0)
    along = (dunit * unit).sum(dim=-1, keepdim=True) / C
    d = (dunit - along * unit) / size
    if case["center"]:
        d -= dunit.sum(dim=-1, keepdim=True) / C / size
    d += st["dsum"].to(f64)
    own_mod = [d * branch, dy * unit, dy]
    if not case["per_token"]:
        own_mod = [t.sum(dim=1) for t in own_mod]
    return (y, s, d, d * gate, *own_mod)


def _exact_product(case, st):
    def values(rows):
        codes, scales, _ = rows
        sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device=_DEV)
        size = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=_DEV)
        v = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device=_DEV)
        for half in (0, 1):
            c = (codes >> (4 * half)).int()
            v[:, half::2] = size[c & 7] * sign[(c >> 3) & 1]
        return v * torch.exp2(scales.double() - 127.0).repeat_interleave(_BLOCK, dim=1)

    y = values(st["x"]) @ values(st["w"]).t()
    if case["bias"]:
        y += st["bias"].to(torch.float64)
    if case["activation"]:
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y.pow(3)))
        y = y.mul_(t.add_(1.0)).mul_(0.5)
    if case["residual"]:
        y += st["residual"].to(torch.float64)
    return y


def _exact_gelu(case, st):
    x = st["x"].to(torch.float64)
    c = math.sqrt(2.0 / math.pi)

    def half(v):  # (1 + tanh z) / 2 and the derivative of z
        return torch.sigmoid(2.0 * c * (v + 0.044715 * v ** 3)), c * (1.0 + 0.134145 * v ** 2)

    y = x * half(x)[0]
    kept = _exact_values(x, 8)
    p, dz = half(kept)
    return y, kept, st["dy"].to(torch.float64) * (p + 2.0 * kept * p * (1.0 - p) * dz)


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rows":
        return _exact_values(st["x"].to(torch.float64), 4)
    return {"norm": _exact_norm, "norm_i4": _exact_norm, "product": _exact_product,
            "gelu": _exact_gelu}[case["op"]](case, st)
