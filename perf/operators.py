"""Performance cases of the operators around the int8 linears and the attention.

``listed()`` names the work that a block of the video transformer, or of its text encoder, hands to
them: RMS norms with the residual's addition and their backward, the same norm with its output as
int8 rows, the product of int8 rows with an int8 weight, rotary positions over time, height and
width, and the clipping of the adapters' gradients by their global norm. ``draw(rng)`` gives more
cases over the same ranges.

A case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is
one pass (with ``own`` the framework's calls, otherwise the same in elementary torch operations) and
``exact`` the result in 64 bits from the definitions.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda"
_EPS = 1e-6
_THETA = 10000.0


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    return [
        # residual addition and norm between two sublayers of the text encoder, one prompt, trained
        # norm weights: forward and backward
        dict(name="norm_prompt", op="norm", M=512, C=4096, dtype="bf16", wtype="bf16",
             residual=True, dweight=True),
        # norm of the queries before the attention of the large video model at full clip length,
        # frozen f32 norm weights (adapters alone are trained): forward and backward
        dict(name="norm_video", op="norm", M=32760, C=5120, dtype="bf16", wtype="f32",
             residual=False, dweight=False),
        # norm per head in Float32 compute at an odd head width: 12 heads of one latent frame
        dict(name="norm_heads_f32", op="norm", M=18720, C=101, dtype="f32", wtype="f32",
             residual=False, dweight=True),
        # one conditioning vector on its way into an int8 product: the smallest call
        dict(name="norm_i8_token", op="norm_i8", M=1, C=5120, dtype="f16", wtype="f16",
             residual=False),
        # residual addition and norm before an int8 product of the video model at full clip length
        dict(name="norm_i8_video", op="norm_i8", M=32760, C=5120, dtype="bf16", wtype="bf16",
             residual=True),
        # one token through the first feed-forward projection with its GELU
        dict(name="product_token", op="product", M=1, K=5120, N=13824, dtype="bf16", bias=True,
             activation=True, residual=False),
        # a layer whose widths are no multiples of the tiles, a few hundred tokens, f32 output
        dict(name="product_ragged", op="product", M=777, K=1000, N=3001, dtype="f32", bias=True,
             activation=False, residual=True),
        # the second feed-forward projection of the large video model at full clip length, bias and
        # the block's residual added: the largest call
        dict(name="product_video", op="product", M=32760, K=13824, N=5120, dtype="bf16", bias=True,
             activation=False, residual=True),
        # queries and keys of one latent frame in the reference's compute precision, forward and
        # backward
        dict(name="rotary_frame", op="rotary", B=1, T=1, H=30, W=52, heads=12, kv_heads=12, D=128,
             dtype="f16", interleaved=True),
        # queries and keys of the large video model at full clip length, forward and backward
        dict(name="rotary_video", op="rotary", B=1, T=21, H=30, W=52, heads=40, kv_heads=40, D=128,
             dtype="bf16", interleaved=True),
        # adapters of rank 3 on the small model's attention, gradients of ragged sizes
        dict(name="clip_small", op="clip", layers=30, K=1536, N=1537, r=3, dtype="f32", norm=0.5),
        # adapters of rank 32 on ten projections of each of 40 blocks (800 tensors)
        dict(name="clip_large", op="clip", layers=400, K=5120, N=5120, r=32, dtype="f32", norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_WIDTHS = [256, 512, 768, 1024, 1536, 2048, 2560, 4096, 5120, 8960, 10240, 13824]


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_i8", "product", "product", "rotary", "rotary", "clip"])
    if op in ("norm", "norm_i8"):
        C = rng.choice(_WIDTHS) if rng.random() < 0.5 else _log(rng, 8, 13824)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        # at most the bytes of the large listed case
        most = max(1, min(65520, 32760 * 5120 * 2 // (C * _SIZE[dtype])))
        case = dict(op=op, M=_log(rng, 1, most), C=C, dtype=dtype,
                    wtype=rng.choice([dtype, "f32"]), residual=rng.random() < 0.5)
        return dict(case, dweight=rng.random() < 0.5) if op == "norm" else case
    if op == "product":
        K = rng.choice(_WIDTHS) if rng.random() < 0.6 else _log(rng, 1, 5120)
        N = rng.choice(_WIDTHS) if rng.random() < 0.6 else _log(rng, 1, 5120)
        most = min(32760, int(2e12 / (K * N)))
        return dict(op="product", M=_log(rng, 1, most), K=K, N=N,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), bias=rng.random() < 0.6,
                    activation=rng.random() < 0.4, residual=rng.random() < 0.4)
    if op == "rotary":
        T, H, W, B = _log(rng, 1, 21), _log(rng, 1, 45), _log(rng, 1, 80), rng.choice([1, 1, 2, 3])
        heads = rng.choice([5, 8, 12, 16, 24, 40])
        kv_heads = heads if rng.random() < 0.7 else rng.choice([1, 2, 4])
        dtype = rng.choice(["bf16", "f16", "f32"])
        D = rng.choice([32, 64, 80, 96, 128, 128, 72, 100])
        # at most the elements of the large listed case
        T = max(1, min(T, 32760 * 2 * 40 * 128 // (B * H * W * (heads + kv_heads) * D)))
        return dict(op="rotary", B=B, T=T, H=H, W=W, heads=heads, kv_heads=kv_heads, D=D,
                    dtype=dtype, interleaved=rng.random() < 0.6)
    K, N = rng.choice(_WIDTHS[:9]), _log(rng, 64, 13824)
    r, dtype = rng.choice([1, 3, 4, 8, 16, 32]), rng.choice(["f32", "f32", "bf16", "f16"])
    return dict(op="clip", layers=_log(rng, 1, max(1, min(300, int(1.2e8 / ((K + N) * r))))), K=K, N=N,
                r=r, dtype=dtype, norm=rng.choice([100.0, 1e6] if dtype == "f16" else [0.1, 1.0, 1e6]))


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _randn(g, shape, sigma, dtype):
    return (torch.randn(shape, generator=g, device=_DEV) * sigma).to(dtype)


def _codes(g, rows, cols, sigma):
    """int8 codes [rows][cols] and scales [rows] of normal values, as packing gives them."""
    w = torch.randn((rows, cols), generator=g, device=_DEV) * sigma
    s = w.abs().amax(dim=1).clamp_min(1e-30) / 127.0
    return torch.round(w / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _axes(D):
    """Pairs of each axis: a third of the pairs for height and for width, the rest for time."""
    third = (D // 2) // 3
    return (D // 2 - 2 * third, third, third)


def _inputs(case, seed):
    g = _gen(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    st = dict(case=case)
    if op in ("norm", "norm_i8"):
        shape = (case["M"], case["C"])
        st["x"] = _randn(g, shape, 1.5, dt)
        st["w"] = (1.0 + _randn(g, (case["C"],), 0.2, torch.float32)).to(_DT[case["wtype"]])
        st["residual"] = _randn(g, shape, 1.0, dt) if case["residual"] else None
        if op == "norm":
            st["dy"] = _randn(g, shape, 1.0, dt)
            # the residual stream's own gradient, which the backward adds
            st["dsum"] = _randn(g, shape, 1.0, dt) if case["residual"] else None
    elif op == "product":
        st["xq"], st["xs"] = _codes(g, case["M"], case["K"], 1.0)
        st["wq"], st["ws"] = _codes(g, case["N"], case["K"], 0.02)
        st["bias"] = _randn(g, (case["N"],), 0.1, dt) if case["bias"] else None
        st["residual"] = _randn(g, (case["M"], case["N"]), 1.0, dt) if case["residual"] else None
    elif op == "rotary":
        n = case["T"] * case["H"] * case["W"]
        q, k = ((case["B"], n, case[h], case["D"]) for h in ("heads", "kv_heads"))
        for name, shape in (("q", q), ("k", k), ("dq", q), ("dk", k)):
            st[name] = _randn(g, shape, 1.0, dt)
        t, h, w = (torch.arange(case[a], device=_DEV, dtype=torch.int32) for a in "THW")
        grid = torch.stack(torch.meshgrid(t, h, w, indexing="ij"), dim=-1).reshape(n, 3)
        # each sequence of a batch starts at a frame of its own
        start = torch.randint(0, 1000, (case["B"], 1, 1), generator=g, device=_DEV, dtype=torch.int32)
        st["positions"] = (grid[None] + start * torch.tensor([1, 0, 0], device=_DEV,
                                                             dtype=torch.int32)).contiguous()
    else:
        shapes = [(case["K"], case["r"]), (case["r"], case["N"])] * case["layers"]
        # binary16 gradients carry a loss scale, and so does the norm they are clipped to
        sigma = 1.0 if dt == torch.float16 else 1e-3
        st["grads"] = [_randn(g, s, sigma, dt) for s in shapes]
        # what the optimizer reads: one buffer that a program keeps, a piece for each tensor
        sizes = [t.numel() for t in st["grads"]]
        st["flat"] = torch.empty(sum(sizes), dtype=dt, device=_DEV)
        st["out"] = [p.view(s) for p, s in zip(st["flat"].split(sizes), shapes)]
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---- one pass ------------------------------------------------------------------------------------
def _gelu(x):
    k = math.sqrt(2.0 / math.pi)
    return 0.5 * x * (1.0 + torch.tanh(k * (x + 0.044715 * x * x * x)))


def _plain_sum(st):
    return st["x"] if st["residual"] is None else (st["x"].float() + st["residual"].float()).to(st["x"].dtype)


def _plain_norm(st):
    case, w = st["case"], st["w"].float()
    s = _plain_sum(st)
    sf = s.float()
    rstd = torch.rsqrt((sf * sf).mean(dim=1, keepdim=True) + _EPS)
    y = sf * rstd * w
    dy = st["dy"].float()
    g = dy * w
    dx = rstd * (g - sf * rstd * rstd * (g * sf).mean(dim=1, keepdim=True))
    if st["dsum"] is not None:
        dx = dx + st["dsum"].float()
    dw = (dy * sf * rstd).sum(dim=0) if case["dweight"] else None
    return y.to(s.dtype), s, dx.to(s.dtype), dw


def _plain_norm_i8(st):
    # in 64 bits: a code next to the border of two whole numbers
    s = _plain_sum(st)
    y = s.double()
    y = y * torch.rsqrt((y * y).mean(dim=1, keepdim=True) + _EPS) * st["w"].double()
    top = y.abs().amax(dim=1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), top / 127.0)
    return (torch.round(y / scale) * scale).to(s.dtype), s


def _plain_product(st):
    case = st["case"]
    y = torch.matmul(st["xq"].float(), st["wq"].float().t()) * st["xs"][:, None] * st["ws"]
    if case["bias"]:
        y = y + st["bias"].float()
    if case["activation"]:
        y = _gelu(y)
    if case["residual"]:
        y = y + st["residual"].float()
    return y.to(_DT[case["dtype"]])


def _plain_rotate(x, cos, sin, interleaved):
    P = cos.shape[-1]
    xf = x.float()
    if interleaved:
        a, b = xf[..., 0::2], xf[..., 1::2]
    else:
        a, b = xf[..., :P], xf[..., P:]
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return y.to(x.dtype)


def _angles(case, positions):
    """[B][S][1][pairs] angles in 64 bits (far positions)."""
    axes = _axes(case["D"])
    freq = [torch.tensor(_THETA, dtype=torch.float64, device=_DEV)
            ** (-torch.arange(n, dtype=torch.float64, device=_DEV) / max(n, 1)) for n in axes]
    p = positions.double()
    return torch.cat([p[..., a:a + 1] * f for a, f in enumerate(freq)], dim=-1)[:, :, None, :]


def _plain_rotary(st):
    case = st["case"]
    ang = _angles(case, st["positions"])
    cos, sin, il = ang.cos().float(), ang.sin().float(), case["interleaved"]
    return (_plain_rotate(st["q"], cos, sin, il), _plain_rotate(st["k"], cos, sin, il),
            _plain_rotate(st["dq"], cos, -sin, il), _plain_rotate(st["dk"], cos, -sin, il))


def _plain_clip(st):
    norm = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt().float()
    factor = (st["case"]["norm"] / (norm + 1e-6)).clamp(max=1.0)
    _ = [o.copy_(g.float() * factor) for g, o in zip(st["grads"], st["out"])]
    return st["flat"], norm


def _values(rows):
    """The values of int8 rows in their type: code times f32 scale, rounded once (dequantize rounds
    the scale to binary16 first where that is the type)."""
    if rows.compute_dtype == torch.float16:
        return rows.dequantize(torch.float32).half()
    return rows.dequantize()


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        import reels_amd as ra
        if op == "norm":
            n = ra.rms_norm(st["x"], st["w"], eps=_EPS, residual=st["residual"])
            g = ra.rms_norm_backward(st["dy"], n.sum, st["w"], n.rstd, dsum=st["dsum"],
                                     want_dweight=case["dweight"])
            return n.output, n.sum, g.x, g.weight
        if op == "norm_i8":
            n = ra.rms_norm_quantized(st["x"], st["w"], eps=_EPS, residual=st["residual"])
            return _values(n.output), n.sum
        if op == "product":
            dt = _DT[case["dtype"]]
            return ra.quantized_linear(ra.QuantizedMatrix(st["xq"], st["xs"], dt),
                                       ra.QuantizedMatrix(st["wq"], st["ws"], dt), bias=st["bias"],
                                       activation="gelu_tanh" if case["activation"] else None,
                                       residual=st["residual"])
        if op == "rotary":
            kw = dict(axes=_axes(case["D"]), theta=_THETA, interleaved=case["interleaved"])
            q, k = ra.rotary_qk(st["q"], st["k"], st["positions"], **kw)
            dq, dk = ra.rotary_qk_backward(st["dq"], st["dk"], st["positions"], **kw)
            return q, k, dq, dk
        norm = ra.clip_gradients(st["grads"], case["norm"], out=st["out"])
        return st["flat"], norm
    return {"norm": _plain_norm, "norm_i8": _plain_norm_i8, "product": _plain_product,
            "rotary": _plain_rotary, "clip": _plain_clip}[op](st)


# ---- the work of one pass ------------------------------------------------------------------------
def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op in ("norm", "norm_i8"):
        n, we = case["M"] * case["C"], _SIZE[case["wtype"]]
        res = 1 if case["residual"] else 0
        # forward: x (and the residual) -> y (and the sum)
        nbytes = n * e * (1 + 2 * res) + case["C"] * we
        if op == "norm_i8":  # the codes are written and read back as values
            return {"bytes": n * (2 + e) + nbytes + 8 * case["M"], "flops": 6 * n}
        # backward: dy, the sum (and the stream's gradient) -> dx, dw
        nbytes += n * e + n * e * (3 + res) + case["C"] * (we + (4 if case["dweight"] else 0)) + 8 * case["M"]
        return {"bytes": nbytes, "flops": 16 * n}
    if op == "product":
        M, K, N = case["M"], case["K"], case["N"]
        out = M * N * e * (2 if case["residual"] else 1) + (N * e if case["bias"] else 0)
        return {"bytes": M * K + N * K + 4 * (M + N) + out, "flops": 2 * M * N * K}
    if op == "rotary":
        n = case["B"] * case["T"] * case["H"] * case["W"]
        x = n * (case["heads"] + case["kv_heads"]) * case["D"]
        return {"bytes": 4 * x * e + 24 * n, "flops": 6 * x}
    n = case["layers"] * (case["K"] + case["N"]) * case["r"]
    return {"bytes": 2 * n * e + 4, "flops": 3 * n}


# ---- the same in 64 bits -------------------------------------------------------------------------
def _exact_norm(case, st):
    f64 = torch.float64
    x, w = st["x"].to(f64), st["w"].to(f64)
    # the sum is rounded where it is stored, and the norm is that of the stored values
    s = x if st["residual"] is None else (x + st["residual"].to(f64)).to(st["x"].dtype).to(f64)
    root = ((s ** 2).sum(dim=1) / case["C"] + _EPS).sqrt()[:, None]
    unit = s / root
    if case["op"] == "norm_i8":
        p = unit * w
        top = p.abs().max(dim=1).values[:, None]
        code = torch.where(top > 0, (p * 127.0 / top.clamp_min(1e-300)).round(), torch.zeros_like(p))
        return code * (top / 127.0), s
    dy = st["dy"].to(f64)
    dunit = dy * w
    # unit = s / |s|: its Jacobian takes off the part along unit
    dx = (dunit - unit * (dunit * unit).sum(dim=1, keepdim=True) / case["C"]) / root
    if st["dsum"] is not None:
        dx += st["dsum"].to(f64)
    return unit * w, s, dx, (dy * unit).sum(dim=0) if case["dweight"] else None


def _exact_product(case, st):
    x = st["xq"].to(torch.float64) * st["xs"].to(torch.float64)[:, None]
    w = st["wq"].to(torch.float64) * st["ws"].to(torch.float64)[:, None]
    y = x @ w.t()
    del x, w
    if case["bias"]:
        y += st["bias"].to(torch.float64)
    if case["activation"]:
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y.pow(3)))
        y = y.mul_(t.add_(1.0)).mul_(0.5)
    if case["residual"]:
        y += st["residual"].to(torch.float64)
    return y


def _exact_rotary(case, st):
    axes, D = _axes(case["D"]), case["D"]
    P = D // 2
    angle = torch.empty(st["positions"].shape[:2] + (P,), dtype=torch.float64, device=_DEV)
    at = 0
    for a, n in enumerate(axes):
        for j in range(n):
            angle[..., at + j] = st["positions"][..., a].to(torch.float64) * math.pow(_THETA, -j / n)
        at += n
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def rotated(x, by):
        x = x.to(torch.float64)
        pairs = (x.unflatten(-1, (P, 2)) if case["interleaved"]
                 else x.unflatten(-1, (2, P)).transpose(-1, -2)).contiguous()
        z = torch.view_as_real(torch.view_as_complex(pairs) * by)
        return z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)

    return (rotated(st["q"], turn), rotated(st["k"], turn), rotated(st["dq"], turn.conj()),
            rotated(st["dk"], turn.conj()))


def _exact_clip(case, st):
    total = torch.zeros((), dtype=torch.float64, device=_DEV)
    for g in st["grads"]:
        total += torch.linalg.vector_norm(g.to(torch.float64)) ** 2
    norm = total.sqrt()
    factor = torch.clamp(case["norm"] / (norm + 1e-6), max=1.0)
    return torch.cat([(g.to(torch.float64) * factor).reshape(-1) for g in st["grads"]]), norm


def exact(case, seed):
    st = _inputs(case, seed)
    return {"norm": _exact_norm, "norm_i8": _exact_norm, "product": _exact_product,
            "rotary": _exact_rotary, "clip": _exact_clip}[case["op"]](case, st)
