"""Microscaled blocks from their definition, in 64 bits: 32 neighbours of a row share a power of two."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exponents(x, bits):
    """floor(log2) of each block's largest magnitude rounded to `bits` significant bits (half up), and
    which blocks hold NaN or infinities. x [M][K] float64."""
    M, K = x.shape
    v = torch.nn.functional.pad(x, (0, -K % 32)).view(M, -1, 32)
    bad = ~torch.isfinite(v).all(dim=2)
    m, e = torch.frexp(v.abs().nan_to_num(0.0, 0.0, 0.0).amax(dim=2))
    e = e.to(torch.int64) - 1
    q = torch.floor(m * 2.0 ** bits + 0.5)   # 2^(bits-1) .. 2^bits
    return v, torch.where(q >= 2.0 ** bits, e + 1, e), bad


def blocks8(x):
    """(codes int8 [M][K], scale bytes [M][blocks], values float64 [M][K]) of a float64 matrix."""
    K = x.shape[1]
    v, e, bad = _exponents(x, 7)
    e = torch.where(v.abs().amax(dim=2) == 0, -127, e).clamp(-127, 127)
    unit = torch.exp2((e[..., None] - 6).double())
    q = torch.where(bad[..., None], 0.0, torch.round(v / unit).clamp(-127, 127))
    values = torch.where(bad[..., None], float("nan"), q * unit)
    return (q.flatten(1)[:, :K].to(torch.int8), torch.where(bad, 255, e + 127).to(torch.uint8),
            values.flatten(1)[:, :K])


def blocks4(x):
    """(codes 0 .. 15 uint8 [M][K], scale bytes, values float64) of a float64 matrix."""
    K = x.shape[1]
    v, e, bad = _exponents(x, 2)
    e = torch.where(v.abs().amax(dim=2) == 0, -127, e - 2).clamp(-127, 125)
    unit = torch.exp2(e[..., None].double())
    a = torch.where(bad[..., None], 0.0, v / unit)
    # the nearest of the grid by distance; of two equally near the one with the even code
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    d = (a.abs()[..., None] - grid).abs() + 1e-9 * (torch.arange(8, device=x.device) % 2)
    far = (a.abs()[..., None] - grid).abs()
    near = far.min(dim=-1, keepdim=True).values
    code = torch.where(far == near, d, float("inf")).argmin(dim=-1)
    sign = torch.signbit(torch.where(bad[..., None], 0.0, v))
    values = torch.where(bad[..., None], float("nan"), torch.where(sign, -1.0, 1.0) * grid[code] * unit)
    return ((code + 8 * sign).flatten(1)[:, :K].to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8),
            values.flatten(1)[:, :K])


def nibbles(q):
    """The codes 0 .. 15 [M][K] of a MicroscaledMatrix."""
    c = torch.stack((q.codes & 15, q.codes >> 4), dim=-1).flatten(1)
    return c[:, :q.shape[1]]


def hard_rows(M, C, dtype, dev, seed=0):
    """Rows whose blocks go over what quantising can meet: ordinary values, ties, borders of a block's
    exponent, tiny and subnormal values, the top of the range, zeros, NaN and infinities."""
    g = torch.Generator(device=dev).manual_seed(seed + 31 * M + C)
    x = torch.randn(M, C, generator=g, device=dev, dtype=torch.float64)
    kind = torch.randint(0, 12, (M, -(-C // 32)), generator=g, device=dev).repeat_interleave(32, 1)[:, :C]
    fi = torch.finfo(dtype)
    pick = torch.randint(0, 1 << 16, (M, C), generator=g, device=dev)
    x = torch.where(kind == 1, torch.round(x * 8) / 8, x)                       # ties of 4 bits
    x = torch.where(kind == 2, (pick % 256 - 128).double() / 2, x)               # ties of 8 bits
    x = torch.where(kind == 3, torch.tensor([1.75, 1.7421875, 1.9921875, 1.984375, 1.0, 2.0], device=dev,
                                            dtype=torch.float64)[pick % 6] * torch.sign(x), x)
    x = torch.where(kind == 4, x * fi.smallest_normal, x)
    x = torch.where(kind == 5, x * fi.smallest_normal * fi.eps * 3, x)
    x = torch.where(kind == 6, torch.sign(x) * fi.max * (1 - (pick % 64).double() / 64), x)
    x = torch.where(kind == 7, torch.zeros_like(x), x)
    x = torch.where((kind == 8) & (pick % 40 == 0), torch.full_like(x, float("nan")), x)
    x = torch.where((kind == 9) & (pick % 40 == 0), torch.full_like(x, float("-inf")), x)
    x = torch.where(kind == 10, x * torch.exp2(-(pick % 20).double()), x)
    return x.to(dtype)
