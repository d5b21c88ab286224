"""CPU tests of the modulated norm, the activations kept in 8 bits and the rows in 4 bits: what the C entry
points and the Python functions refuse, before any GPU work, and the layout of the 4-bit scales."""
import ctypes

import pytest
import torch

import reels_amd as ra
from reels_amd import _lib, modulation
from tests._blocks import blocks4, hard_rows

F = ctypes.c_void_p(4096)
BF = torch.bfloat16


def _err():
    return _lib.lib().reels_hip_last_error().decode()


def test_modulated_norm_c_refusals():
    L = _lib.lib()

    def norm(x=F, ldx=8, b=None, ldb=8, g=None, sc=F, sh=F, mt=0, dt=1, M=4, C=8, rpg=2, eps=1e-6, s=None, y=F, st=F,
             ks=None, kss=None, kb=None, kbs=None):
        return L.reels_hip_modulated_norm(x, ldx, b, ldb, g, 8, sc, 8, sh, 8, mt, dt, M, C, rpg, eps, 1, s, y, st, ks, kss, kb, kbs, None)

    def mx4(x=F, b=None, g=None, sc=F, sh=F, dt=1, M=4, C=8, rpg=2, s=None, q=F, qs=F):
        return L.reels_hip_modulated_norm_mx4(x, 8, b, 8, g, 8, sc, 8, sh, 8, 0, dt, M, C, rpg, 1e-6, 1, s, q, qs, None)
    assert norm(dt=3) == -2 and norm(mt=2) == -2 and norm(dt=0, mt=1) == -2
    assert norm(M=-1) == -1 and norm(C=0) == -1 and norm(C=16385, ldx=20000) == -1 and norm(M=1 << 31, rpg=1) == -1
    assert norm(rpg=0) == -1 and norm(rpg=3) == -1 and "rows_per_group" in _err()
    assert norm(eps=-1.0) == -1 and norm(eps=float("nan")) == -1 and norm(eps=float("inf")) == -1
    assert norm(sh=None) == -1 and norm(sc=None) == -1 and "together" in _err()
    assert norm(g=F) == -1 and "branch" in _err()
    assert norm(ldx=7) == -1 and norm(b=F, ldb=7, s=F) == -1 and "strides" in _err()
    assert norm(b=F) == -1 and norm(x=None) == -1 and norm(y=None) == -1 and norm(st=None) == -1 and "NULL" in _err()
    assert norm(ks=F) == -1 and norm(kss=F) == -1 and norm(kb=F, kbs=F, b=F, s=F) == -1
    assert norm(ks=F, kss=F, kb=F, kbs=F) == -1 and "kept" in _err()
    assert norm(M=0, x=None, y=None, st=None) == 0 and _err() == ""
    assert mx4(q=None) == -1 and mx4(qs=None) == -1 and mx4(b=F) == -1
    assert mx4(q=ctypes.c_void_p(4098)) == -1 and "aligned" in _err()
    assert mx4(dt=9) == -2 and mx4(g=F) == -1 and mx4(M=0, x=None, q=None, qs=None) == 0

    def bwd(dy=F, s=F, ss=None, b=None, bs=None, g=None, sc=F, st=F, mt=0, dt=1, M=64, C=8, rpg=64, dx=F, db=None, dg=None,
            dsc=None, dsh=None, ws=None, n=0):
        return L.reels_hip_modulated_norm_bwd(dy, s, ss, None, b, bs, g, 8, sc, 8, st, mt, dt, M, C, rpg, 1, dx, db, dg, dsc, dsh, ws, n, None)
    assert bwd(dt=4) == -2 and bwd(mt=2) == -2 and bwd(rpg=5) == -1 and bwd(C=1 << 20) == -1
    assert bwd(g=F) == -1 and bwd(db=F) == -1 and bwd(g=F, db=F, dg=F) == -1 and bwd(b=F, dg=F) == -1 and "dgate" in _err()
    assert bwd(dsc=F) == -1 and bwd(dsh=F) == -1 and bwd(sc=None, dsc=F, dsh=F) == -1 and "dscale" in _err()
    assert bwd(g=F, db=F, dg=F, b=F, ss=F) == -1 and bwd(g=F, db=F, dg=F, b=F, bs=F) == -1 and "8 bits" in _err()
    nb = L.reels_hip_modulated_norm_workspace_bytes(64, 8, 64)
    assert nb > 0 and bwd(dsc=F, dsh=F) == -3 and bwd(dsc=F, dsh=F, ws=F, n=nb - 1) == -3
    for name in ("dy", "s", "st", "dx"):
        assert bwd(**{name: None}) == -1 and "NULL" in _err()
    assert bwd(M=0, dy=None, s=None, st=None, dx=None) == 0
    ws = L.reels_hip_modulated_norm_workspace_bytes
    assert ws(0, 8, 1) == 0 and ws(8, 0, 1) == 0 and ws(100, 8, 1) == 0 and ws(8, 1 << 20, 8) == 0
    assert ws(32760, 5120, 32760) >= 3 * 5120 * 4 and ws(32760, 5120, 32760) % 256 == 0
    # a launch holds less than 2^32 threads: a wave for a row
    assert norm(M=1 << 28, rpg=1) == -1 and bwd(M=1 << 28, rpg=1) == -1 and "launch" in _err()


def test_act8_c_refusals():
    L = _lib.lib()
    keep, gelu, back, bwd = (L.reels_hip_act8_keep, L.reels_hip_act8_gelu_tanh, L.reels_hip_act8_restore,
                             L.reels_hip_act8_gelu_tanh_bwd)
    calls = [lambda dt, M, C, p=F: keep(p, dt, M, C, F, F, None), lambda dt, M, C, p=F: gelu(F, dt, M, C, p, F, F, None),
             lambda dt, M, C, p=F: back(F, p, dt, M, C, F, None), lambda dt, M, C, p=F: bwd(F, F, p, dt, M, C, F, None)]
    for call in calls:
        assert call(3, 4, 8) == -2 and call(-1, 4, 8) == -2
        assert call(1, -1, 8) == -1 and call(1, 4, 0) == -1 and call(1, 4, (1 << 30) + 1) == -1 and call(1, 1 << 31, 8) == -1
        assert call(1, 1 << 30, 64) == -1 and "launch" in _err()
        assert call(1, 4, 8, None) == -1 and "NULL" in _err()
        assert call(1, 0, 8, None) == 0 and _err() == ""


def test_mx4_c_refusals():
    L = _lib.lib()
    cb, sb = L.reels_hip_mx4_codes_bytes, L.reels_hip_mx4_scales_bytes
    assert cb(3, 1) == 3 * 128 and cb(3, 257) == 3 * 256 and sb(64, 256) == 512 and sb(65, 257) == 4 * 512
    assert cb(-1, 4) == 0 and cb(4, 0) == 0 and sb(0, 4) == 0
    odd = ctypes.c_void_p(4104)

    def pack(x=F, ld=8, dt=1, M=4, C=8, q=F, s=F):
        return L.reels_hip_mx4_pack(x, ld, dt, M, C, q, s, None)

    def unpack(q=F, s=F, dt=1, M=4, C=8, y=F):
        return L.reels_hip_mx4_unpack(q, s, dt, M, C, y, None)

    def lin(x=F, xs=F, w=F, ws=F, act=0, dt=1, M=40, K=64, N=8, y=F):
        return L.reels_hip_mx4_linear(x, xs, w, ws, None, None, act, dt, M, K, N, y, None)
    assert pack(dt=3) == -2 and unpack(dt=3) == -2 and lin(dt=3) == -2
    assert pack(ld=7) == -1 and pack(M=-1) == -1 and pack(C=0) == -1 and unpack(C=1 << 24) == -1 and unpack(M=1 << 31) == -1
    assert pack(q=odd) == -1 and pack(s=odd) == -1 and unpack(q=odd) == -1 and lin(x=odd) == -1 and lin(ws=odd) == -1
    assert "aligned" in _err()
    assert lin(act=2) == -1 and "activation" in _err()
    assert lin(M=-1) == -1 and lin(K=0) == -1 and lin(N=0) == -1 and lin(N=-1) == -1
    for f, names in ((pack, ("x", "q", "s")), (unpack, ("q", "s", "y")), (lin, ("x", "xs", "w", "ws", "y"))):
        for name in names:
            assert f(**{name: None}) == -1 and "NULL" in _err()
    assert pack(M=0, x=None, q=None, s=None) == 0 and unpack(M=0, q=None, s=None, y=None) == 0 and lin(M=0, x=None, y=None) == 0
    assert pack(M=(1 << 31) - 1, C=1000, ld=1000) == -1 and lin(M=1 << 30, N=1 << 30) == -1 and "launch" in _err()


def test_modulations_by_shape():
    def g(shape, t):
        return modulation._groups(torch.Size(shape), torch.Size(t), "m")
    assert g((3, 5, 8), (8,)) == 1 and g((3, 5, 8), (3, 8)) == 3
    assert g((3, 5, 8), (3, 1, 8)) == 3 and g((3, 5, 8), (3, 5, 8)) == 15
    assert g((3, 2, 5, 8), (3, 1, 1, 8)) == 3 and g((4, 8), (1, 8)) == 1
    assert g((4, 8), (4, 8)) == 4
    for shape, t in (((3, 5, 8), (5, 8)), ((3, 5, 8), (1, 1, 8)), ((3, 5, 8), (3, 5, 1)), ((4, 8), (2, 8)), ((3, 5, 8), (7,)),
                     ((3, 5, 8), ())):
        with pytest.raises(ValueError):
            g(shape, t)

    def mods(gate, scale, shift=None):
        return modulation._modulations(torch.zeros(3, 5, 8, dtype=BF), BF, ((gate, "gate"), (scale, "scale"), (shift, "shift")))
    six = torch.zeros(3, 6, 8)
    out, code, rpg = mods(six[:, 1:2], six[:, 2])
    assert rpg == 5 and code == _lib.F32 and out[1] == 48 and out[3] == 48 and out[4] is None
    assert out[0].data_ptr() == six[:, 1:2].data_ptr()  # taken as it lies
    assert mods(None, torch.zeros(8, dtype=BF))[1:] == (_lib.BF16, 15)
    with pytest.raises(ValueError, match="one kind"):
        mods(torch.zeros(8), torch.zeros(3, 8))
    with pytest.raises(ValueError, match="one kind"):
        mods(torch.zeros(3, 8, dtype=BF), torch.zeros(3, 8))
    with pytest.raises(TypeError):
        mods(torch.zeros(8, dtype=torch.float16), None)


def test_python_refusals():
    x = torch.zeros(4, 8, dtype=BF)
    k = ra.CompressedActivations(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8))
    q = ra.MicroscaledMatrix(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), (4, 8))
    for call in (lambda: ra.modulated_norm(x), lambda: ra.modulated_norm_quantized(x),
                 lambda: ra.modulated_norm_backward(x, x, torch.zeros(4, 3)), lambda: ra.compress_activations(x),
                 lambda: ra.gelu_tanh_compressed(x), lambda: ra.gelu_tanh_backward(k, x), lambda: k.restore(),
                 lambda: ra.quantize_microscaled(x), lambda: q.dequantize(), lambda: ra.microscaled_linear(q, q)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(TypeError):
        k.restore(torch.float64)
    with pytest.raises(TypeError):
        q.dequantize(torch.int8)
    with pytest.raises(ValueError):
        k.reshape(8, 4)
    assert k.reshape(2, 2, 8).scales.shape == (2, 2, 1) and k.reshape((-1, 8)).shape == (4, 8)
    with pytest.raises(ValueError):
        ra.microscaled_linear(ra.MicroscaledMatrix(q.codes, q.scales, (4, 0)), q)


def test_blocks_of_a_microscaled_matrix():
    """from_blocks and block_scales are each other's inverse, in the order that the header gives."""
    for M, K in ((1, 1), (70, 300), (130, 513)):
        c, s, _ = blocks4(hard_rows(M, K, torch.float32, "cpu").double())
        p = torch.nn.functional.pad(c, (0, K % 2))
        p = p[:, 0::2] + 16 * p[:, 1::2]
        q = ra.MicroscaledMatrix.from_blocks(p, s, K)
        assert q.shape == (M, K) and q.codes.shape == (M, -(-K // 256) * 128) and q.scales.shape == (-(-M // 64), -(-K // 256), 512)
        assert torch.equal(q.codes[:, :p.shape[1]], p) and not q.codes[:, p.shape[1]:].any()
        assert torch.equal(q.block_scales(), s)
        for r in range(0, M, 23):
            for b in range(s.shape[1]):
                i = b % 8
                at = (i % 2 * 32 + r % 64 % 32) * 8 + i // 2 * 2 + r % 64 // 32
                assert q.scales[r // 64, b // 8, at] == s[r, b]
    for bad in ((p[:, :3], s, K), (p, s[:, :1], K), (p.int(), s, K), (p[0], s, K), (p, s, 0)):
        with pytest.raises(ValueError):
            ra.MicroscaledMatrix.from_blocks(*bad)
    empty = ra.MicroscaledMatrix.from_blocks(p[:0], s[:0], K)
    assert empty.shape == (0, K) and empty.block_scales().shape == (0, s.shape[1])
    turned = q.scales.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ra.MicroscaledMatrix(q.codes, turned, q.size).block_scales(), s)


def test_sum_over_strided_rows_is_refused():
    """sum may be x or branch themselves, but not where their rows lie further apart than the sum's."""
    L = _lib.lib()
    G = ctypes.c_void_p(1 << 20)
    for x, b, ldx, ldb in ((F, G, 9, 8), (G, F, 8, 9)):
        assert L.reels_hip_modulated_norm(x, ldx, b, ldb, None, 8, None, 8, None, 8, 0, 1, 4, 8, 2, 1e-6, 1, F, G, G, None, None, None,
                                          None, None) == -1 and "stride" in _err()
        assert L.reels_hip_modulated_norm_mx4(x, ldx, b, ldb, None, 8, None, 8, None, 8, 0, 1, 4, 8, 2, 1e-6, 1, F, G, G, None) == -1
        assert "stride" in _err()


def test_kept_rows_on_another_device_are_refused():
    """The restored values would lie on the kept rows' device, where the linear's backward on dy's reads them."""
    from reels_amd import layers
    k = ra.CompressedActivations(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8))
    for needed in (True, False):
        with pytest.raises(ValueError, match="dy on cuda:1"):
            layers._saved_x(k, BF, needed, torch.device("cuda", 1))
    assert layers._saved_x(k, BF, False, torch.device("cpu")) is None
