"""CPU tests of the operators around the linears: what the C entry points and the Python functions
refuse, before any GPU work."""
import ctypes

import pytest
import torch

import reels_amd as ra
from reels_amd import _lib

F = ctypes.c_void_p(4096)
BF = torch.bfloat16


def _err():
    return _lib.lib().reels_hip_last_error().decode()


def test_rms_norm_c_refusals():
    L = _lib.lib()

    def norm(x=F, ld_x=8, r=None, ld_r=8, w=F, wt=1, dt=1, M=4, C=8, eps=1e-6, s=None, y=F, rstd=F):
        return L.reels_hip_rms_norm(x, ld_x, r, ld_r, w, wt, dt, M, C, eps, s, y, rstd, None)
    assert norm(dt=3) == -2 and norm(dt=7) == -2 and norm(wt=2) == -2
    assert norm(wt=2, w=None, x=None) == -1  # without a weight its type does not matter
    assert norm(M=-1) == -1 and norm(C=0) == -1 and norm(C=1 << 31, ld_x=1 << 31) == -1 and norm(M=1 << 31) == -1
    assert norm(eps=-1.0) == -1 and norm(eps=float("nan")) == -1 and norm(eps=float("inf")) == -1
    assert "eps" in _err()
    assert norm(ld_x=7) == -1 and norm(r=F, ld_r=7, s=F) == -1 and norm(r=F) == -1
    assert norm(x=None) == -1 and norm(y=None) == -1 and norm(rstd=None) == -1
    assert "reels_hip_rms_norm" in _err() and "NULL" in _err()
    assert norm(M=0, x=None, y=None, rstd=None) == 0 and _err() == ""
    q = L.reels_hip_rms_norm_i8
    assert q(F, 8, None, 8, F, 1, 1, 4, 8, 1e-6, None, None, F, None) == -1
    assert q(F, 8, None, 8, F, 1, 1, 4, 8, 1e-6, None, F, None, None) == -1
    assert "reels_hip_rms_norm_i8" in _err()
    ws = L.reels_hip_rms_norm_workspace_bytes
    assert ws(-1, 8) == 0 and ws(8, 0) == 0
    assert ws(0, 8) > 0 and ws(32760, 5120) >= 5120 * 4 and ws(32760, 5120) % 256 == 0
    b = L.reels_hip_rms_norm_bwd
    assert b(F, F, None, F, 1, F, 1, 4, 8, F, F, None, 0, None) == -3
    assert b(F, F, None, F, 1, F, 1, 4, 8, F, F, F, 1, None) == -3
    assert b(None, F, None, F, 1, F, 1, 4, 8, F, None, None, 0, None) == -1
    assert b(F, F, None, F, 1, None, 1, 4, 8, F, None, None, 0, None) == -1
    assert b(F, F, None, F, 1, F, 9, 4, 8, F, None, None, 0, None) == -2
    assert b(None, None, None, None, 1, None, 1, 0, 8, None, None, None, 0, None) == 0


def test_product_c_refusals():
    L = _lib.lib()
    nb = L.reels_hip_i8i8_workspace_bytes
    assert nb(-1, 4, 4) == 0 and nb(1, 0, 4) == 0 and nb(1, 4, 0) == 0
    assert nb(0, 1, 1) == 0 and nb(16, 5120, 13824) == 0  # few tokens take the codes as they lie
    for size in ((17, 1, 1), (777, 1000, 3001), (32760, 13824, 5120)):
        assert nb(*size) >= (size[0] + size[2]) * size[1] and nb(*size) % 256 == 0

    def prod(x=F, xs=F, w=F, ws=F, act=0, dt=1, M=40, K=64, N=8, y=F, work=F, n=1 << 30):
        return L.reels_hip_i8i8_linear(x, xs, w, ws, None, None, act, dt, M, K, N, y, work, n, None)
    assert prod(dt=3) == -2
    assert prod(act=2) == -1 and "activation" in _err()
    assert prod(M=-1) == -1 and prod(K=0) == -1 and prod(N=0) == -1 and prod(K=1 << 17) == -1
    assert prod(work=None, K=63) == -3 and prod(n=0, K=63) == -3
    for name in ("x", "xs", "w", "ws", "y"):
        assert prod(**{name: None}) == -1 and "NULL" in _err()
    assert prod(M=0, x=None, y=None) == 0


def test_rotary_c_refusals():
    L = _lib.lib()
    pairs = (ctypes.c_int32 * 3)(2, 1, 1)

    def rot(q=F, ldq=16, k=F, ldk=16, pos=F, pt=3, pb=1, dt=1, B=2, S=3, Hq=2, Hk=2, D=8, ap=pairs, n=3,
            theta=1e4, yq=F, yk=F):
        return L.reels_hip_rotary(q, ldq, k, ldk, pos, pt, pb, dt, B, S, Hq, Hk, D, ap, n, theta, 1, 0, yq, yk, None)
    assert rot(dt=3) == -2 and rot(pt=1) == -2
    assert rot(D=7) == -1 and rot(D=0) == -1 and rot(D=514, ldq=1 << 20, ldk=1 << 20) == -1
    assert rot(D=6) == -1 and "pairs" in _err()  # four pairs do not fit three
    assert rot(n=0) == -1 and rot(n=5) == -1 and rot(ap=None) == -1
    assert rot(ap=(ctypes.c_int32 * 3)(2, -1, 1)) == -1
    assert rot(theta=0.0) == -1 and rot(theta=float("nan")) == -1 and rot(theta=float("inf")) == -1
    assert rot(pb=3) == -1 and rot(ldq=15) == -1 and rot(ldk=15) == -1
    assert rot(B=-1) == -1 and rot(S=1 << 31) == -1 and rot(B=1 << 20, S=1 << 20, pb=1) == -1
    for name in ("q", "k", "pos", "yq", "yk"):
        assert rot(**{name: None}) == -1 and "NULL" in _err()
    assert rot(S=0, q=None) == 0 and rot(Hq=0, Hk=0, q=None, k=None) == 0


def test_clip_c_refusals():
    L = _lib.lib()
    assert L.reels_hip_grad_workspace_bytes(-1) == 0 and L.reels_hip_grad_workspace_bytes(0) > 0
    nb = L.reels_hip_grad_workspace_bytes(3)

    def clip(g=(4096, 8192, 12288), o=(4096, 8192, 12288), n=(4, 4, 4), t=(0, 0, 0), m=1.0, norm=F, ws=F, nbytes=nb,
             count=3):
        def arr(ct, v):
            return None if v is None else ctypes.cast((ct * len(v))(*v), ctypes.c_void_p)
        return L.reels_hip_clip_gradients(arr(ctypes.c_int64, g), arr(ctypes.c_int64, o), arr(ctypes.c_int64, n),
                                          arr(ctypes.c_int32, t), count, m, norm, ws, nbytes, None)
    assert clip(count=-1) == -1 and clip(g=None) == -1 and clip(o=None) == -1 and clip(norm=None) == -1
    assert clip(t=(0, 5, 0)) == -2 and clip(n=(4, -1, 4)) == -1 and clip(g=(4096, 0, 12288)) == -1
    assert clip(m=-1.0) == -1 and clip(m=float("nan")) == -1
    assert clip(ws=None) == -3 and clip(nbytes=8) == -3
    # the same tensor twice, an output on the next one's end, an output on another's gradient
    assert clip(g=(4096, 4096, 12288), o=(4096, 4096, 12288)) == -1 and "overlap" in _err()
    assert clip(o=(4096, 4108, 12288)) == -1
    assert clip(o=(8192, 16384, 12288)) == -1
    assert clip(g=(4096, 4100, 12288), o=(20000, 30000, 40000), norm=None) == -1  # (gradients may overlap; norm NULL)


def test_launches_of_2_to_32_threads_are_refused():
    """A launch holds less than 2^32 threads: 16 for a row of up to 512 (f32 256) elements, 1024 for the
    longest; 256 for each 16 tokens of a small head; 512 for 16 columns of a few tokens' product."""
    L = _lib.lib()
    pairs = (ctypes.c_int32 * 1)(1)
    for C, rows in ((8, 1 << 28), (8, (1 << 28) - 1), (1 << 20, 1 << 22)):
        assert L.reels_hip_rms_norm(F, C, None, C, None, 1, 1, rows, C, 1e-6, None, F, F, None) == -1
        assert L.reels_hip_rms_norm_i8(F, C, None, C, None, 1, 1, rows, C, 1e-6, None, F, F, None) == -1
        assert L.reels_hip_rms_norm_bwd(F, F, None, None, 1, F, 1, rows, C, F, None, None, 0, None) == -1
        assert "rows" in _err()
    C = 1 << 28
    assert L.reels_hip_rms_norm_bwd(F, F, None, None, 1, F, 1, 1, C, F, F, F, 1 << 62, None) == -1 and "columns" in _err()
    S = (1 << 31) - 1
    assert L.reels_hip_rotary(F, 2, None, 0, F, 3, 1, 1, 1, S, 1, 0, 2, pairs, 1, 1e4, 1, 0, F, None, None) == -1
    assert "tokens" in _err()
    prod = L.reels_hip_i8i8_linear
    for M, K, N in ((1, 4096, 1 << 26), (4, 64, 1 << 30), (1 << 30, 64, 1 << 30)):
        assert prod(F, F, F, F, None, None, 0, 1, M, K, N, F, None, 0, None) == -1 and "launch" in _err()


def test_python_refusals():
    x = torch.zeros(4, 8, dtype=BF)
    for call in (lambda: ra.rms_norm(x), lambda: ra.rms_norm_quantized(x), lambda: ra.quantize_rows(x),
                 lambda: ra.rms_norm_backward(x, x, None, torch.zeros(4)),
                 lambda: ra.rotary(torch.zeros(1, 4, 2, 8), torch.zeros(4, 1), (4,)),
                 lambda: ra.clip_gradients([x], 1.0), lambda: ra.gradient_norm([x])):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    W = ra.QuantizedMatrix(torch.zeros((5, 8), dtype=torch.int8), torch.ones(5))
    X = ra.QuantizedMatrix(torch.zeros((3, 8), dtype=torch.int8), torch.ones(3))
    with pytest.raises(ValueError, match="ROCm device"):
        ra.quantized_linear(X, W)
    bad = ra.QuantizedMatrix(torch.zeros((3, 9), dtype=torch.int8), torch.ones(3))
    for kw in (dict(x=bad), dict(bias=torch.zeros(4, dtype=BF)), dict(residual=torch.zeros(3, 4, dtype=BF)),
               dict(activation="relu")):
        with pytest.raises(ValueError):
            ra.quantized_linear(**{**dict(x=X, weight=W), **kw})
    with pytest.raises(TypeError):
        ra.quantized_linear(X, W, dtype=torch.float64)
    with pytest.raises(ValueError):
        ra.rms_norm_quantized(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError):
        ra.clip_gradients([], 1.0)
    with pytest.raises(ValueError):
        ra.clip_gradients([None], 1.0)
    with pytest.raises(ValueError):
        ra.clip_gradients([x], float("nan"))
    with pytest.raises(ValueError):
        ra.clip_gradients([x], 1.0, out=[None])
    with pytest.raises(ValueError):
        ra.clip_gradients([x], 1.0, out=[])
    with pytest.raises(TypeError):
        ra.gradient_norm([torch.zeros(3, dtype=torch.float64)])


def test_rotary_axes_and_grid():
    assert ra.rotary_axes(128) == (22, 21, 21) and ra.rotary_axes(64) == (12, 10, 10) and ra.rotary_axes(2) == (1, 0, 0)
    with pytest.raises(ValueError):
        ra.rotary_axes(3)
    p = ra.grid_positions(2, 3, 4)
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [0, 0, 0] and p[5].tolist() == [0, 1, 1] and p[23].tolist() == [1, 2, 3]


def test_dense_runs():
    from reels_amd.gradients import _dense
    t = torch.zeros(4, 6)
    assert _dense(t) and _dense(t.t()) and _dense(t[1:3]) and _dense(torch.zeros(0, 3)) and _dense(torch.zeros(()))
    assert _dense(torch.zeros(2, 3, 4, 5).contiguous(memory_format=torch.channels_last))
    assert not _dense(t[:, :3]) and not _dense(t[:, ::2]) and not _dense(torch.zeros(1, 3).expand(2, 3))
