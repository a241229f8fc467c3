"""The norm, the 8-bit rows and the products of 8-bit integers without a GPU: the host packers against the
layout written out, every refusal of the C entries (before any device call: the pointers are never
followed), the workspace query, and the torch operators' fake implementations and checks."""
from __future__ import annotations

import numpy as np
import pytest

import ternocl_amd as T

torch = pytest.importorskip("torch")
INVALID, SHAPE = 1, 2
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("K,N", [(16, 1), (64, 3), (256, 48)])
def test_int8_pack(K, N):
    g = np.random.default_rng(K + N)
    W = g.integers(-128, 128, (K, N)).astype(np.int8)
    B = T.int8_pack(W)
    assert B.shape == (K // 16, N, 16) and B.dtype == np.int8
    for k in range(K):
        assert (B[k // 16, :, k % 16] == W[k]).all()
    assert (T.int8_unpack(B, K) == W).all()


def test_int8_pack_refusals():
    L = T.lib()
    W, B = np.zeros((32, 16), np.int8), np.zeros((2, 16, 16), np.int8)
    p = lambda a: a.ctypes.data
    for f in (L.ternocl_int8_pack, L.ternocl_int8_unpack):
        assert f(p(W), p(B), 32, 16) == 0
        assert f(p(W), p(B), 24, 16) == SHAPE
        assert f(p(W), p(B), 0, 16) == SHAPE
        assert f(p(W), p(B), 32, 0) == SHAPE
        assert f(None, p(B), 32, 16) == INVALID
        assert f(p(W), None, 32, 16) == INVALID
    with pytest.raises(T.TernoclError):
        T.int8_unpack(B, 48)


def _norm(**kw):
    a = dict(dtype=1, X=4096, ldx=256, R=8192, ldr=256, wtype=1, W=4096, woff=0.0, eps=1e-6, H=16384, Y=16384, quant=1,
             Q=4096, SQ=4096, M=2, K=256, stream=None)
    a.update(kw)
    return T.lib().ternocl_rmsnorm(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), INVALID), (dict(dtype=-1), INVALID), (dict(X=None), INVALID), (dict(X=4097), INVALID),
    (dict(ldx=255), SHAPE), (dict(ldr=255), SHAPE), (dict(wtype=3), INVALID), (dict(wtype=-1), INVALID),
    (dict(W=4097), INVALID), (dict(W=4098, wtype=2), INVALID), (dict(woff=INF), INVALID), (dict(woff=NAN), INVALID),
    (dict(eps=0.0), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=NAN), INVALID), (dict(eps=INF), INVALID),
    (dict(quant=3), INVALID), (dict(quant=-1), INVALID), (dict(Q=None), INVALID), (dict(SQ=None), INVALID),
    (dict(SQ=4098), INVALID), (dict(quant=2, SQ=4097), INVALID), (dict(quant=0, Y=None), INVALID), (dict(R=None), INVALID),
    (dict(R=8193), INVALID), (dict(H=16385), INVALID), (dict(Y=16385), INVALID), (dict(quant=2, K=200), SHAPE),
    (dict(M=0), SHAPE), (dict(M=(1 << 23) + 1), SHAPE), (dict(K=0), SHAPE), (dict(H=4096, ldx=264), INVALID),
    (dict(H=8192, ldr=264), INVALID)])
def test_rmsnorm_refusals(kw, status):
    assert _norm(**kw) == status
    assert T.lib().ternocl_last_error().decode()


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), INVALID), (dict(X=None), INVALID), (dict(X=4097), INVALID), (dict(ldx=255), SHAPE), (dict(Q=None), INVALID),
    (dict(SQ=None), INVALID), (dict(SQ=4098), INVALID), (dict(M=0), SHAPE), (dict(M=(1 << 23) + 1), SHAPE), (dict(K=0), SHAPE)])
def test_quant_rows_refusals(kw, status):
    a = dict(dtype=0, X=4096, ldx=256, Q=4096, SQ=4096, M=2, K=256, stream=None)
    a.update(kw)
    assert T.lib().ternocl_quant_rows(*a.values()) == status
    assert T.lib().ternocl_last_error().decode()


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), INVALID), (dict(A=None), INVALID), (dict(SA=None), INVALID), (dict(B=None), INVALID), (dict(SB=None), INVALID),
    (dict(C=None), INVALID), (dict(B=4104), INVALID), (dict(SA=4098), INVALID), (dict(SB=4098), INVALID), (dict(postop=6), INVALID),
    (dict(postop=1), INVALID), (dict(postop=2), INVALID), (dict(postop=3), INVALID), (dict(postop=5), INVALID),
    (dict(out_f32=2), INVALID), (dict(M=0), SHAPE), (dict(N=8), SHAPE), (dict(N=4100), SHAPE), (dict(K=64), SHAPE),
    (dict(K=4000), SHAPE), (dict(K=1 << 17), SHAPE)])
def test_int8_gemm_refusals(kw, status):
    a = dict(dtype=0, A=4096, SA=4096, B=4096, SB=4096, C=4096, Other=None, Bias=None, M=1, N=4096, K=4096, postop=0, out_f32=0,
             ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    assert T.lib().ternocl_int8_gemm(*a.values()) == status
    assert T.lib().ternocl_last_error().decode()


def test_ws_bytes_query():
    q = T.int8_gemm_ws_bytes
    for M, N, K in ((0, 4096, 4096), (1, 8, 4096), (1, 4100, 4096), (1, 4096, 64), (1, 4096, 1 << 17), (-1, 16, 128)):
        assert q(M, N, K) == 0
    for M, N, K in ((1, 4096, 4096), (24, 4096, 14336), (200, 5120, 5120), (4096, 34816, 5120)):
        n = q(M, N, K)
        assert n == 0 or n >= T.WS_HEADER_BYTES + 2 * 4 * M * N  # counters and at least two slices' sums


def test_python_refusals():
    with pytest.raises(T.TernoclError, match="quant"):
        T.rmsnorm(None, None, None, None, None, None, None, 1, 1, quant="row")


# ---- the torch operators' checks, on meta tensors ----------------------------------------

def meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_shapes():
    import ternocl_amd.torch_ops  # noqa: F401
    o = torch.ops.ternocl
    x = meta(5, 256, dtype=torch.bfloat16)
    h, y, q, s = o.rmsnorm(x, x, meta(256, dtype=torch.float32), 1e-6, 0.0, "rows", True)
    assert h.shape == y.shape == q.shape == (5, 256) and s.shape == (5,)
    assert h.dtype == y.dtype == torch.bfloat16 and q.dtype == torch.int8 and s.dtype == torch.float32
    h, y, q, s = o.rmsnorm(x, None, None, 1e-6, 0.0, "groups", False)
    assert h.shape == y.shape == (0,) and q.shape == (5, 256) and s.shape == (2, 32) and s.dtype == torch.bfloat16
    h, y, q, s = o.rmsnorm(x, None, None, 1e-6, 0.0, "none", True)
    assert y.shape == (5, 256) and q.shape == s.shape == (0,)
    q, s = o.quant_rows(meta(0, 77))
    assert q.shape == (0, 77) and s.shape == (0,)
    i8 = dict(dtype=torch.int8)
    f = dict(dtype=torch.float32)
    a = (meta(5, 256, **i8), meta(5, **f), meta(16, 48, 16, **i8), meta(48, **f))
    assert o.int8_gemm(*a, torch.bfloat16, None, None, 0, False).dtype == torch.bfloat16
    c = o.int8_gemm(*a, torch.float16, meta(5, 48), meta(48, **f), 5, True)
    assert c.shape == (5, 48) and c.dtype == torch.float32


@pytest.mark.parametrize("call", [
    lambda o: o.rmsnorm(meta(5, 256, dtype=torch.float32), None, None, 1e-6, 0.0, "rows", False),
    lambda o: o.rmsnorm(meta(5, 256), meta(5, 256, dtype=torch.bfloat16), None, 1e-6, 0.0, "rows", False),
    lambda o: o.rmsnorm(meta(5, 256), meta(4, 256), None, 1e-6, 0.0, "rows", False),
    lambda o: o.rmsnorm(meta(5, 256), None, meta(255), 1e-6, 0.0, "rows", False),
    lambda o: o.rmsnorm(meta(5, 200), None, None, 1e-6, 0.0, "groups", False),
    lambda o: o.rmsnorm(meta(5, 256), None, None, 1e-6, 0.0, "cols", False),
    lambda o: o.rmsnorm(meta(256, 5).t(), None, None, 1e-6, 0.0, "rows", False),
    lambda o: o.rmsnorm(meta(1, 256).expand(5, 256), None, None, 1e-6, 0.0, "rows", False),
    lambda o: o.quant_rows(meta(5, 0)),
    lambda o: o.quant_rows(meta(5, 8, dtype=torch.float32)),
    lambda o: o.int8_gemm(meta(5, 256), meta(5, dtype=torch.float32), meta(16, 48, 16, dtype=torch.int8),
                          meta(48, dtype=torch.float32), torch.float16, None, None, 0, False),
    lambda o: o.int8_gemm(meta(5, 256, dtype=torch.int8), meta(5), meta(16, 48, 16, dtype=torch.int8),
                          meta(48, dtype=torch.float32), torch.float16, None, None, 0, False),
    lambda o: o.int8_gemm(meta(5, 256, dtype=torch.int8), meta(5, dtype=torch.float32), meta(16, 40, 16, dtype=torch.int8),
                          meta(40, dtype=torch.float32), torch.float16, None, None, 0, False),
    lambda o: o.int8_gemm(meta(5, 256, dtype=torch.int8), meta(5, dtype=torch.float32), meta(16, 48, 16, dtype=torch.int8),
                          meta(48, dtype=torch.float32), torch.float32, None, None, 0, True),
    lambda o: o.int8_gemm(meta(5, 256, dtype=torch.int8), meta(5, dtype=torch.float32), meta(16, 48, 16, dtype=torch.int8),
                          meta(48, dtype=torch.float32), torch.bfloat16, meta(5, 48), None, 2, False)])
def test_fake_refusals(call):
    import ternocl_amd.torch_ops  # noqa: F401
    with pytest.raises(Exception):
        call(torch.ops.ternocl)


@pytest.mark.parametrize("M,N", [((1 << 30) + 200, 16), ((1 << 31) - 1, 16), ((1 << 31) - 128, 16), (1 << 20, 1 << 20), (1, 1 << 30),
                                 (1, (1 << 31) - 16), ((1 << 31) - 1, (1 << 31) - 16)])
def test_int8_gemm_past_a_launch(M, N):
    """Refused as a shape before any device call, and no tile or workspace named for it."""
    L = T.lib()
    assert L.ternocl_int8_gemm(0, 4096, 4096, 4096, 4096, 4096, None, None, M, N, 128, 0, 0, None, 0, None) == SHAPE
    assert L.ternocl_last_error().decode()
    assert T.kw_tile_of(4, M, N, 128) is None and T.int8_gemm_ws_bytes(M, N, 128) == 0


def test_fake_refuses_nothing_to_compute():
    """As the operator itself, so that a trace does not pass what a run refuses."""
    import ternocl_amd.torch_ops  # noqa: F401
    with pytest.raises(Exception, match="nothing to compute"):
        torch.ops.ternocl.rmsnorm(meta(5, 256), None, None, 1e-6, 0.0, "none", False)


@pytest.mark.parametrize("kw,word", [(dict(R=None), "R must be non-null"), (dict(H=4096, ldx=264), "rows of K"),
                                     (dict(H=8192, ldr=264), "rows of K")])
def test_rmsnorm_says_when_h_is_refused(kw, word):
    """The sum with R only with R, and in place of X or R only where these have rows of K; the interface says both."""
    from pathlib import Path
    assert _norm(**kw) == INVALID
    assert word in T.lib().ternocl_last_error().decode()
    text = " ".join((Path(__file__).resolve().parents[1] / "include" / "ternocl_amd.h").read_text().replace("*", " ").split())
    assert "H = DT(h) [M, K], only with R; may be X or R itself where that has rows of K" in text
