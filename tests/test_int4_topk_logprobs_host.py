"""The 4-bit products, routing and log probabilities without a GPU: the host packers against the
layout written out, every refusal of the C entries (before any device call: the pointers are never
followed), the workspace queries, and the torch operators' fake implementations."""
from __future__ import annotations

import numpy as np
import pytest

import ternocl_amd as T

torch = pytest.importorskip("torch")
INVALID, SHAPE = 1, 2


@pytest.mark.parametrize("K,N", [(32, 1), (64, 3), (256, 48)])
def test_int4_pack(K, N):
    g = np.random.default_rng(K + N)
    W = g.integers(-8, 8, (K, N)).astype(np.int8)
    B = T.int4_pack(W)
    assert B.shape == (K // 32, N, 4) and B.dtype == np.uint32
    for k in range(K):  # row 2i of a word in nibble i, row 2i + 1 in nibble i + 4
        r = k % 8
        nib = r // 2 + (4 if r % 2 else 0)
        q = (B[k // 32, :, k % 32 // 8] >> (4 * nib)) & 15
        assert (np.where(q > 7, q.astype(int) - 16, q) == W[k]).all()
    assert (T.int4_unpack(B, K) == W).all()


def test_int4_pack_refusals():
    L = T.lib()
    W, B = np.zeros((32, 16), np.int8), np.zeros((1, 16, 4), np.uint32)
    p = lambda a: a.ctypes.data
    assert L.ternocl_int4_pack(p(W), p(B), 32, 16) == 0
    assert L.ternocl_int4_pack(p(W), p(B), 31, 16) == SHAPE
    assert L.ternocl_int4_pack(p(W), p(B), 32, 0) == SHAPE
    assert L.ternocl_int4_pack(None, p(B), 32, 16) == INVALID
    for bad in (8, -9):
        W[5, 3] = bad
        assert L.ternocl_int4_pack(p(W), p(B), 32, 16) == INVALID
    assert L.ternocl_int4_unpack(p(B), None, 32, 16) == INVALID
    assert L.ternocl_int4_unpack(p(B), p(W), 16, 16) == SHAPE


def _int4(**kw):
    a = dict(dtype=0, A=4096, B=4096, S=4096, Z=None, C=4096, Other=None, Bias=None, M=1, N=4096, K=4096, group=128,
             postop=0, out_f32=0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return T.lib().ternocl_int4_gemm(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), INVALID), (dict(A=None), INVALID), (dict(B=None), INVALID), (dict(S=None), INVALID),
    (dict(C=None), INVALID), (dict(B=4104), INVALID), (dict(group=16), INVALID), (dict(group=256), INVALID),
    (dict(group=0), INVALID), (dict(postop=6), INVALID), (dict(postop=1), INVALID), (dict(postop=3), INVALID),
    (dict(out_f32=2), INVALID), (dict(M=0), SHAPE), (dict(N=8), SHAPE), (dict(N=4100), SHAPE), (dict(K=64), SHAPE),
    (dict(K=4000), SHAPE)])
def test_int4_refusals(kw, status):
    assert _int4(**kw) == status
    assert T.lib().ternocl_last_error().decode()


def test_int4_ws_bytes():
    for M, N, K, g in [(0, 4096, 4096, 128), (1, 4100, 4096, 128), (1, 4096, 100, 128), (1, 4096, 4096, 48)]:
        assert T.int4_gemm_ws_bytes(M, N, K, g) == 0
    for M, N, K in [(1, 4096, 4096), (4, 4096, 14336), (24, 4096, 14336), (300, 5120, 5120)]:
        n = T.int4_gemm_ws_bytes(M, N, K, 128)
        assert n == 0 or n > T.WS_HEADER_BYTES


def _topk(**kw):
    a = dict(ltype=2, logits=4096, ld=64, bias=None, ids=4096, wtype=1, RW=4096, T=4, E=64, topk=8, score=0, n_group=1,
             topk_group=1, group_best=1, renorm=1, scale=1.0, stream=None)
    a.update(kw)
    return T.lib().ternocl_moe_topk(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(ltype=3), INVALID), (dict(wtype=-1), INVALID), (dict(logits=None), INVALID), (dict(ids=None), INVALID),
    (dict(RW=None), INVALID), (dict(score=2), INVALID), (dict(renorm=2), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(T=0), SHAPE), (dict(T=2**25 + 1), SHAPE), (dict(logits=4098), INVALID), (dict(ltype=0, logits=4097), INVALID), (dict(E=0), SHAPE), (dict(E=513, ld=513), SHAPE),
    (dict(ld=63), SHAPE), (dict(n_group=0), SHAPE), (dict(n_group=5), SHAPE), (dict(E=128, ld=128, n_group=128), SHAPE),
    (dict(n_group=4, topk_group=5), SHAPE), (dict(topk_group=0), SHAPE), (dict(group_best=0), SHAPE),
    (dict(group_best=3), SHAPE), (dict(n_group=64, topk_group=8, group_best=2), SHAPE), (dict(topk=0), SHAPE),
    (dict(topk=65, E=128, ld=128), SHAPE), (dict(E=4, ld=4, topk=5), SHAPE), (dict(n_group=16, topk_group=1, topk=5), SHAPE)])
def test_topk_refusals(kw, status):
    assert _topk(**kw) == status
    assert T.lib().ternocl_last_error().decode()


def _logprobs(**kw):
    a = dict(ltype=2, logits=4096, ld=1000, tokens=4096, logp=4096, entropy=4096, top_ids=4096, top_logp=4096, M=4, V=1000,
             topn=5, scale=1.0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return T.lib().ternocl_logprobs(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(ltype=7), INVALID), (dict(logits=None), INVALID), (dict(logits=4098), INVALID), (dict(ltype=0, logits=4097), INVALID),
    (dict(tokens=None), INVALID), (dict(logp=None), INVALID), (dict(topn=65), INVALID), (dict(topn=-1), INVALID),
    (dict(top_ids=None), INVALID), (dict(top_logp=None), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(scale=2.0**101), INVALID),
    (dict(scale=2.0**-101), INVALID), (dict(M=0), SHAPE), (dict(M=2**23 + 1), SHAPE), (dict(V=0), SHAPE),
    (dict(ld=999), SHAPE), (dict(tokens=None, logp=None, entropy=None, topn=0), INVALID)])
def test_logprobs_refusals(kw, status):
    assert _logprobs(**kw) == status
    assert T.lib().ternocl_last_error().decode()


def test_logprobs_ws_bytes():
    assert T.logprobs_ws_bytes(0, 1000, 5) == 0 and T.logprobs_ws_bytes(1, 1000, 65) == 0
    assert all(T.logprobs_ws_bytes(1, V, 5) == 0 for V in (1, 2, 3, 4))
    assert T.logprobs_ws_bytes(1, 1000, 5) == 0  # one workgroup holds the row
    assert T.logprobs_ws_bytes(4096, 151680, 5) == 0  # the rows fill the chip
    assert T.logprobs_ws_bytes(1, 151680, 5) > T.logprobs_ws_bytes(1, 151680, 0) > T.WS_HEADER_BYTES


def test_python_refusals():
    x = torch.zeros(2, 8)
    with pytest.raises(T.TernoclError):
        T.moe_topk(x, None, x, x, 2, 8, 2, score="tanh", stream=0)
    B = np.zeros((2, 3, 4), np.uint32)
    assert T.int4_unpack(B, 64).shape == (64, 3)
    for b, K in ((B, 96), (B, 32), (B[:, :, :2], 64), (B[0], 32)):  # (never read past B)
        with pytest.raises(T.TernoclError):
            T.int4_unpack(b, K)
    with pytest.raises(T.TernoclError):
        T.logprobs(x.double(), None, None, x, None, None, 2, 8, stream=0)


def test_ops_fake_shapes_and_refusals():
    import ternocl_amd.torch_ops  # noqa: F401
    ops = torch.ops.ternocl
    m = dict(device="meta")
    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32

    def bad(fn, *args):
        with pytest.raises(RuntimeError):
            fn(*args)
    A, B = torch.empty((5, 256), dtype=bf, **m), torch.empty((8, 48, 4), dtype=i32, **m)
    S = torch.empty((4, 48), dtype=bf, **m)
    assert ops.int4_gemm(A, B, S, None, 64, None, None, 0, False).shape == (5, 48)
    assert ops.int4_gemm(A, B, S, S, 64, None, None, 0, True).dtype == f32
    assert ops.int4_gemm(A[:0], B, S, S, 64, None, None, 0, True).shape == (0, 48)
    bad(ops.int4_gemm, A, B, S, None, 128, None, None, 0, False)              # S rows for another group
    bad(ops.int4_gemm, A, B, S, None, 48, None, None, 0, False)
    bad(ops.int4_gemm, A, B, S, S.half(), 64, None, None, 0, False)
    bad(ops.int4_gemm, A, B.long(), S, None, 64, None, None, 0, False)
    bad(ops.int4_gemm, A, B.transpose(0, 1), S, None, 64, None, None, 0, False)
    bad(ops.int4_gemm, A, B[:, :, :2], S, None, 64, None, None, 0, False)
    bad(ops.int4_gemm, A, B, S, None, 64, None, torch.empty(48, dtype=bf, **m), 3, True)  # fp32 out: fp32 bias
    lg = torch.empty((7, 64), dtype=f32, **m)
    args = ("softmax", 1, 1, 1, True, 1.0)
    ids, rw = ops.moe_topk(lg, None, 8, bf, *args)
    assert ids.shape == rw.shape == (7, 8) and ids.dtype == i32 and rw.dtype == bf
    bad(ops.moe_topk, lg.double(), None, 8, bf, *args)
    bad(ops.moe_topk, lg.t(), None, 7, bf, *args)
    bad(ops.moe_topk, lg, torch.empty(63, dtype=f32, **m), 8, bf, *args)
    bad(ops.moe_topk, lg, torch.empty(64, dtype=bf, **m), 8, bf, *args)
    bad(ops.moe_topk, lg, None, 0, bf, *args)
    bad(ops.moe_topk, lg, None, 8, i32, *args)
    tok = torch.empty(7, dtype=i32, **m)
    out = ops.logprobs(lg, tok, 5, 1.0)
    assert [tuple(o.shape) for o in out] == [(7,), (7,), (7, 5), (7, 5)] and out[2].dtype == i32
    bad(ops.logprobs, lg, tok.long(), 5, 1.0)
    bad(ops.logprobs, lg, tok[:6], 5, 1.0)
    bad(ops.logprobs, lg, tok, 65, 1.0)
    bad(ops.logprobs, lg[:1].expand(7, 64), tok, 5, 1.0)
