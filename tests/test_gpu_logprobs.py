"""logprobs on the GPU against the definition in 64 bits.

Tolerances: with n = V / 256 + 64 additions at most on the way of a term (a lane's share of an unsplit row,
then the lanes, waves and chunks), sums of fp32 terms are good to n 2^-24, relative; a term's exponent d =
scale (x - max) is rounded three times (the difference, the scale, the change of base), an error of 3 |d|
2^-24 in its logarithm, and terms with |d| > 40 weigh less than 2^-57.  So ln p is good to (n + 120 + 4
|ln p|) 2^-24, and where the row is peaked (ln p of the largest entry -r) to that relative to r; the
entropy to 2 (n + 160) 2^-24 of 1 + H (absolutely) or of H where it is small."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
NAMES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def gold(x, tokens, topn, scale):
    raw = x.double()
    M, V = raw.shape
    top = torch.sort(raw, dim=1, descending=True, stable=True).indices
    d = (raw - raw.gather(1, top[:, :1])) * scale
    e = torch.exp(d).scatter(1, top[:, :1], 0.0)
    r = e.sum(1)
    l1 = torch.log1p(r)
    H = l1 - torch.where(e > 0, d * e, 0.0).sum(1) / (1 + r)
    t = tokens.long()
    ok = (t >= 0) & (t < V)
    lp = torch.where(ok, d.gather(1, t.clamp(0, V - 1)[:, None])[:, 0] - l1, 0.0)
    n = min(topn, V)
    ids = top[:, :n]
    tl = d.gather(1, ids) - l1[:, None]
    dead = raw.gather(1, ids) == -math.inf
    ids, tl = ids.masked_fill(dead, -1), tl.masked_fill(dead, -math.inf)
    if n < topn:
        ids = torch.cat([ids, torch.full((M, topn - n), -1)], 1)
        tl = torch.cat([tl, torch.full((M, topn - n), -math.inf, dtype=torch.float64)], 1)
    return lp, H, ids.to(torch.int32), tl


def call(T, x, tokens, topn, scale=1.0, ld=None, ws=True, at=0):
    M, V = x.shape
    ld = ld or V
    buf = torch.full((at + M * ld,), 50.0, dtype=x.dtype, device="cuda")
    L = buf[at:].view(M, ld)
    L[:, :V] = x.cuda()
    lp = torch.full((M + 1,), 7.0, device="cuda")
    H = torch.full((M + 1,), 7.0, device="cuda")
    ids = torch.full((M + 1, topn), 77, dtype=torch.int32, device="cuda")
    tl = torch.full((M + 1, topn), 7.0, device="cuda")
    nb = T.logprobs_ws_bytes(M, V, topn)
    w = torch.randint(0, 255, (nb,), dtype=torch.uint8, device="cuda") if nb and ws else None
    T.logprobs(L, tokens.cuda(), lp, H, ids if topn else None, tl if topn else None, M, V, ld, topn, scale, ws=w)
    torch.cuda.synchronize()
    assert lp[M] == 7 and H[M] == 7 and (ids[M] == 77).all() and (tl[M] == 7).all()
    return lp[:M].cpu(), H[:M].cpu(), ids[:M].cpu(), tl[:M].cpu()


def check(T, x, tokens, topn, scale=1.0, **kw):
    lp, H, ids, tl = call(T, x, tokens, topn, scale, **kw)
    glp, gH, gids, gtl = gold(x, tokens, topn, scale)
    n, u = x.shape[1] / 256 + 64, 2.0**-24

    def close(a, b):
        same = a.double() == b
        tol = (n + 120 + 4 * b.abs()) * u
        tol = torch.where(b.abs() < 0.1, 2 * tol * b.abs() + 4 * u * (b < -1e-3) , tol)
        return (same | ((a.double() - b).abs() <= tol)).all()
    assert torch.equal(ids, gids)
    assert close(lp, glp), (lp.double() - glp).abs().max()
    assert close(tl, gtl)
    tol = 2 * (n + 160) * u
    assert ((H.double() - gH).abs() <= torch.minimum(tol * (1 + gH), 4 * tol * gH + 1e-30)).all(), (H.double() - gH).abs().max()


def rows(seed, M, V, lt, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, V), generator=g) * sigma
    return x.to(NAMES[lt]), torch.randint(-1, V, (M,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 64, 255, 256, 1000, 1023, 4095, 4096, 4097, 8191, 8200, 32000, 151643])
@pytest.mark.parametrize("lt", list(NAMES))
def test_vocabularies(dev, V, lt):
    import ternocl_amd as T
    for M, topn in ((1, 20), (3, 5)):
        x, t = rows(V, M, V, lt)
        check(T, x, t, topn)
        check(T, x, t, topn, 0.7, ws=False)


@pytest.mark.parametrize("topn", [0, 1, 2, 19, 63, 64])
@pytest.mark.parametrize("M", [1, 2, 27, 300, 600])
def test_rows_and_alternatives(dev, M, topn):
    import ternocl_amd as T
    x, t = rows(M, M, 5003, "bf16")
    check(T, x, t, topn, 1.25)
    x, t = rows(M, M, 9001, "f32")
    check(T, x, t, topn)


@pytest.mark.parametrize("lt", list(NAMES))
@pytest.mark.parametrize("at", [0, 1, 3, 7])
def test_alignment_and_pitch(dev, lt, at):
    import ternocl_amd as T
    x, t = rows(at, 5, 4999, lt)
    check(T, x, t, 9, ld=5001, at=at)
    check(T, x, t, 9, ld=4999, at=at)
    x, t = rows(at, 5, 11, lt)
    check(T, x, t, 9, ld=13, at=at)


@pytest.mark.parametrize("ws", [True, False])
def test_ties(dev, ws):
    """Equal logits rank by index: a constant row, a row of a few values, a row with the type's lowest value
    everywhere but in three places, and whole pieces above the rest."""
    import ternocl_amd as T
    V = 40000
    low = torch.finfo(torch.float32).min
    x = torch.zeros(7, V)
    g = torch.Generator().manual_seed(0)
    x[1] = torch.randint(0, 3, (V,), generator=g).float()
    x[2] = low
    x[2, [39999, 5, 77]] = torch.tensor([1.0, 2.0, 1.0])
    x[3] = torch.arange(V).float() / 1000
    x[4] = -torch.arange(V).float() / 1000
    x[5, ::1024] = 3.0  # one thread's entries
    x[6, 1::2] = -0.0
    t = torch.tensor([0, 1, 5, 39999, -1, V, 3], dtype=torch.int32)
    for topn in (1, 20, 64):
        check(T, x, t, topn, ws=ws)
    h = (torch.randn(4, V, generator=g) * 2).to(torch.bfloat16)
    check(T, h, t[:4], 64, ws=ws)
    # more entries above any bound that one thread's would give than are ranked at once
    y = torch.randn(2, 300000, generator=g)
    for j in range(4):
        y[:, 4 * 7 + j::1024] += 50
    check(T, y, t[:2], 64, ws=ws)


@pytest.mark.parametrize("ws", [True, False])
def test_masks(dev, ws):
    """-inf entries weigh nothing and are not listed; empty rows; rows with one entry left."""
    import ternocl_amd as T
    V = 20000
    x, t = rows(1, 5, V, "f32")
    x[0, 3:] = -math.inf
    x[1, :V - 2] = -math.inf
    x[2, 1:] = -math.inf
    x[3, torch.rand(V, generator=torch.Generator().manual_seed(3)) < 0.9] = -math.inf
    t = torch.tensor([1, 0, 0, 17, 5], dtype=torch.int32)
    check(T, x, t, 20, ws=ws)
    e = torch.full((2, V), -math.inf)
    lp, H, ids, tl = call(T, e, torch.tensor([4, -1], dtype=torch.int32), 5, ws=ws)
    assert lp.tolist() == [-math.inf, 0.0] and H.tolist() == [0.0, 0.0]
    assert (ids == -1).all() and (tl == -math.inf).all()


@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", [0, 9999, 19999])
def test_not_finite(dev, ws, bad, where):
    import ternocl_amd as T
    x, t = rows(1, 3, 20000, "f32")
    t[:] = 3
    x[1, where] = bad
    lp, H, ids, tl = call(T, x, t, 5, ws=ws)
    assert torch.isnan(lp[1]) and torch.isnan(H[1]) and (ids[1] == -1).all() and torch.isnan(tl[1]).all()
    keep = [0, 2]
    good = call(T, x[keep], t[keep], 5, ws=False)
    assert torch.equal(ids[keep], good[2]) and torch.allclose(lp[keep], good[0], rtol=1e-6, atol=1e-5)
    assert torch.isfinite(H[keep]).all()
    x[1] = -math.inf
    x[1, where] = float("nan")
    assert torch.isnan(call(T, x, t, 5, ws=ws)[1][1])


@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("gap", [12.0, 25.0, 40.0, 80.0])
def test_peaked(dev, ws, gap):
    """ln p near 0 keeps its digits (4 u absolute is not enough: see check's close)."""
    import ternocl_amd as T
    x, _ = rows(2, 4, 50001, "f32", 0.5)
    t = torch.tensor([0, 50000, 25000, 1027], dtype=torch.int32)
    x[torch.arange(4), t.long()] = gap
    check(T, x, t, 3, ws=ws)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 30.0])
def test_scales(dev, scale):
    import ternocl_amd as T
    x, t = rows(6, 3, 12345, "f16")
    x[:, 7] = 65504.0 if scale < 1 else 9.0
    check(T, x, t, 8, scale)


@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("scale", [2.0**-100, 2.0**100])
def test_scale_limits(dev, scale, ws):
    """Both ends of the scales, logits to match, and logits whose difference is past fp32's range."""
    import ternocl_amd as T
    x, t = rows(12, 3, 40001, "f32")
    x = x / scale
    if scale < 1:
        x[1, 100], x[1, 200], t[1] = 3e38, -3e38, 200
        x[2, 100], x[2, 200], x[2, 40000], t[2] = 3e38, -3e38, 3e38, 200
    check(T, x, t, 8, scale, ws=ws)


@pytest.mark.parametrize("scale", [0.25, 1.0])
def test_widest_difference(dev, scale):
    """The type's lowest value beside its largest: listed with its ln p where that is in fp32."""
    import ternocl_amd as T
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[-big, big, 0.0, -big, -math.inf]])
    lp, H, ids, tl = call(T, x, torch.tensor([3], dtype=torch.int32), 5, scale)
    want = [0.0, -big * scale, -2 * big * scale, -2 * big * scale, -math.inf]
    want = [w if w >= -big else -math.inf for w in want]
    assert ids.tolist() == [[1, 2, 0, 3, -1]] and H.tolist() == [0.0]
    assert lp.item() == want[3] and tl.tolist() == [want]


def test_parts_may_be_left_out(dev):
    import ternocl_amd as T
    x, t = rows(6, 3, 12345, "f16")
    L, tk = x.cuda(), t.cuda()
    full = call(T, x, t, 4)
    lp, H = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    ids, tl = torch.empty((3, 4), dtype=torch.int32, device="cuda"), torch.empty((3, 4), device="cuda")
    T.logprobs(L, tk, lp, None, None, None, 3, 12345)
    T.logprobs(L, None, None, H, None, None, 3, 12345)
    T.logprobs(L, None, None, None, ids, tl, 3, 12345, topn=4)
    for a, b in zip((lp, H, tl), (full[0], full[1], full[3])):
        assert torch.allclose(a.cpu(), b, rtol=1e-5, atol=1e-5)
    assert torch.equal(ids.cpu(), full[2])


def test_op_graph_and_stream(dev):
    import ternocl_amd.torch_ops  # noqa: F401
    op = torch.ops.ternocl.logprobs
    x = torch.randn(5, 30001, device="cuda") * 3
    t = torch.arange(5, dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        op(x, t, 10, 0.9)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = op(x, t, 10, 0.9)
    for _ in range(4):
        x.normal_()
        want = op(x, t, 10, 0.9)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert [o.shape[0] for o in op(x[:0], t[:0], 10, 1.0)] == [0, 0, 0, 0]
    a, b = op(x[:, 5:29990], t, 10, 1.0), op(x[:, 5:29990].contiguous(), t, 10, 1.0)
    assert torch.equal(a[2], b[2]) and torch.allclose(a[0], b[0], rtol=1e-5, atol=1e-5)
    torch.library.opcheck(op.default, (x, t, 10, 0.9), test_utils=("test_schema", "test_faketensor"))


def test_offsets_past_32_bits(dev):
    """Rows past 2^32 bytes and 2^31 elements: the first and the last."""
    import ternocl_amd as T
    M, V = 15000, 151680
    x = torch.randn((M, V), dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2**31
    t = torch.randint(0, V, (M,), dtype=torch.int32, device="cuda")
    lp, H = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    ids, tl = torch.empty((M, 3), dtype=torch.int32, device="cuda"), torch.empty((M, 3), device="cuda")
    T.logprobs(x, t, lp, H, ids, tl, M, V, topn=3)
    for r in ([0, 1], [M // 2, M // 2 + 1], [M - 2, M - 1]):
        glp, gH, gids, gtl = gold(x[r].cpu(), t[r].cpu(), 3, 1.0)
        assert torch.equal(ids[r].cpu(), gids) and torch.allclose(lp[r].cpu().double(), glp, atol=1e-4)
        assert torch.allclose(H[r].cpu().double(), gH, atol=1e-4) and torch.allclose(tl[r].cpu().double(), gtl, atol=1e-4)


@pytest.mark.parametrize("Tk", [1, 5, 70])
def test_decode_step(dev, Tk):
    """The calls as a model makes them: router logits -> moe_topk -> the ternary MoE layer -> a 4-bit head ->
    logprobs, each against its definition on the inputs it was given."""
    import numpy as np
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    from gpu_util import dev_dt, dev_raw, dev_raw as raw  # noqa: F401
    from ternocl_amd import synth
    import test_gpu_topk as tt
    import test_gpu_int4 as t4
    ops = torch.ops.ternocl
    E, topk, H, I, V = 16, 4, 256, 256, 1504
    g = synth.rng(5)
    st = lambda K, N: (torch.stack([dev_raw(synth.int2_weights(g, K, N)) for _ in range(E)]),
                       torch.stack([dev_dt(synth.scales(g, K, N, True), True) for _ in range(E)]))
    (Bg, Sg), (Bu, Su), (Bd, Sd) = st(H, I), st(H, I), st(I, H)
    X = torch.randn(Tk, H, device="cuda").to(torch.bfloat16)
    router = torch.randn(H, E, device="cuda") * 0.1
    lg = X.float() @ router
    ids, RW = ops.moe_topk(lg, None, topk, torch.bfloat16, "softmax", 1, 1, 1, True, 1.0)
    want_ids, want_w = tt.gold(lg.cpu(), None, topk, "softmax", 1, 1, 1, True, 1.0)
    assert torch.equal(ids.cpu(), want_ids)
    layer = ops.moe_decode if Tk <= 8 else ops.moe_prefill
    O = layer(X, ids, RW, E, Bg, Sg, Bu, Su, Bd, Sd)
    hid = (X.float() + O.float()).to(torch.bfloat16)
    A, W, S, Z, dt = t4.make(4, Tk, H, V, 64, True, True)
    B = torch.from_numpy(T.int4_pack(W.numpy()).view(np.int32)).cuda()
    logits = ops.int4_gemm(hid, B, S.cuda(), Z.cuda(), 64, None, None, 0, True)
    want, d = t4.gold(hid.cpu(), W, S, Z, 64, None, None, 0)
    assert ((logits.cpu().double() - want).abs() <= 2.0**-24 * want.abs() + d).all()
    tok = logits.argmax(1).to(torch.int32)
    lp, ent, ti, tl = ops.logprobs(logits, tok, 6, 1.0)
    glp, gH, gids, gtl = gold(logits.cpu(), tok.cpu(), 6, 1.0)
    assert torch.equal(ti.cpu(), gids) and torch.allclose(lp.cpu().double(), glp, atol=2e-5) and torch.allclose(ent.cpu().double(), gH, atol=1e-4)
