"""rmsnorm and quant_rows on the GPU against the formulas in 64 bits.

H = DT(x + r): one rounding to fp32 and one to DT, compared bit for bit.  Y: the same two roundings of n,
whose own 64-bit error (K + 10 roundings of 2^-53) can move a value across a rounding border: half a step of
DT and 2^-20 of that more.  Codes are those of the 64-bit formula: the kernel makes the same operations
(x + r, times the weight, 127 t, the quotient), each correctly rounded, so they are equal.  Row scales: one
fp32 rounding, 2^-24, and 2^-40 for the 64-bit sums.  Group codes and scales are quant_a's of Y, bit for bit."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def make(seed, M, K, bf16, res, wtype, dist="normal", ldx=None, ldr=None, shift=0):
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(seed)

    def rows(ld, sigma):  # [M, K] with ld elements from row to row, `shift` elements past a 16-byte boundary
        ld = ld or K
        buf = torch.full((M * ld + 16,), 9.0, dtype=dt)
        v = buf[shift:shift + M * ld].view(M, ld)[:, :K]
        x = torch.randn((M, K), generator=g) * sigma
        if dist == "outliers":
            x[:, torch.randint(0, K, (max(1, K // 100),), generator=g)] *= 200
        elif dist == "ties":  # few whole values: quotients on halves
            x = torch.randint(-6, 7, (M, K), generator=g).float()
            x[:, 0] = 127 * 2
        elif dist == "tiny":
            x = x * (1e-37 if bf16 else 1e-7)
        elif dist == "huge":
            x = x * (5e37 if bf16 else 15000)
        v.copy_(x.to(dt))
        return buf.cuda()[shift:shift + M * ld].view(M, ld)[:, :K]

    X = rows(ldx, 1.0)
    R = rows(ldr, 3.0) if res else None
    W = None
    if wtype is not None:
        W = torch.rand(K, generator=g) * 0.9 + 0.1
        if dist == "ties":
            W = torch.ones(K)
        W = W.to(wtype).cuda()
    return X, R, W, dt


def gold(X, R, W, woff, eps=1e-6):
    x = X.double().cpu()
    h = x if R is None else x + R.double().cpu()
    s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + torch.tensor(eps, dtype=torch.float32).double())
    t = h if W is None else h * (W.double().cpu() + torch.tensor(woff, dtype=torch.float32).double())
    return h, t, s


def near(got, want, dt):
    e = torch.finfo(dt).eps / 2 * (1 + 2.0**-20)
    tiny = 2.0**-25 if dt == torch.float16 else 0.0 if dt == torch.float32 else 2.0**-134
    top = torch.finfo(dt).max
    ok = (got.double() - want).abs() <= e * want.abs() + tiny
    ok = ok | (got.isnan() & want.isnan())  # (what the formula makes of infinities)
    return (ok | (got.isinf() & (want.abs() > top * (1 - 1e-3)) & (got.sign() == want.sign()))).all()


def codes_of(t):
    """Codes 0 and a largest of NaN in a row with a value that is not finite."""
    fine = t.isfinite().all(1, keepdim=True)
    top = torch.where(fine, t.abs().amax(1, keepdim=True), torch.nan)
    return torch.where(top > 0, torch.round(127 * t / top), 0.0).to(torch.int8), top


def same_scales(got, want):
    ok = (got.double() - want).abs() <= (2.0**-24 + 2.0**-40) * want + 2.0**-150
    return (ok | (got.isnan() & want.isnan())).all()


def run(T, X, R, W, dt, quant, y, h=True, woff=0.0, place=None, eps=1e-6):
    M, K = X.shape
    new = lambda *s, d=dt: torch.full(s, 7, dtype=d, device="cuda")
    H = None if R is None or not h else X if place == "x" else R if place == "r" else new(M + 1, K)
    Y = new(M + 1, K) if y else None
    Q = new(M + 1, K, d=torch.int8) if quant != "none" else None
    SQ = None if quant == "none" else new(M + 1, d=torch.float32) if quant == "rows" else new(K // 128 + 1, T.ldsa(M))
    T.rmsnorm(X, R, W, H, Y, Q, SQ, M, K, eps, woff, quant, ldx=X.stride(0) if M > 1 else K,
              ldr=None if R is None else R.stride(0) if M > 1 else K)
    torch.cuda.synchronize()
    for t in (H if place is None else None, Y, Q):  # rows behind the last stay as they were
        assert t is None or (t[M:] == 7).all()
    if quant == "rows":
        assert SQ[M] == 7
    if quant == "groups":
        assert (SQ[:, M:] == 7).all() and (SQ[K // 128] == 7).all()
    cut = lambda t: None if t is None else t[:M]
    return cut(H), cut(Y), cut(Q), SQ if quant == "groups" else cut(SQ)


def check(T, seed, M, K, bf16, res=True, wtype=torch.float32, quant="rows", y=True, woff=0.0, place=None, **kw):
    X, R, W, dt = make(seed, M, K, bf16, res, wtype, **kw)
    h, t, s = gold(X, R, W, woff)
    H, Y, Q, SQ = run(T, X, R, W, dt, quant, y, woff=woff, place=place)
    n = t * s
    if R is not None:
        same = H.cpu() == h.float().to(dt)
        assert (same | (H.cpu().isnan() & h.isnan())).all()  # (NaN: infinities of both signs added)
    if y:
        assert near(Y.cpu(), n, dt)
    if quant == "rows":
        want, top = codes_of(t)
        assert torch.equal(Q.cpu(), want), (Q.cpu() != want).nonzero()[:4]
        assert same_scales(SQ.cpu(), (top * s / 127)[:, 0])
    elif quant == "groups":
        yy = Y if y else run(T, X, R, W, dt, "none", True, woff=woff)[1]
        want, sa = torch.empty_like(Q), torch.empty_like(SQ)
        T.quant_a(yy.contiguous(), sa, want, M, K)
        torch.cuda.synchronize()
        assert torch.equal(Q, want)
        assert torch.equal(SQ[:K // 128, :M], sa[:K // 128, :M])


KS = [1, 2, 7, 8, 63, 64, 65, 127, 128, 256, 511, 512, 513, 520, 1000, 1024, 1152, 2048, 2056, 4096, 4104, 5120, 5376, 8192,
      14336, 16384, 16392, 28672, 32768, 32776, 40960]


@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M", [1, 5])
def test_rows(dev, K, bf16, M):
    import ternocl_amd as T
    check(T, K + M, M, K, bf16, y=K % 2 == 0)


@pytest.mark.parametrize("K", [k for k in KS if k % 128 == 0])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M", [1, 5, 33])
def test_groups(dev, K, bf16, M):
    import ternocl_amd as T
    check(T, K + M, M, K, bf16, quant="groups", y=M == 5)


@pytest.mark.parametrize("K", [64, 77, 4096, 5120, 36872])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("wtype,woff", [(None, 0.0), (torch.float16, 0.0), (torch.bfloat16, 1.0), (torch.float32, 1.0)])
@pytest.mark.parametrize("quant", ["none", "rows"])
def test_variants(dev, K, bf16, res, wtype, woff, quant):
    import ternocl_amd as T
    check(T, K + 3, 6, K, bf16, res, wtype, quant, True, woff)


@pytest.mark.parametrize("K", [8, 384, 1001, 4096, 14336])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dist", ["outliers", "ties", "tiny", "huge"])
def test_values(dev, K, bf16, dist):
    import ternocl_amd as T
    check(T, K + 5, 9, K, bf16, dist=dist, y=True)
    check(T, K + 6, 9, K, bf16, dist=dist, res=False, wtype=None, y=False)
    if K % 128 == 0:
        check(T, K + 7, 9, K, bf16, dist=dist, quant="groups", y=True)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 8, 15, 16, 17, 63, 64, 255, 256, 257, 300, 1023, 2049])
@pytest.mark.parametrize("K", [64, 200, 1024, 4096])
def test_row_counts(dev, M, K):
    import ternocl_amd as T
    check(T, M + K, M, K, True)


@pytest.mark.parametrize("K,ldx,ldr,shift", [(4096, 4104, 4096, 0), (4096, 4096, 8192, 0), (4096, 4097, 4096, 0),
                                             (4096, 4096, 4099, 0), (512, 520, 512, 1), (512, 512, 512, 4), (1000, 1001, 1003, 3),
                                             (128, 1024, 2048, 8)])
@pytest.mark.parametrize("quant", ["rows", "groups"])
def test_pitches(dev, K, ldx, ldr, shift, quant):
    import ternocl_amd as T
    if quant == "groups" and K % 128:
        quant = "none"
    check(T, K + ldx, 7, K, True, quant=quant, ldx=ldx, ldr=ldr, shift=shift)


@pytest.mark.parametrize("K", [100, 4096, 36864])
@pytest.mark.parametrize("place", ["x", "r"])
@pytest.mark.parametrize("quant", ["rows", "groups"])
def test_in_place(dev, K, place, quant):
    """H over X or R."""
    import ternocl_amd as T
    if K % 128:
        quant = "rows"
    X, R, W, dt = make(K, 11, K, True, True, torch.bfloat16)
    want = run(T, X, R, W, dt, quant, True)
    got = run(T, X.clone() if place == "r" else X, R.clone() if place == "x" else R, W, dt, quant, True, place=place)
    for i, (a, b) in enumerate(zip(got, want)):
        if i == 3 and quant == "groups":
            a, b = a[:, :11], b[:, :11]
        assert torch.equal(a, b)
    assert torch.equal(X if place == "x" else R, want[0])


@pytest.mark.parametrize("K", [64, 333, 4096, 36864])
@pytest.mark.parametrize("bf16", [False, True])
def test_not_finite(dev, K, bf16):
    """A row with an infinity or a NaN: scale NaN, codes 0, H and Y by the formula; the other rows as without it.  A
    row of zeros: scale and codes 0."""
    import ternocl_amd as T
    X, R, W, dt = make(K, 8, K, bf16, True, torch.float32)
    X[1, K // 2] = float("inf")
    X[3, K - 1] = float("nan")
    R[4, 0] = -float("inf")
    X[6] = 0
    R[6] = 0
    bad = torch.tensor([False, True, False, True, True, False, False, False])
    for quant in ("rows", "none"):
        h, t, s = gold(X, R, W, 0.0)
        H, Y, Q, SQ = run(T, X, R, W, dt, quant, True)
        assert torch.equal(H.cpu().isnan(), h.isnan()) and torch.equal(H.cpu().isinf(), h.isinf())
        n = t * s
        assert torch.equal(Y.cpu().isnan(), n.isnan())
        assert near(Y.cpu()[~bad], n[~bad], dt) and (Y[6] == 0).all()
        if quant == "rows":
            assert torch.equal(SQ.cpu().isnan(), bad) and (Q[bad.cuda()] == 0).all()
            want, _ = codes_of(t[~bad])
            assert torch.equal(Q.cpu()[~bad], want) and SQ[6] == 0
    Q, SQ = torch.ones((8, K), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    T.quant_rows(X, Q, SQ, 8, K)
    x = X.double().cpu()
    bad[4] = False
    assert torch.equal(SQ.cpu().isnan(), bad) and (Q[bad.cuda()] == 0).all() and SQ[6] == 0
    assert torch.equal(Q.cpu()[~bad], codes_of(x[~bad])[0])
    W[K // 3] = float("inf")  # a weight that is not finite: every row's scale
    assert run(T, X, R, W, dt, "rows", False)[3].isnan().all()
    if K % 128 == 0:
        X[0, 5] = float("nan")
        _, Y, Q, SA = run(T, X, R, W, dt, "groups", True)
        want, sa = torch.empty_like(Q), torch.empty_like(SA)
        T.quant_a(Y.contiguous(), sa, want, 8, K)
        assert torch.equal(Q, want) and torch.equal(SA[:K // 128, :8].isnan(), sa[:K // 128, :8].isnan())


def test_row_lost_in_the_norm(dev):
    """eps far above a row's mean square: scales far below the values' own, to fp32's last bits."""
    import ternocl_amd as T
    X, _, _, dt = make(1, 4, 512, True, False, None, dist="tiny")
    h, t, s = gold(X, None, None, 0.0, 1e30)
    _, Y, Q, SQ = run(T, X, None, None, dt, "rows", True, eps=1e30)
    want, top = codes_of(t)
    assert torch.equal(Q.cpu(), want)
    sc = (top * s / 127)[:, 0]
    assert ((SQ.cpu().double() - sc).abs() <= 2.0**-23 * sc + 2.0**-149).all()


@pytest.mark.parametrize("K", [1, 5, 64, 1000, 1024, 4096, 14336, 20480, 32768, 32769, 50000])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pad", [(1, 0), (6, 8), (300, 0), (6, 3)])
@pytest.mark.parametrize("dist", ["outliers", "ties"])
def test_quant_rows(dev, K, bf16, M, pad, dist):
    import ternocl_amd as T
    X, _, _, _ = make(K + M, M, K, bf16, False, None, dist=dist, ldx=K + pad)
    Q = torch.full((M + 1, K), 7, dtype=torch.int8, device="cuda")
    SQ = torch.full((M + 1,), 7.0, device="cuda")
    T.quant_rows(X, Q, SQ, M, K, ld=K + pad)
    want, top = codes_of(X.double().cpu())
    assert torch.equal(Q[:M].cpu(), want) and (Q[M] == 7).all()
    assert same_scales(SQ[:M].cpu(), top[:, 0] / 127) and SQ[M] == 7


def test_far_rows(dev):
    """Elements past 2^31 of a wide tensor: pitches of 2^28, and 2^31 + outputs."""
    import ternocl_amd as T
    ld = 1 << 28
    buf = torch.zeros(9 * ld, dtype=torch.bfloat16, device="cuda")
    X = buf.view(9, ld)[:, :512]
    g = torch.Generator().manual_seed(3)
    X.copy_(torch.randn((9, 512), generator=g).to(torch.bfloat16))
    Q, SQ = torch.empty((9, 512), dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
    T.quant_rows(X, Q, SQ, 9, 512, ld=ld)
    assert torch.equal(Q.cpu(), codes_of(X.double().cpu())[0])
    H, Y, Q, SQ = run(T, X, X, None, torch.bfloat16, "rows", True)
    h, t, s = gold(X, X, None, 0.0)
    assert torch.equal(H.cpu(), h.float().bfloat16()) and near(Y.cpu(), t * s, torch.bfloat16)
    assert torch.equal(Q.cpu(), codes_of(t)[0])
    del X, buf
    M = (1 << 31) // 1024 + 3
    X = torch.randn((M, 1024), device="cuda", dtype=torch.bfloat16)
    Q, SQ = torch.empty((M, 1024), dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    T.quant_rows(X, Q, SQ, M, 1024)
    for i in (0, M // 2, M - 1):
        assert torch.equal(Q[i:i + 1].cpu(), codes_of(X[i:i + 1].double().cpu())[0])


def test_streams_and_graph(dev):
    """On another stream, and captured: replays on new inputs equal eager calls."""
    import ternocl_amd as T
    X, R, W, dt = make(1, 6, 5120, True, True, torch.bfloat16)
    st = torch.cuda.Stream()
    H, Y = torch.empty_like(X), torch.empty_like(X)
    Q, SQ = torch.empty((6, 5120), dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        T.rmsnorm(X, R, W, H, Y, Q, SQ, 6, 5120, quant="rows")
    for i in range(4):
        X.copy_(make(10 + i, 6, 5120, True, True, None)[0])
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (H, Y, Q, SQ)]
        with torch.cuda.stream(st):
            want = run(T, X, R, W, dt, "rows", True)
        st.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("K", [64, 77, 264])
def test_many_rows(dev, K):
    """More rows than one launch holds."""
    import ternocl_amd as T
    M = (1 << 21) + 3
    X = torch.randn((M, K), device="cuda", dtype=torch.bfloat16)
    Q, SQ = torch.full((M + 1, K), 7, dtype=torch.int8, device="cuda"), torch.full((M + 1,), 7.0, device="cuda")
    Y, H = torch.empty_like(X), torch.empty_like(X)
    for norm in (False, True):
        if norm:
            T.rmsnorm(X, X, None, H, Y, Q, SQ, M, K, quant="rows")
        else:
            T.quant_rows(X, Q, SQ, M, K)
        torch.cuda.synchronize()
        assert (Q[M] == 7).all() and SQ[M] == 7
        for i in (0, (1 << 21) - 2, M - 4):
            x = X[i:i + 4].double().cpu()
            assert torch.equal(Q[i:i + 4].cpu(), codes_of(x)[0])  # (x + x scales by a power of two: the same codes)
            if norm:
                h, t, s = gold(X[i:i + 4], X[i:i + 4], None, 0.0)
                assert torch.equal(H[i:i + 4].cpu(), h.float().bfloat16()) and near(Y[i:i + 4].cpu(), t * s, torch.bfloat16)
    want = codes_of(X[::1001].double().cpu())[0]
    assert torch.equal(Q[:M][::1001].cpu(), want)


@pytest.mark.parametrize("K", [64, 77, 256, 4096, 36864])
@pytest.mark.parametrize("off", [1, 2, 4, 7])
@pytest.mark.parametrize("quant", ["rows", "groups"])
def test_outputs_at_any_element(dev, K, off, quant):
    """H, Y, codes, scales and weights that start `off` elements past a 16-byte boundary: the bits of aligned ones, and
    nothing before or behind them written.  In the group case with an infinity and a NaN, whose scales are compared
    bit for bit with quant_a's."""
    import ternocl_amd as T
    if K % 128:
        quant = "rows"
    M = 5
    X, R, W, dt = make(K + off, M, K, True, True, torch.float32)
    if quant == "groups":
        X[1, 3], X[3, K - 1] = float("inf"), float("nan")
    want = run(T, X, R, W, dt, quant, True)
    bufs = []

    def at(n, d):
        bufs.append(torch.full((n + 32,), 7, dtype=d, device="cuda"))
        return bufs[-1][off:off + n]

    w = at(K, torch.float32)
    w.copy_(W)
    ns = M if quant == "rows" else K // 128 * T.ldsa(M)
    got = [at(M * K, dt), at(M * K, dt), at(M * K, torch.int8), at(ns, torch.float32 if quant == "rows" else dt)]
    T.rmsnorm(X, R, w, *got, M, K, quant=quant)
    torch.cuda.synchronize()
    bits = lambda t: t.contiguous().view(torch.uint8)
    for g, x in zip(got[:3], want):
        assert torch.equal(bits(g), bits(x).flatten())
    if quant == "rows":
        assert torch.equal(bits(got[3]), bits(want[3]))
    else:
        sa, q = torch.empty((K // 128, T.ldsa(M)), dtype=dt, device="cuda"), torch.empty((M, K), dtype=torch.int8, device="cuda")
        T.quant_a(got[1].clone(), sa, q, M, K)
        g = got[3].view(K // 128, T.ldsa(M))
        assert torch.equal(bits(g[:, :M]), bits(sa[:, :M])) and torch.equal(got[2].view(M, K), q)
        assert (g[:, M:] == 7).all()
    for b, t in zip(bufs, [w] + got):
        assert (b[:off] == 7).all() and (b[off + t.numel():] == 7).all()
