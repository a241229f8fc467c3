"""int8_gemm on the GPU against the product in whole numbers, at every type, epilogue and engine.

Sums are exact.  fp32 outputs without an epilogue are (float(sum) * SB) * SA, bit for bit.  Others: three
roundings of that (3.01 2^-24), one of each addition or product of the epilogue, and one of the output."""
from __future__ import annotations

import pytest

from gpu_util import off16

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def make(seed, M, K, N, dist="normal"):
    g = torch.Generator().manual_seed(seed)
    if dist == "normal":
        r = lambda *s: (torch.randn(s, generator=g) * 40).round().clamp(-128, 127).to(torch.int8)
    elif dist == "any":
        r = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int8)
    else:  # the largest sums
        r = lambda *s: torch.full(s, -128, dtype=torch.int8)
    A, W = r(M, K), r(K, N)
    SA, SB = torch.rand(M, generator=g) * 0.02 + 0.01, torch.rand(N, generator=g) * 1e-3 + 1e-4
    return A, SA, W, SB


def packed(W):
    K, N = W.shape
    return W.view(K // 16, 16, N).transpose(1, 2).contiguous()


def exact_sums(A, W):
    """(64-bit floats: whole numbers below 2^53)"""
    return (A.cuda().double() @ W.cuda().double()).cpu() if A.shape[0] * W.numel() > 1e8 else A.double() @ W.double()


def gold(A, SA, W, SB, other, bias, postop):
    s = exact_sums(A, W)
    v32 = (s.float() * SB) * SA[:, None]
    acc = s * SB.double() * SA.double()[:, None]
    d = 3.01 * 2.0**-24 * acc.abs()
    if postop in (1, 4):
        sg = torch.where(acc <= -10, 0.0, 1 / (1 + torch.exp(-acc)))
        # (the epilogue's sigmoid is good to about 2^-20; a product near -10 may fall on either side of its cut)
        cut = torch.where((acc + 10).abs() <= d, 5e-5, 0.0)
        if postop == 4:
            return sg, d + 2.0**-20 + cut, v32
        o = other.double()
        return acc * sg * o, (1.1 * d + 2.0**-20 * acc.abs() * sg + 10 * cut) * o.abs(), v32
    v, m = acc, acc.abs()
    if postop in (3, 5):
        v, m = v + bias.double(), m + bias.double().abs()
    if postop in (2, 5):
        v, m = v + other.double(), m + other.double().abs()
    return v, d + 2 * 2.0**-24 * m, v32


def run(T, A, SA, W, SB, dt, other, bias, postop, f32, ws="random", move=()):
    M, K = A.shape
    N = W.shape[1]
    dev = lambda t: None if t is None else t.cuda()
    B = packed(dev(W))
    a = dict(A=dev(A), SA=dev(SA), SB=dev(SB), other=dev(other), bias=dev(bias),
             C=torch.full((M + 2, N), 7.0, dtype=torch.float32 if f32 else dt, device="cuda"))
    for k in move:
        if a[k] is not None:
            a[k] = off16(a[k])
    nb = T.int8_gemm_ws_bytes(M, N, K)
    w = None
    if nb and ws == "random":
        w = torch.randint(0, 255, (nb,), dtype=torch.uint8, device="cuda")
    elif nb and ws:
        w = torch.zeros(nb, dtype=torch.uint8, device="cuda")
    if other is None and f32:  # (nothing else says the type: not read)
        dt = None
    T.int8_gemm(a["A"], a["SA"], B, a["SB"], a["C"], a["other"], a["bias"], M, N, K, postop, f32, ws=w)
    torch.cuda.synchronize()
    C = a["C"]
    assert (C[M:] == 7.0).all()  # rows behind the last stay as they were
    return C[:M]


def check(T, seed, M, K, N, bf16=False, postop=0, f32=True, dist="normal", **kw):
    A, SA, W, SB = make(seed, M, K, N, dist)
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(seed + 1)
    other = torch.randn((M, N), generator=g).to(dt) if postop in (1, 2, 5) else None
    bias = torch.randn(N, generator=g).to(torch.float32 if f32 else dt) if postop in (3, 5) else None
    got = run(T, A, SA, W, SB, dt, other, bias, postop, f32, **kw).cpu()
    want, d, v32 = gold(A, SA, W, SB, other, bias, postop)
    if postop == 0:
        assert torch.equal(got, v32 if f32 else v32.to(dt)), ((got.float() - v32).abs().max(), (got != v32.to(got.dtype)).sum())
    u = torch.finfo(torch.float32 if f32 else dt).eps / 2
    tiny = 0.0 if f32 or bf16 else 2.0**-25  # (fp16 subnormals)
    err = (got.double() - want).abs() - (u * want.abs() + d * (1 + u) + tiny)
    big = want.abs() > torch.finfo(got.dtype).max * 0.999
    assert not ((err > 0) & ~big).any(), (err.max().item(), (err > 0).sum().item())
    return got


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256,
                               257, 500])
@pytest.mark.parametrize("K,N", [(512, 208), (1152, 1040)])
def test_rows(dev, M, K, N):
    import ternocl_amd as T
    check(T, 11 * M, M, K, N)


@pytest.mark.parametrize("M", [1, 6, 20, 40, 100, 300])
@pytest.mark.parametrize("postop", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("bf16,f32", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(dev, M, postop, bf16, f32):
    import ternocl_amd as T
    check(T, 100 + postop, M, 384, 528, bf16, postop, f32)


@pytest.mark.parametrize("K,N", [(128, 16), (128, 4096), (256, 32), (640, 48), (1152, 16), (4096, 16), (5376, 80), (14336, 64),
                                 (17408, 32), (40960, 16), (130944, 16)])
@pytest.mark.parametrize("M", [1, 4, 8, 17, 24, 130, 270])
def test_shapes(dev, K, N, M):
    import ternocl_amd as T
    check(T, K + N + M, M, K, N, dist="any")


@pytest.mark.parametrize("M,K,N", [(1, 4096, 4096), (1, 14336, 4096), (4, 1024, 16400), (8, 4096, 6144), (2, 2048, 40000), (24, 14336, 1024),
                                   (64, 4096, 4096), (96, 5120, 5120), (300, 1024, 1552), (700, 512, 2064), (1000, 256, 4112),
                                   (333, 512, 11024), (130, 1152, 16400), (1024, 4096, 4096), (257, 14336, 2048), (2048, 1024, 4096),
                                   (4096, 512, 9216), (3000, 640, 10256)])
def test_engines(dev, M, K, N):
    import ternocl_amd as T
    check(T, M + K + N, M, K, N)


@pytest.mark.parametrize("M,K", [(1, 130944), (16, 130944), (40, 65536), (300, 130944)])
def test_largest_sums(dev, M, K):
    """-128 * -128 over the longest K: 2^31 - 2^21."""
    import ternocl_amd as T
    check(T, 1, M, K, 48, dist="lowest")


@pytest.mark.parametrize("M,K,N", [(1, 4096, 4096), (5, 14336, 512), (24, 14336, 4096), (200, 5120, 5120), (100, 8192, 1024), (1024, 14336, 1040)])
def test_split_same_bits(dev, M, K, N):
    """With a workspace of any contents, with a zeroed one used twice, and without: the same bits."""
    import ternocl_amd as T
    A, SA, W, SB = make(M, M, K, N)
    o = torch.randn((M, N)).bfloat16()
    got = [run(T, A, SA, W, SB, torch.bfloat16, o, None, 2, False, ws=ws) for ws in ("random", "zero", None, "zero")]
    assert all(torch.equal(got[0], x) for x in got[1:])


def test_workspace_left_zero(dev):
    """A zeroed workspace's counters are zero after each call: every shape can follow every other on it."""
    import ternocl_amd as T
    shapes = [(24, 14336, 4096), (1, 14336, 4096), (200, 5120, 5120), (100, 8192, 1024), (24, 14336, 4096)]
    ws = torch.zeros(max(T.int8_gemm_ws_bytes(M, N, K) for M, K, N in shapes) + 16, dtype=torch.uint8, device="cuda")
    for M, K, N in shapes:
        A, SA, W, SB = make(M, M, K, N)
        C = torch.empty((M, N), device="cuda")
        for _ in range(3):
            T.int8_gemm(A.cuda(), SA.cuda(), packed(W.cuda()), SB.cuda(), C, None, None, M, N, K, 0, True, ws=ws)
            torch.cuda.synchronize()
            assert (ws[:T.WS_HEADER_BYTES] == 0).all()
        assert torch.equal(C.cpu(), (exact_sums(A, W).float() * SB) * SA[:, None])


@pytest.mark.parametrize("M", [1, 7, 40, 300])
@pytest.mark.parametrize("move", [("A",), ("SA",), ("SB",), ("C",), ("other",), ("bias",), ("A", "SA", "SB", "C", "other", "bias")])
@pytest.mark.parametrize("f32", [False, True])
def test_alignment(dev, M, move, f32):
    import ternocl_amd as T
    check(T, M, M, 512, 144, True, 5, f32, move=move)


@pytest.mark.parametrize("shift", [1, 2, 3, 5, 8, 15])
def test_any_byte_of_A(dev, shift):
    import ternocl_amd as T
    A, SA, W, SB = make(shift, 9, 256, 48)
    buf = torch.zeros(9 * 256 + 16, dtype=torch.int8, device="cuda")
    a = buf[shift:shift + 9 * 256].view(9, 256)
    a.copy_(A)
    C = torch.empty((9, 48), device="cuda")
    T.int8_gemm(a, SA.cuda(), packed(W.cuda()), SB.cuda(), C, None, None, 9, 48, 256, 0, True)
    assert torch.equal(C.cpu(), (exact_sums(A, W).float() * SB) * SA[:, None])


@pytest.mark.parametrize("M", [1, 8, 20, 40, 300])
def test_scales(dev, M):
    """NaN, zero, huge and tiny scales: of a token its row, of a channel its column."""
    import ternocl_amd as T
    A, SA, W, SB = make(M, M, 512, 208)
    SA[0], SB[3], SB[5] = float("nan"), 0.0, float("nan")
    if M > 2:
        SA[1], SA[2] = 2.0**120, 2.0**-140
    got = run(T, A, SA, W, SB, torch.bfloat16, None, None, 0, True).cpu()
    want = (exact_sums(A, W).float() * SB) * SA[:, None]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~got.isnan()], want[~want.isnan()])


def test_far_weights(dev):
    """Weights, outputs and activations past 2^31 bytes."""
    import ternocl_amd as T
    g = torch.Generator("cuda").manual_seed(5)
    K, N = 14336, 151680  # 2.2 GB of weights
    B = torch.randint(-128, 128, (K // 16, N, 16), dtype=torch.int8, device="cuda", generator=g)
    SB = torch.rand(N, device="cuda", generator=g)
    for M in (1, 20, 70, 300):
        A = torch.randint(-128, 128, (M, K), dtype=torch.int8, device="cuda", generator=g)
        SA = torch.rand(M, device="cuda", generator=g)
        C = torch.empty((M, N), device="cuda")
        T.int8_gemm(A, SA, B, SB, C, None, None, M, N, K, 0, True)
        for n in (0, N // 2, N - 16):
            want = A.double() @ B[:, n:n + 16].transpose(1, 2).reshape(K, 16).double()
            assert torch.equal(C[:, n:n + 16], (want.float() * SB[n:n + 16]) * SA[:, None])
    del B, C
    M, K, N = (1 << 31) // 4096 + 300, 4096, 272  # 2.1 GB of activations
    A = torch.randint(-128, 128, (M, K), dtype=torch.int8, device="cuda", generator=g)
    B = torch.randint(-128, 128, (K // 16, N, 16), dtype=torch.int8, device="cuda", generator=g)
    SA, SB = torch.rand(M, device="cuda", generator=g), torch.rand(N, device="cuda", generator=g)
    C = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    T.int8_gemm(A, SA, B, SB, C, None, None, M, N, K, 0, False)
    for m in (0, M // 2, M - 64):
        want = A[m:m + 64].double() @ B.transpose(1, 2).reshape(K, N).double()
        assert torch.equal(C[m:m + 64], ((want.float() * SB) * SA[m:m + 64, None]).bfloat16())


def test_streams_and_graphs(dev):
    """Two captured graphs, each with a workspace of its own, replayed in turn with eager work between: equal to eager
    calls."""
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    M, K, N = 24, 8192, 1024
    A, SA, W, SB = make(3, M, K, N)
    A, SA, B, SB = A.cuda(), SA.cuda(), packed(W.cuda()), SB.cuda()
    o = torch.ops.ternocl
    graphs = []
    for _ in range(2):
        a = A.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c = o.int8_gemm(a, SA, B, SB, torch.bfloat16, None, None, 0, False)
        graphs.append((a, g, c))
    for i in range(4):
        for j, (a, g, c) in enumerate(graphs):
            a.copy_(A.roll(i + 5 * j, 0))
            g.replay()
        torch.cuda.synchronize()
        for a, g, c in graphs:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                want = o.int8_gemm(a, SA, B, SB, torch.bfloat16, None, None, 0, False)
            st.synchronize()
            assert torch.equal(c, want)


@pytest.mark.parametrize("M", [1, 19, 300])
@pytest.mark.parametrize("bf16", [False, True])
def test_mlp(dev, M, bf16):
    """The calls together, as a model uses them: the residual's addition and norm, two products with silu(gate) * up
    between, codes of that, the second product and its residual, against the same steps in 64 bits on the codes that
    the library made: each product within the output's rounding."""
    import ternocl_amd.torch_ops  # noqa: F401
    o = torch.ops.ternocl
    H, I = 512, 1280
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randn(s, generator=g)
    x, res, w = r(M, H).to(dt).cuda(), (3 * r(M, H)).to(dt).cuda(), (r(H) * 0.1).to(dt).cuda()
    Wu, Wg, Wd = [(r(*s) * 40).round().clamp(-127, 127).to(torch.int8).cuda() for s in ((H, I), (H, I), (I, H))]
    Su, Sg, Sd = [(torch.rand(n, generator=g) * 1e-3 + 1e-4).cuda() for n in (I, I, H)]
    h, _, q, s = o.rmsnorm(x, res, w, 1e-6, 1.0, "rows", False)
    up = o.int8_gemm(q, s, packed(Wu), Su, dt, None, None, 0, False)
    act = o.int8_gemm(q, s, packed(Wg), Sg, dt, up, None, 1, False)
    q2, s2 = o.quant_rows(act)
    y = o.int8_gemm(q2, s2, packed(Wd), Sd, dt, h, None, 2, False)
    u = torch.finfo(dt).eps / 2
    mul = lambda q, s, W, S: (q.double() @ W.double()) * S.double() * s.double()[:, None]
    hd = x.double() + res.double()
    n = hd / (hd.square().mean(1, keepdim=True) + 1e-6).sqrt() * (1 + w.double())
    # a code is half a step off at most (the step: the row's largest / 127)
    assert ((q.double() * s.double()[:, None] - n).abs() <= 0.5001 * s.double()[:, None]).all()
    close = lambda got, want, d: ((got.double() - want).abs() <= u * want.abs() + d + 2.0**-25).all()
    v = mul(q, s, Wu, Su)
    assert close(up, v, 4 * 2.0**-24 * v.abs())
    v = mul(q, s, Wg, Sg)
    a = torch.where(v <= -10, 0.0, v / (1 + torch.exp(-v))) * up.double()
    assert close(act, a, 2.0**-19 * (a.abs() + up.double().abs() * 1e-4))
    assert ((q2.double() * s2.double()[:, None] - act.double()).abs() <= 0.5001 * s2.double()[:, None]).all()
    v = mul(q2, s2, Wd, Sd) + h.double()
    assert close(y, v, 5 * 2.0**-24 * (v.abs() + 2 * h.double().abs()))


def test_norm_before_ternary_product(dev):
    """rmsnorm's groups into int2_int8_gemm: the bits of rmsnorm, quant_a and the product."""
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    o = torch.ops.ternocl
    M, K, N = 7, 512, 256
    g = torch.Generator().manual_seed(2)
    x = torch.randn((M, K), generator=g).half().cuda()
    B = torch.randint(-2**31, 2**31 - 1, (K // 16, N), generator=g, dtype=torch.int64).to(torch.int32).cuda()
    S = (torch.rand((K // 128, N), generator=g) * 0.01).half().cuda()
    h, y, q, s = o.rmsnorm(x, x, None, 1e-6, 0.0, "groups", True)
    sa, aq = o.quant_a(y)
    assert torch.equal(q, aq) and torch.equal(s[:, :M], sa[:, :M])
    assert torch.equal(o.int2_int8_gemm(q, s, B, S, None, None, 0, False), o.int2_int8_gemm(aq, sa, B, S, None, None, 0, False))


@pytest.mark.parametrize("M,K,N,postop", [(1152, 1024, 14480, 5), (2300, 1024, 7376, 0), (2560, 1024, 6784, 1), (1024, 1024, 16848, 0)])
def test_last_round_in_halves(dev, M, K, N, postop):
    """A little more than 256 tiles of 128 x 512: those past the last whole round run as two of half the width, of a
    last column of tiles that ends inside the first half too."""
    import ternocl_amd as T
    check(T, M, M, K, N, True, postop, False)


@pytest.mark.parametrize("M,K,N", [(1, 14336, 64), (5, 14336, 512), (9, 8192, 64), (24, 14336, 512), (60, 8192, 64), (64, 14336, 2048),
                                   (100, 4096, 64), (100, 14336, 512), (130, 14336, 2048), (300, 14336, 2048), (1000, 8192, 96)])
@pytest.mark.parametrize("postop", [0, 5])
def test_k_slices(dev, M, K, N, postop):
    """Shapes that split K over workgroups with a workspace, at every tile that does: whole, short and no workspace, any
    contents, the same bits."""
    import ternocl_amd as T
    nb = T.int8_gemm_ws_bytes(M, N, K)
    assert nb > T.WS_HEADER_BYTES
    A, SA, W, SB = make(M + N, M, K, N)
    g = torch.Generator().manual_seed(M)
    o = torch.randn((M, N), generator=g).half() if postop else None
    b = torch.randn(N, generator=g).half() if postop else None
    want = run(T, A, SA, W, SB, torch.float16, o, b, postop, False, ws=None)
    if postop == 0:
        assert torch.equal(want.cpu(), ((exact_sums(A, W).float() * SB) * SA[:, None]).half())
    B, C = packed(W.cuda()), torch.empty((M, N), dtype=torch.float16, device="cuda")
    a = [t if t is None else t.cuda() for t in (A, SA, SB, o, b)]
    for n in (nb, nb - 4, T.WS_HEADER_BYTES + 8 * M * N, T.WS_HEADER_BYTES):
        ws = torch.full((n + 16,), 0x5a, dtype=torch.uint8, device="cuda")
        for _ in range(2):  # (as left by another use, then as the first call leaves it)
            C.zero_()
            T.int8_gemm(a[0], a[1], B, a[2], C, a[3], a[4], M, N, K, postop, False, ws=ws[:n])
            torch.cuda.synchronize()
            assert torch.equal(C, want)
            assert (ws[n:] == 0x5a).all()


@pytest.mark.parametrize("M,K,N", [(1, 512, 256), (6, 14336, 512), (20, 1024, 256), (70, 512, 512), (300, 256, 1024), (1152, 1024, 14480)])
def test_residual_in_place(dev, M, K, N):
    """C over Other: each output is read and written by one lane."""
    import ternocl_amd as T
    A, SA, W, SB = make(M, M, K, N)
    o = torch.randn((M, N), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    a = (A.cuda(), SA.cuda(), packed(W.cuda()), SB.cuda())
    nb = T.int8_gemm_ws_bytes(M, N, K)
    for ws in (None, torch.zeros(nb, dtype=torch.uint8, device="cuda")) if nb else (None,):
        C = torch.empty_like(o)
        T.int8_gemm(*a, C, o, None, M, N, K, 2, False, ws=ws)
        D = o.clone()
        T.int8_gemm(*a, D, D, None, M, N, K, 2, False, ws=ws)
        assert torch.equal(C, D)


def test_captured_layer(dev):
    """A captured MLP with its norm, replayed on new inputs with eager work between, equals eager calls."""
    import ternocl_amd.torch_ops  # noqa: F401
    o = torch.ops.ternocl
    M, H, I = 5, 1024, 2048
    g = torch.Generator("cuda").manual_seed(4)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)
    x, res, w = r(M, H).bfloat16(), r(M, H).bfloat16(), torch.rand(H, device="cuda", generator=g)
    Ws = [packed((r(*s) * 40).round().clamp(-127, 127).to(torch.int8)) for s in ((H, I), (H, I), (I, H))]
    Ss = [torch.rand(n, device="cuda", generator=g) * 1e-3 for n in (I, I, H)]

    def layer():
        h, y, q, s = o.rmsnorm(x, res, w, 1e-6, 0.0, "rows", True)
        up = o.int8_gemm(q, s, Ws[0], Ss[0], torch.bfloat16, None, None, 0, False)
        act = o.int8_gemm(q, s, Ws[1], Ss[1], torch.bfloat16, up, None, 1, False)
        q2, s2 = o.quant_rows(act)
        return h, y, q, s, act, o.int8_gemm(q2, s2, Ws[2], Ss[2], torch.bfloat16, h, None, 2, False)

    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for i in range(4):
        x.copy_(r(M, H))
        res.copy_(r(M, H))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, layer()))
