"""int4_gemm on the GPU against the product in 64 bits, at every type, group, epilogue and engine.

Tolerance: one rounding of the output (eps / 2 of its type, relative) and D roundings of fp32 sums, D 2^-24
of sum_k |a| (|q - z| + 32) |s|.  D = 160 + K / 64 covers the longest chain of additions a term goes
through in any engine (the plain kernel: 128 in a group, K / 128 groups; the matrix cores: 16 in a group,
K / 32 groups, 16 waves and slices); the 32 is for engines that multiply codes with an offset of up to 32
and take it off again.  fp16 activations below 2^-11 of their group's largest, bf16 below 2^-14, are
rounded to 2^-22 of that: within the same bound."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import off16

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def make(seed, M, K, N, group, bf16, zero, dist="normal"):
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(seed)
    A = torch.randn((M, K), generator=g)
    if dist == "positive":
        A = A.abs()
    elif dist == "outliers":  # a few channels 300 times the rest
        A[:, torch.randint(0, K, (3,), generator=g)] *= 300
    elif dist == "zero":
        A[:, :K // 2] = 0
    W = torch.randint(-8, 8, (K, N), generator=g, dtype=torch.int8)
    S = torch.rand((K // group, N), generator=g) * 0.015 + 0.005
    Z = torch.randn((K // group, N), generator=g) * 3 if zero else None
    c = lambda t: None if t is None else t.to(dt)
    return c(A), W, c(S), c(Z), dt


def gold(A, W, S, Z, group, other, bias, postop):
    K = A.shape[1]
    q = W.double()
    w = q if Z is None else q - Z.double().repeat_interleave(group, 0)
    s = S.double().repeat_interleave(group, 0)
    acc = A.double() @ (w * s)
    mag = A.double().abs() @ ((w.abs() + 32) * s.abs())
    d = (160 + K / 64) * 2.0**-24 * mag
    if postop in (1, 4):
        sg = torch.where(acc <= -10, 0.0, 1 / (1 + torch.exp(-acc)))
        # (the epilogue's sigmoid is good to about 2^-20; a sum near -10 may fall on either side of its cut)
        cut = torch.where((acc + 10).abs() <= d, 5e-5, 0.0)
        if postop == 4:
            return sg, d + 2.0**-20 + cut
        o = other.double()
        return acc * sg * o, (1.1 * d + 2.0**-20 * acc.abs() * sg + 10 * cut) * o.abs()
    v, m = acc, acc.abs()
    if postop in (3, 5):
        v, m = v + bias.double(), m + bias.double().abs()
    if postop in (2, 5):
        v, m = v + other.double(), m + other.double().abs()
    return v, d + 2 * 2.0**-24 * m


def run(T, A, W, S, Z, group, other, bias, postop, f32, ws=True, move=None):
    M, K = A.shape
    N = W.shape[1]
    dev = lambda t: None if t is None else t.cuda()
    B = torch.from_numpy(T.int4_pack(W.numpy()).view(np.int32)).cuda()
    a = dict(A=dev(A), S=dev(S), Z=dev(Z), other=dev(other), bias=dev(bias))
    C = torch.full((M + 2, N), 7.0, dtype=torch.float32 if f32 else A.dtype, device="cuda")
    if move:
        for k in move:
            if a[k] is not None:
                a[k] = off16(a[k])
    nb = T.int4_gemm_ws_bytes(M, N, K, group)
    w = torch.randint(0, 255, (nb,), dtype=torch.uint8, device="cuda") if nb and ws else None
    T.int4_gemm(a["A"], B, a["S"], a["Z"], C, a["other"], a["bias"], M, N, K, group, postop, f32, ws=w)
    torch.cuda.synchronize()
    assert (C[M:] == 7.0).all()  # rows behind the last stay as they were
    return C[:M]


def check(T, seed, M, K, N, group, bf16, zero, postop, f32, dist="normal", **kw):
    A, W, S, Z, dt = make(seed, M, K, N, group, bf16, zero, dist)
    g = torch.Generator().manual_seed(seed + 1)
    other = torch.randn((M, N), generator=g).to(dt) if postop in (1, 2, 5) else None
    bias = torch.randn(N, generator=g).to(torch.float32 if f32 else dt) if postop in (3, 5) else None
    got = run(T, A, W, S, Z, group, other, bias, postop, f32, **kw).cpu().double()
    want, d = gold(A, W, S, Z, group, other, bias, postop)
    u = torch.finfo(torch.float32 if f32 else dt).eps / 2
    tiny = 0.0 if f32 or bf16 else 2.0**-25  # (fp16 subnormals)
    err = (got - want).abs() - (u * want.abs() + d * (1 + u) + tiny)
    assert not (err > 0).any() and torch.isfinite(got).all(), (err.max().item(), (err > 0).sum().item())
    return got


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows(dev, M, bf16, group):
    import ternocl_amd as T
    check(T, 11 * M + group, M, 512, 208, group, bf16, M % 2 == 0, 0, True)


@pytest.mark.parametrize("M", [1, 6, 40])
@pytest.mark.parametrize("postop", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("bf16,f32", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(dev, M, postop, bf16, f32):
    import ternocl_amd as T
    check(T, 100 + postop, M, 384, 144, 128, bf16, True, postop, f32)


@pytest.mark.parametrize("K,N", [(128, 16), (128, 4096), (256, 32), (640, 48), (1152, 16), (4096, 16), (5376, 80),
                                 (14336, 64), (17408, 32), (40960, 16)])
@pytest.mark.parametrize("M", [1, 4, 8, 24, 130])
def test_shapes(dev, K, N, M):
    import ternocl_amd as T
    check(T, K + N + M, M, K, N, 128 if K % 256 else 64, (K // 128) % 2 == 0, False, 0, True)


@pytest.mark.parametrize("M,K,N,group", [(1, 4096, 4096, 128), (4, 1024, 16400, 128), (8, 4096, 6144, 32), (2, 2048, 40000, 64),
                                         (24, 14336, 1024, 128), (300, 1024, 1552, 32), (700, 512, 2064, 64),
                                         (1000, 256, 4112, 128), (333, 512, 11024, 32), (130, 1152, 16400, 64)])
@pytest.mark.parametrize("bf16", [False, True])
def test_real_sizes(dev, M, K, N, group, bf16):
    import ternocl_amd as T
    check(T, M, M, K, N, group, bf16, True, 0, False)


@pytest.mark.parametrize("dist", ["positive", "outliers", "zero"])
@pytest.mark.parametrize("M", [1, 8, 33])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("zero", [False, True])
def test_distributions(dev, dist, M, bf16, zero):
    import ternocl_amd as T
    check(T, 5, M, 1024, 96, 128, bf16, zero, 0, True, dist)


@pytest.mark.parametrize("M", [1, 9, 70])
@pytest.mark.parametrize("move", [("A",), ("S",), ("Z",), ("other",), ("bias",)])
def test_unaligned_operands(dev, M, move):
    import ternocl_amd as T
    check(T, 9, M, 256, 48, 64, True, True, 5, False, move=move)


@pytest.mark.parametrize("M,K,N", [(1, 14336, 512), (4, 14336, 256), (24, 14336, 256), (48, 7040, 512), (8, 28672, 128)])
def test_workspace(dev, M, K, N):
    """With its workspace (any contents), without one, and twice: the same within the tolerance, and twice the
    same bits."""
    import ternocl_amd as T
    a = check(T, 3, M, K, N, 128, True, True, 2, False)
    b = check(T, 3, M, K, N, 128, True, True, 2, False)
    assert torch.equal(a, b)
    check(T, 3, M, K, N, 128, True, True, 2, False, ws=False)


@pytest.mark.parametrize("M", [1, 8, 20])
@pytest.mark.parametrize("bf16", [False, True])
def test_not_finite_rows(dev, M, bf16):
    """A row with an infinity or a NaN is not finite; the others are as without it."""
    import ternocl_amd as T
    A, W, S, Z, dt = make(2, M, 512, 64, 128, bf16, False)
    W[W == 0] = 3
    clean = run(T, A, W, S, Z, 128, None, None, 0, True)
    for bad in (float("inf"), float("nan")):
        X = A.clone()
        X[M // 2, 77] = bad
        got = run(T, X, W, S, Z, 128, None, None, 0, True)
        assert not torch.isfinite(got[M // 2]).any()
        keep = [m for m in range(M) if m != M // 2]
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("M", [1, 8, 20])
def test_extremes(dev, M):
    """Activations at the ends of bf16's range and rows of zeros."""
    import ternocl_amd as T
    for scale in (2.0**100, 2.0**-120, 0.0):
        A, W, S, Z, dt = make(4, M, 256, 32, 128, True, False)
        A = (A.float() * scale).to(dt)
        got = run(T, A, W, S, None, 128, None, None, 0, True).cpu().double()
        want, d = gold(A, W, S, None, 128, None, None, 0)
        # (results and partial sums below 2^-126 may be flushed: 2^-126 for each of the 256 terms, times 32)
        assert ((got - want).abs() <= 2.0**-23 * want.abs() + d + 2.0**-113).all()


@pytest.mark.parametrize("M", [1, 8, 20, 300])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_largest_scales(dev, M, zero, group):
    """Scales near the end of bf16's range: sums that they bring back into fp32 are no infinities on the way."""
    import ternocl_amd as T
    A, W, S, Z, dt = make(6, M, 256, 272, group, True, zero)
    A, S = (A.double() * 2.0**-100).to(dt), (S.double() * 2.0**131).to(dt)
    got = run(T, A, W, S, Z, group, None, None, 0, True).cpu().double()
    want, d = gold(A, W, S, Z, group, None, None, 0)
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + d).all()


@pytest.mark.parametrize("M", [1, 4, 24, 200])
def test_graph_and_stream(dev, M):
    """Captured on a side stream and replayed with new inputs between eager calls, its workspace reused."""
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    op = torch.ops.ternocl.int4_gemm
    K, N = 7168, 512
    A, W, S, Z, dt = make(8, M, K, N, 64, True, True)
    B = torch.from_numpy(T.int4_pack(W.numpy()).view(np.int32)).cuda()
    A, S, Z = A.cuda(), S.cuda(), Z.cuda()
    other = torch.randn(M, N, device="cuda").to(dt)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        warm = op(A, B, S, Z, 64, other, None, 2, False)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = op(A, B, S, Z, 64, other, None, 2, False)
    torch.cuda.synchronize()
    for i in range(4):
        A.copy_(torch.randn(M, K).to(dt))
        want = op(A, B, S, Z, 64, other, None, 2, False)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert warm.shape == out.shape


def test_ops_match_direct_calls(dev):
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    A, W, S, Z, dt = make(8, 3, 256, 64, 32, False, True)
    B = torch.from_numpy(T.int4_pack(W.numpy()).view(np.int32)).cuda()
    got = torch.ops.ternocl.int4_gemm(A.cuda(), B, S.cuda(), Z.cuda(), 32, None, None, 0, False)
    assert torch.equal(got, run(T, A, W, S, Z, 32, None, None, 0, False))
    assert torch.ops.ternocl.int4_gemm(A[:0].cuda(), B, S.cuda(), None, 32, None, None, 0, False).shape == (0, 64)
    with pytest.raises(RuntimeError):
        torch.ops.ternocl.int4_gemm(A.cuda(), B, S.cuda(), None, 32, None, None, 3, False)  # no bias
    torch.library.opcheck(torch.ops.ternocl.int4_gemm.default, (A.cuda(), B, S.cuda(), Z.cuda(), 32, None, None, 0, False),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("M", [2, 12])
def test_offsets_past_32_bits(dev, M):
    """Weights of more than 2^32 bytes: the columns at both ends."""
    import ternocl_amd as T
    K, N, group = 4096, (1 << 21) + 48 * 1024, 128
    A, _, _, _, dt = make(5, M, K, 16, group, True, False)
    A = A.cuda()
    B = torch.randint(-2**31, 2**31 - 1, (K // 32, N, 4), dtype=torch.int32, device="cuda")
    S = (torch.rand((K // group, N), device="cuda") * 0.01 + 0.005).to(dt)
    assert B.numel() * 4 > 2**32
    C = torch.empty((M, N), dtype=torch.float32, device="cuda")
    T.int4_gemm(A, B, S, None, C, None, None, M, N, K, group, 0, True)
    torch.cuda.synchronize()
    for n0 in (0, N // 2, N - 64):
        cols = slice(n0, n0 + 64)
        W = T.int4_unpack(B[:, cols].contiguous().cpu().numpy().view(np.uint32), K)
        want, d = gold(A.cpu(), torch.from_numpy(W), S[:, cols].cpu(), None, group, None, None, 0)
        assert ((C[:, cols].cpu().double() - want).abs() <= 2.0**-24 * want.abs() + d).all()


@pytest.mark.parametrize("M", [1, 4, 8, 20, 300])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_largest_zero_points(dev, M, group):
    """Zero points up to bf16's largest: rows and groups of zeros stay zero, sums within fp32 stay finite."""
    import ternocl_amd as T
    A, W, S, Z, dt = make(7, M, 256, 272, group, True, True)
    g = torch.Generator().manual_seed(8)
    Z = (Z.sign() * 2.0**124 * (1 + 14 * torch.rand(Z.shape, generator=g))).to(dt)
    Z[:, :8] = torch.finfo(dt).max
    A = (A.double() * 2.0**-60).to(dt)
    A[0] = 0
    A[:, 128:] = 0
    got = run(T, A, W, S, Z, group, None, None, 0, True).cpu().double()
    want, d = gold(A, W, S, Z, group, None, None, 0)
    assert (got[0] == 0).all()
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + d).all()


@pytest.mark.parametrize("M", [1, 4, 8, 20, 300])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_largest_sums(dev, M, group):
    """Sums in the last octaves of fp32's range are no infinities at any number of rows (bf16; positive terms, so
    that no partial sum is larger)."""
    import ternocl_amd as T
    A, W, S, _, dt = make(9, M, 256, 272, group, True, False, "positive")
    W = W.abs().clamp(1, 7)
    A, S = (A.double() * 2.0**60).to(dt), (S.double() * 2.0**62.5).to(dt)
    got = run(T, A, W, S, None, group, None, None, 0, True).cpu().double()
    want, d = gold(A, W, S, None, group, None, None, 0)
    assert 2.0**125 < want.max() < 2.0**127.5
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + d).all()


@pytest.mark.parametrize("M", [1, 8])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("exp", [-110, -124, -130])
def test_smallest_activations(dev, M, zero, exp):
    """The decode rows' fixed point at the lower end of bf16, subnormal values among the activations."""
    import ternocl_amd as T
    A, W, S, Z, dt = make(10, M, 256, 32, 128, True, zero)
    A, S = (A.double() * 2.0**exp).to(dt), (S.double() * 2.0**100).to(dt)
    got = run(T, A, W, S, Z, 128, None, None, 0, True).cpu().double()
    want, d = gold(A, W, S, Z, 128, None, None, 0)
    # (a group's sum is a multiple of 2^-149 within half a unit, two of them with Z: times S, two groups)
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + d + 4 * 2.0**-149 * S.double().max()).all()


@pytest.mark.parametrize("M", [1, 4, 8, 9, 33, 200])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_largest_activation_on_zero_codes(dev, M, bf16, group):
    """One activation of each group far above the others, on weights of 0.  Up to 8 rows: each activation within 2^-22 of
    its group's largest, the exact ones (2^-14 of it and more, and 0) as they are.  More rows at fp16: nothing is lost."""
    import ternocl_amd as T
    K, N = 512, 96
    A, W, S, _, dt = make(12, M, K, N, group, bf16, False)
    g = torch.Generator().manual_seed(13)
    far = 2.0 ** -torch.randint(4, 31, (M, K // group, 1), generator=g)  # (of the largest, by row and group)
    A = (A.view(M, K // group, group) * 1000 * far).reshape(M, K)
    A[:, 5::group] = 20000.0
    A = A.to(dt)
    W[5::group] = 0
    got = run(T, A, W, S, None, group, None, None, 0, True).cpu().double()
    a, w = A.double(), W.double() * S.double().repeat_interleave(group, 0)
    want = a @ w
    d = (160 + K / 64) * 2.0**-24 * (a.abs() @ w.abs())
    if M <= 8:
        step = 2.0 ** (a.abs().view(M, K // group, group).amax(2).log2().floor() - 21)
        off = torch.where(a % step.repeat_interleave(group, 1) == 0, 0.0, step.repeat_interleave(group, 1) / 2)
        d += off @ w.abs()
    elif bf16:  # (codes with an offset of 24, the largest activations' products with it taken off again)
        d += (160 + K / 64) * 2.0**-24 * 32 * (a.abs() @ S.double().repeat_interleave(group, 0))
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + d).all()
