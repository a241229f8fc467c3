"""int8_gemm on each tile that it compiles, with and without K slices, with weights past the last-level
cache, at every epilogue and type.

The tile of a size is chosen by a fitted model, so each case names its tile and the tests without a GPU
assert that it runs there and that no tile is left out.  Gold: sums of whole numbers in 64-bit floats
(exact).  Without an epilogue outputs are the sums' three roundings in order, bit for bit; with one,
three of those, one of each addition or product, and the output's own.  The sigmoid is 1 / (1 + 2^(-x log2 e)) in
fp32: the exponent's constant and product are off by 1.5 2^-24 of it, 15 2^-24 of the power for the -10 < x where
the power matters; 2^x and the reciprocal by an ulp each (4 2^-24), the sum by a rounding: 20 2^-24 in all."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

# (rows, columns, waves over K, activations through LDS) of every tile
EVERY = {(16, 16, 4, False), (16, 32, 4, False), (16, 16, 4, True), (16, 32, 4, True), (16, 64, 4, True), (32, 32, 4, True),
         (32, 64, 4, True), (32, 128, 1, True), (32, 128, 2, True), (64, 128, 1, True), (64, 128, 2, True), (64, 256, 1, True),
         (128, 256, 1, True), (128, 512, 1, True)}

# (M, K, N): its tile and slices, without (one slice) or with a workspace
WHOLE = {
    (1, 256, 16): (16, 16, 4, 1, False), (3, 12928, 848): (16, 16, 4, 1, False),
    (1, 256, 4112): (16, 32, 4, 1, False), (7, 640, 4112): (16, 32, 4, 1, False),
    (5, 256, 16): (16, 16, 4, 1, True), (33, 1152, 1040): (16, 16, 4, 1, True),
    (12, 384, 9440): (16, 32, 4, 1, True), (47, 256, 1744): (16, 32, 4, 1, True),
    (47, 1280, 3856): (16, 64, 4, 1, True), (48, 5120, 5120): (16, 64, 4, 1, True),
    (49, 256, 16): (32, 32, 4, 1, True), (59, 1152, 2064): (32, 32, 4, 1, True),
    (97, 512, 16): (32, 64, 4, 1, True), (130, 640, 1040): (32, 64, 4, 1, True),
    (97, 256, 16): (32, 128, 1, 1, True), (367, 256, 7056): (32, 128, 1, 1, True),
    (550, 1536, 1104): (32, 128, 2, 1, True), (2094, 1280, 208): (32, 128, 2, 1, True),
    (128, 4096, 14336): (64, 128, 1, 1, True), (2402, 896, 400): (64, 128, 1, 1, True),
    (139, 2432, 9680): (64, 128, 2, 1, True), (2079, 1024, 400): (64, 128, 2, 1, True),
    (246, 8448, 8896): (64, 256, 1, 1, True), (2448, 256, 1168): (64, 256, 1, 1, True),
    (2450, 384, 2464): (128, 256, 1, 1, True), (2437, 256, 4128): (128, 512, 1, 1, True),
}
SLICED = {
    (5, 6912, 16): (16, 16, 4, 3, False), (3, 12928, 848): (16, 16, 4, 2, False), (1, 40960, 2464): (16, 32, 4, 3, False),
    (6, 7168, 16): (16, 16, 4, 3, True), (17, 11264, 160): (16, 16, 4, 3, True), (37, 12288, 688): (16, 32, 4, 3, True),
    (4, 11776, 8240): (16, 64, 4, 3, True), (59, 5760, 432): (32, 32, 4, 3, True), (105, 2944, 80): (32, 64, 4, 3, True),
    (66, 11776, 8288): (32, 128, 1, 2, True), (2091, 9088, 80): (32, 128, 2, 3, True), (103, 11776, 8208): (64, 128, 1, 3, True),
    (2049, 9984, 208): (64, 128, 2, 3, True), (2096, 12800, 400): (64, 256, 1, 3, True), (293, 14336, 6896): (128, 256, 1, 3, True),
    (537, 13824, 7264): (128, 512, 1, 3, True),
}
# more than 10^8 weights: loaded past the cache, by the tiles of few rows
FAR = {
    (1, 130944, 784): (16, 16, 4, 1, False), (1, 13056, 7664): (16, 32, 4, 1, False), (17, 130944, 784): (16, 16, 4, 1, True),
    (7, 5888, 17040): (16, 32, 4, 1, True), (16, 5120, 34816): (16, 64, 4, 1, True), (20, 12288, 8336): (32, 32, 4, 1, True),
}
FAR_SLICED = {(5, 130944, 784): (16, 32, 4, 8, False), (40, 130944, 784): (32, 32, 4, 5, True), (1, 12160, 8224): (16, 64, 4, 3, True)}
CASES = [(s, t) for d in (WHOLE, SLICED, FAR, FAR_SLICED) for s, t in d.items()]


def ws_bytes(T, M, K, N, tile):
    return T.int8_gemm_ws_bytes(M, N, K) if tile[3] > 1 else 0


@pytest.mark.parametrize("shape,tile", CASES)
def test_tile_of(shape, tile):
    import ternocl_amd as T
    M, K, N = shape
    assert T.kw_tile_of(4, M, N, K, ws_bytes=ws_bytes(T, M, K, N, tile)) == tile


def test_every_tile():
    name = lambda t: t[:3] + t[4:]
    assert {name(t) for t in WHOLE.values()} == EVERY
    assert {name(t) for t in SLICED.values()} == EVERY
    assert {name(t) for t in FAR.values()} == {t for t in EVERY if t[2] == 4 and t[:2] != (32, 64)}
    assert all(t[3] > 1 for t in list(SLICED.values()) + list(FAR_SLICED.values()))
    assert all(K * N > 10**8 for _, K, N in list(FAR) + list(FAR_SLICED))


def test_tile_of_refusals():
    import ternocl_amd as T
    for M, K, N in ((0, 256, 16), (1, 64, 16), (1, 200, 16), (1, 256, 8), (1, 256, 24), (1, 1 << 17, 16), (1, 256, (1 << 26) + 16)):
        assert T.kw_tile_of(4, M, N, K) is None


@pytest.mark.gpu
@pytest.mark.parametrize("shape,tile", CASES)
def test_tile(dev, shape, tile):
    """Every epilogue and type, a workspace of any contents where K is sliced."""
    import ternocl_amd as T
    M, K, N = shape
    nb = ws_bytes(T, M, K, N, tile)
    assert T.kw_tile_of(4, M, N, K, ws_bytes=nb) == tile
    g = torch.Generator("cuda").manual_seed(M + K + N)
    A = torch.randint(-128, 128, (M, K), dtype=torch.int8, device="cuda", generator=g)
    B = torch.randint(-128, 128, (K // 16, N, 16), dtype=torch.int8, device="cuda", generator=g)
    SA = torch.rand(M, device="cuda", generator=g) * 0.02 + 0.01
    SB = (torch.rand(N, device="cuda", generator=g) + 0.5) * (0.02 / K**0.5)  # (products of about 1)
    sums = A.double() @ B.transpose(1, 2).reshape(K, N).double()
    v32 = (sums.float() * SB) * SA[:, None]
    acc = sums * SB.double() * SA.double()[:, None]
    d = 3.01 * 2.0**-24 * acc.abs()
    sg = torch.where(acc <= -10, 0.0, 1 / (1 + torch.exp(-acc)))
    # (a product near -10 may fall on either side of the sigmoid's cut)
    cut = torch.where((acc + 10).abs() <= d, 5e-5, 0.0)
    ws = torch.full((nb,), 0x5a, dtype=torch.uint8, device="cuda") if nb else None
    for dt in (torch.float16, torch.bfloat16):
        o = torch.randn((M, N), device="cuda", generator=g).to(dt)
        for f32 in (False, True):
            ct = torch.float32 if f32 else dt
            b = torch.randn(N, device="cuda", generator=g).to(ct)
            od, bd, u = o.double(), b.double(), torch.finfo(ct).eps / 2
            for p in range(6):
                C = torch.full((M + 1, N), 7.0, dtype=ct, device="cuda")
                T.int8_gemm(A, SA, B, SB, C, o if p in (1, 2, 5) else None, b if p in (3, 5) else None, M, N, K, p, f32, ws=ws)
                assert (C[M] == 7.0).all()  # the row behind the last stays as it was
                C = C[:M]
                if p == 0:
                    assert torch.equal(C, v32.to(ct)), (dt, f32)
                    continue
                if p == 1:
                    want, e = acc * sg * od, (1.1 * d + 22 * 2.0**-24 * acc.abs() * sg + 10 * cut) * od.abs()
                elif p == 4:
                    want, e = sg, d + 20 * 2.0**-24 * sg + cut
                else:
                    want, m = acc, acc.abs()
                    for on, t in ((p in (3, 5), bd), (p in (2, 5), od)):
                        want, m = (want + t, m + t.abs()) if on else (want, m)
                    e = d + 2 * 2.0**-24 * m
                over = (C.double() - want).abs() - (u * want.abs() + e * (1 + u) + (2.0**-25 if ct == torch.float16 else 0.0))
                assert not (over > 0).any(), (dt, f32, p, over.max().item())
