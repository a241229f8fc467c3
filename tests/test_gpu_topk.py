"""moe_topk on the GPU against the definition in 64 bits: ids equal, weights within the two roundings of the
output (fp32, then its type: eps / 2 and 2^-24, relative) and 2^-40 for the fp64 exponentials."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
NAMES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def gold(logits, bias, topk, score, n_group, topk_group, group_best, renorm, scale):
    """Row by row, in Python's own order of comparison: (-value, index)."""
    ids, ws = [], []
    per = logits.shape[1] // n_group
    b = [0.0] * logits.shape[1] if bias is None else bias.double().tolist()
    for row in logits.double().tolist():
        if score == "softmax":
            mx = max(row)
            ex = [0.0 if x == -math.inf else math.exp(x - mx) for x in row]
            tot = math.fsum(ex)
            s = [e / tot if tot else 0.0 for e in ex]
        else:
            s = [1 / (1 + math.exp(-x)) if x > -700 else 0.0 for x in row]
        v = [-math.inf if x == -math.inf else si + bi for x, si, bi in zip(row, s, b)]
        order = [-math.inf if x == -math.inf else x for x in row] if bias is None else v
        pool = range(len(row))
        if topk_group < n_group:
            src = v if group_best == 2 or bias is not None else order
            gv = []
            for g in range(n_group):
                top = [x for x in sorted(src[g * per:(g + 1) * per], reverse=True)[:group_best] if x != -math.inf]
                gv.append(sum(top) if top else -math.inf)
            kept = sorted(range(n_group), key=lambda g: (-gv[g], g))[:topk_group]
            pool = [e for e in pool if e // per in kept]
        pick = sorted((e for e in pool if order[e] != -math.inf and v[e] != -math.inf), key=lambda e: (-order[e], e))[:topk]
        w = [s[e] for e in pick]
        if renorm:
            t = math.fsum(w)
            w = [x / t if t else 0.0 for x in w]
        ids.append(pick + [-1] * (topk - len(pick)))
        ws.append([x * scale for x in w] + [0.0] * (topk - len(pick)))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(ws, dtype=torch.float64)


def check(T, logits, bias, topk, wt, score="softmax", n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0, ld=None):
    Tk, E = logits.shape
    L = logits.cuda()
    if ld:
        buf = torch.full((Tk, ld), 99.0, dtype=logits.dtype, device="cuda")
        buf[:, :E] = L
        L = buf
    ids = torch.full((Tk + 1, topk), 77, dtype=torch.int32, device="cuda")
    RW = torch.full((Tk + 1, topk), 7.0, dtype=NAMES[wt], device="cuda")
    T.moe_topk(L, None if bias is None else bias.cuda(), ids, RW, Tk, E, topk, score, n_group, topk_group, group_best, renorm,
               scale, ld=ld)
    torch.cuda.synchronize()
    assert (ids[Tk] == 77).all() and (RW[Tk] == 7).all()
    want, w = gold(logits, bias, topk, score, n_group, topk_group, group_best, renorm, scale)
    assert torch.equal(ids[:Tk].cpu(), want)
    got = RW[:Tk].cpu().double()
    u = torch.finfo(NAMES[wt]).eps / 2
    tiny = {"f16": 2.0**-25, "bf16": 2.0**-126, "f32": 2.0**-126}[wt]  # (subnormal weights)
    assert ((got - w).abs() <= (u + 2.0**-24 + 2.0**-40) * w.abs() + tiny).all()


def logits_of(seed, Tk, E, lt, sigma=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((Tk, E), generator=g) * sigma).to(NAMES[lt]), torch.randn(E, generator=g) * 0.1


@pytest.mark.parametrize("E,topk", [(1, 1), (2, 2), (3, 1), (8, 2), (17, 5), (60, 4), (64, 8), (65, 8), (100, 10), (128, 8),
                                    (200, 1), (256, 8), (257, 64), (384, 6), (512, 10), (512, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_experts(dev, E, topk, score, biased):
    import ternocl_amd as T
    for i, lt in enumerate(NAMES):
        x, b = logits_of(E + topk, 37, E, lt)
        check(T, x, b if biased else None, topk, ("bf16", "f16", "f32")[i], score, renorm=i != 1, scale=(1.0, 2.5, 1.0)[i])


@pytest.mark.parametrize("Tk", [1, 2, 3, 4, 5, 63, 1001])
def test_tokens(dev, Tk):
    import ternocl_amd as T
    x, b = logits_of(Tk, Tk, 128, "bf16")  # (many equal logits)
    check(T, x, None, 8, "bf16")
    check(T, x, b, 8, "f32", "sigmoid", 8, 3, 2)


@pytest.mark.parametrize("Tk", [4095, 4097])
@pytest.mark.parametrize("E,n_group,topk_group,group_best", [(256, 8, 4, 2), (160, 5, 2, 2), (512, 16, 3, 1), (60, 15, 7, 1),
                                                             (128, 4, 2, 2), (96, 3, 2, 1), (64, 1, 1, 1)])
def test_many_tokens(dev, Tk, E, n_group, topk_group, group_best):
    """Enough tokens for several to share a wave, their scores close now and then."""
    import ternocl_amd as T
    x, b = logits_of(Tk + E, Tk, E, "f32")
    x[::97, ::3] = x[::97, :1] + 2.0**-23 * torch.arange(len(range(0, E, 3)))
    x[5, 7], x[9, 1:] = -math.inf, -math.inf
    check(T, x, b, 6, "f32", "sigmoid", n_group, topk_group, group_best, True, 2.5)
    check(T, x, None, 6, "bf16", "softmax", n_group, topk_group, group_best, False)
    if topk_group * (E // n_group) >= 20:
        check(T, x[:500], b, 14, "f32", "sigmoid", n_group, topk_group, group_best)
        check(T, x[:500], b, 15, "f32", "sigmoid", n_group, topk_group, group_best)
        check(T, x[:500], None, 16, "f32", "softmax", n_group, topk_group, group_best)
        check(T, x[:500], None, 17, "f32", "softmax", n_group, topk_group, group_best)


@pytest.mark.parametrize("biased", [False, True])
def test_equal_and_uneven_rows(dev, biased):
    """Rows of one value, of few, and with all large values in the same places of every 16."""
    import ternocl_amd as T
    g = torch.Generator().manual_seed(4)
    x = torch.zeros(40, 256)
    x[10:20] = torch.randint(0, 3, (10, 256), generator=g).float()
    x[20:30] = torch.randn(10, 256, generator=g)
    x[20:30, 3::16] += 8
    x[30:] = torch.randn(10, 256, generator=g) - 300
    b = torch.randint(-1, 2, (256,), generator=g) * 0.25 if biased else None
    for score in ("softmax", "sigmoid"):
        check(T, x, b, 8, "f32", score)
        check(T, x, b, 8, "f32", score, 8, 2, 1)


@pytest.mark.parametrize("E,n_group,topk_group", [(64, 8, 4), (64, 8, 8), (256, 8, 4), (160, 8, 3), (512, 64, 7), (48, 3, 1),
                                                  (64, 64, 32), (126, 9, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("group_best", [1, 2])
def test_groups(dev, E, n_group, topk_group, score, biased, group_best):
    import ternocl_amd as T
    if group_best > E // n_group:
        pytest.skip("a group of one expert")
    x, b = logits_of(E + n_group, 41, E, "f32")
    check(T, x, b if biased else None, min(6, topk_group * (E // n_group)), "f32", score, n_group, topk_group, group_best, True, 2.5)


@pytest.mark.parametrize("E,n_group,topk_group", [(392, 2, 1), (418, 2, 1), (330, 3, 2), (510, 6, 2), (126, 2, 1), (34, 2, 1),
                                                  (306, 17, 5), (320, 64, 9), (500, 50, 30), (512, 1, 1), (91, 1, 1), (60, 1, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_wide_groups_and_many_choices(dev, E, n_group, topk_group, biased):
    """Groups of no power of two, a lane's part of each; lists of nearly as many choices as lanes."""
    import ternocl_amd as T
    x, b = logits_of(E, 103, E, "f32")
    b = b if biased else None
    for score in ("softmax", "sigmoid"):
        for topk in (13, 14, 15, 16):
            check(T, x, b, topk, "f32", score, n_group, topk_group, 1 + topk % 2, topk % 3 == 0)
    y = x.half().float() * 4  # (some equal)
    check(T, y, b, 15, "bf16", "softmax", n_group, topk_group, 2, False)
    y[::5] = y[::5].round()  # (many)
    check(T, y, b, 15, "f32", "sigmoid", n_group, topk_group, 1)


def test_close_scores(dev):
    """Scores closer than fp32 tells apart are ordered as in 64 bits; equal ones by index."""
    import ternocl_amd as T
    g = torch.Generator().manual_seed(1)
    x = torch.full((64, 96), 3.0) + torch.randint(0, 4, (64, 96), generator=g) * 2.0**-22
    check(T, x, None, 12, "f32")
    check(T, x, None, 12, "f32", "sigmoid")
    check(T, x, torch.randint(0, 3, (96,), generator=g) * 2.0**-25, 12, "f32", "sigmoid", 6, 3, 1)
    check(T, torch.zeros(3, 40), None, 5, "f32")
    check(T, torch.zeros(3, 40), torch.zeros(40), 5, "f32", "sigmoid", 4, 2, 2)
    z = torch.zeros(2, 40)
    z[:, ::2] = -0.0
    check(T, z, None, 5, "f32")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_masks(dev, score, biased):
    """Experts at -inf are never chosen; rows with few or none left end in -1 and 0; the type's lowest value
    is a value like any other."""
    import ternocl_amd as T
    x, b = logits_of(3, 6, 64, "f32")
    x[0] = -math.inf
    x[1, 5:] = -math.inf
    x[2, :60] = -math.inf
    x[3] = torch.finfo(torch.float32).min
    x[4, 1:] = torch.finfo(torch.float32).min
    b = b if biased else None
    check(T, x, b, 8, "f32", score)
    check(T, x, b, 8, "bf16", score, renorm=False)
    check(T, x[[0, 1, 2, 5]], b, 8, "f32", score, 8, 2, 2)
    if biased:
        b2 = b.clone()
        b2[7:] = -math.inf
        check(T, x[5:], b2, 8, "f32", score)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite(dev, bad):
    """A NaN (softmax: an infinity too) makes its row's weights NaN and no other row's."""
    import ternocl_amd as T
    x, _ = logits_of(3, 3, 64, "f32")
    x[1, 9] = bad
    ids = torch.empty((3, 4), dtype=torch.int32, device="cuda")
    w = torch.empty((3, 4), device="cuda")
    for renorm in (False, True):
        T.moe_topk(x.cuda(), None, ids, w, 3, 64, 4, "softmax", renorm=renorm)
        assert torch.isnan(w[1]).all() and ids[1, 0] == 9 and torch.isfinite(w[[0, 2]]).all()
        assert len(set(ids[1].tolist())) == 4
        T.moe_topk(x.cuda(), None, ids, w, 3, 64, 4, "sigmoid", renorm=renorm)
        assert ids[1, 0] == 9 and torch.isfinite(w[[0, 2]]).all()
        if bad != bad:
            assert torch.isnan(w[1, 0]) and (torch.isnan(w[1]).all() if renorm else torch.isfinite(w[1, 1:]).all())


def test_pitch(dev):
    import ternocl_amd as T
    x, b = logits_of(3, 9, 60, "bf16")
    check(T, x, b, 6, "f16", ld=61)
    x, b = logits_of(3, 9, 128, "f32")
    check(T, x, None, 6, "f16", ld=131)


def test_op_graph_and_stream(dev):
    import ternocl_amd as T
    import ternocl_amd.torch_ops  # noqa: F401
    op = torch.ops.ternocl.moe_topk
    x = torch.randn(33, 256, device="cuda")
    b = torch.randn(256, device="cuda") * 0.1
    args = (8, torch.bfloat16, "sigmoid", 8, 4, 2, True, 2.5)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        op(x, b, *args)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ids, w = op(x, b, *args)
    for _ in range(3):
        x.normal_()
        i2, w2 = op(x, b, *args)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, i2) and torch.equal(w, w2)
    v = x[:, :128]  # rows with a pitch
    i1, w1 = op(v, None, 4, torch.float32, "softmax", 1, 1, 1, True, 1.0)
    i2, w2 = op(v.contiguous(), None, 4, torch.float32, "softmax", 1, 1, 1, True, 1.0)
    assert torch.equal(i1, i2) and torch.equal(w1, w2)
    assert op(x[:0], None, 4, torch.float32, "softmax", 1, 1, 1, True, 1.0)[0].shape == (0, 4)
    with pytest.raises(RuntimeError):
        op(x, None, 4, torch.float32, "softmax", 7, 1, 1, True, 1.0)
    torch.library.opcheck(op.default, (x, b, *args), test_utils=("test_schema", "test_faketensor"))


def close_ones(seed, Tk, E, close, score, at):
    """Logits and biases that bring `close` experts of every token within some 2^-24 of `at`, the others at least
    a tenth below: bias[e] = fp32(at - s(l[e])) for one row l, whose logits differ by up to 2 units of 2^-23 from
    token to token."""
    g = torch.Generator().manual_seed(seed)
    row = torch.randn(E, generator=g) * 1.5
    x = row * (1 + torch.randint(-2, 3, (Tk, E), generator=g) * 2.0**-23)
    s = torch.softmax(row.double(), 0) if score == "softmax" else torch.sigmoid(row.double())
    low = torch.rand(E, generator=g).double() * 0.5 + 0.1
    low[torch.randperm(E, generator=g)[:close]] = 0
    return x, (at - low - s).float()


@pytest.mark.parametrize("E,topk", [(16, 1), (16, 8), (60, 2), (64, 4), (64, 15), (200, 1), (256, 8), (384, 2), (64, 17)])
@pytest.mark.parametrize("close", [3, 5, 8, 12, 999])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("at", [0.9, -0.3])
def test_few_close_scores(dev, E, topk, close, score, at):
    """A few experts closer than fp32 tells apart, or all of them: the choice is the 64-bit one also where the
    close ones go past those that were to be ranked."""
    import ternocl_amd as T
    x, b = close_ones(E + topk, 120, E, min(close, E), score, at)
    check(T, x, b, topk, "f32", score)


@pytest.mark.parametrize("E,n_group,topk_group", [(16, 8, 4), (64, 8, 4), (126, 9, 4), (256, 8, 3), (320, 64, 20), (512, 16, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [0.5, 50.0, 1000.0])
def test_groups_of_opposite_biases(dev, E, n_group, topk_group, score, size):
    """Best twos of opposite sign, whose sums are far smaller than their terms and nearly equal: the groups kept are
    those of 64 bits.  (s1 + s2 = c in every group, up to 2^-22 to 2^-10 of c by token; biases w and -w, w = size..2 size.)"""
    import ternocl_amd as T
    g = torch.Generator().manual_seed(E + n_group)
    Tk, per = 150, E // n_group
    part = torch.rand((n_group, 1), generator=g).double() * 0.6 + 0.2
    part = torch.cat((part, 1 - part), 1)
    pair = torch.log(part) if score == "softmax" else torch.logit(part * 0.9)
    x = torch.full((Tk, n_group, per), -6.0)
    away = 2.0 ** (-22 + 12 * torch.rand((Tk, 1, 1), generator=g))
    x[:, :, :2] = pair.float() * (1 + torch.randn((Tk, n_group, 2), generator=g) * away)
    b = torch.full((n_group, per), -4.0 * size)
    b[:, 0] = size * (1 + torch.rand(n_group, generator=g))
    b[:, 1] = -b[:, 0]
    order = torch.rand((n_group, per), generator=g).argsort(1)
    x, b = x.gather(2, order.expand(Tk, -1, -1)), b.gather(1, order)
    check(T, x.reshape(Tk, E), b.reshape(E), min(6, topk_group * per), "f32", score, n_group, topk_group, 2)


@pytest.mark.parametrize("E", [16, 24, 60, 64, 100])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_at_the_lowest_value(dev, E, score):
    """A group whose experts all have a bias of fp32's lowest value is worth the sum of two of them, below fp32's range,
    and still comes before a group without experts."""
    import ternocl_amd as T
    x, b = logits_of(E, 20, E, "f32")
    per, low = E // 4, torch.finfo(torch.float32).min
    x[:10, per:2 * per] = -math.inf
    b[2 * per:] = low
    b[3 * per:] /= 1 + torch.arange(1, per + 1) * 2.0**-10  # (a little above it)
    for kept in (1, 2, 3):
        for topk in {min(15, kept * per), min(64, kept * per)}:
            check(T, x, b, topk, "f32", score, 4, kept, 2)


@pytest.mark.parametrize("E,topk", [(64, 8), (200, 8), (512, 20)])
def test_weights_as_they_are(dev, E, topk):
    """Weights of a softmax that is not renormalised: fp32 ones over a 64-bit sum, 16-bit ones over an fp32 sum within
    2^-18 of it.  (Most logits of a row lie together, so that the 32-bit terms are off the same way: |l - max| <= 6.5
    in two roundings and a constant, 2.5 x 2^-24 of it each, 2 x 2^-24 for the exponential and 37 x 2^-24 for the
    additions of 32 in a lane and 16 lanes are 55 x 2^-24.)"""
    import ternocl_amd as T
    g = torch.Generator().manual_seed(E)
    Tk = 1500
    x = -(2 + 4 * torch.rand((Tk, 1), generator=g)) * (1 + torch.randint(0, 256, (Tk, E), generator=g) * 2.0**-20)
    x[:, ::E // topk] = torch.rand((Tk, len(range(0, E, E // topk))), generator=g) * 0.5
    check(T, x, None, topk, "f32", renorm=False)
    ids = torch.empty((Tk, topk), dtype=torch.int32, device="cuda")
    want, w = gold(x, None, topk, "softmax", 1, 1, 1, False, 1.0)
    for wt in ("f16", "bf16"):
        RW = torch.empty((Tk, topk), dtype=NAMES[wt], device="cuda")
        T.moe_topk(x.cuda(), None, ids, RW, Tk, E, topk, "softmax", renorm=False)
        torch.cuda.synchronize()
        assert torch.equal(ids.cpu(), want)
        u = torch.finfo(NAMES[wt]).eps / 2
        assert ((RW.cpu().double() - w).abs() <= ((1 + u) * (1 + 2.0**-24) * (1 + 2.0**-18 + 2.0**-36) - 1) * w).all()
