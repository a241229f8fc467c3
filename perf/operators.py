"""The calls around a model's ternary layers, as cases for timing and comparing.

  int4      products with 4-bit weights and group scales (int4_gemm): the head and
            the projections that a model keeps at 4 bits, from one row to a prompt
  topk      routing to experts (moe_topk): router logits in, expert ids and weights
            out, as the MoE layers take them
  logprobs  log probabilities of given tokens, entropy and top alternatives of a
            head's logits (logprobs)

``run`` computes a case in its plain form, elementary torch operations in 32 bits
(64 where a choice between close values is made), or, with ``own``, by the
library's calls; ``exact`` is the definition in 64 bits, on its own.
"""
import math

import torch

own = False
DEV = "cuda:0"


def listed():
    return [
        # one token through a square projection: launch latency included
        {"name": "int4 one row", "kind": "int4", "bf16": False, "M": 1, "K": 4096, "N": 4096, "group": 128, "zero": False,
         "postop": 0, "f32": False},
        # one token through an MLP's widest projection, groups of 64 with zero points
        {"name": "int4 one wide row", "kind": "int4", "bf16": True, "M": 1, "K": 5120, "N": 34816, "group": 64, "zero": True,
         "postop": 0, "f32": False},
        # the language-model head over four sequences, fp32 logits
        {"name": "int4 head", "kind": "int4", "bf16": False, "M": 4, "K": 4096, "N": 151680, "group": 128, "zero": False,
         "postop": 0, "f32": True},
        # one decode step of a batch through an MLP's second projection, residual added
        {"name": "int4 batch", "kind": "int4", "bf16": True, "M": 24, "K": 14336, "N": 4096, "group": 128, "zero": False,
         "postop": 2, "f32": False},
        # a short ragged prompt, the finest groups with zero points, bias added
        {"name": "int4 short prompt", "kind": "int4", "bf16": True, "M": 200, "K": 5120, "N": 5120, "group": 32, "zero": True,
         "postop": 3, "f32": False},
        # a prompt through an MLP's first projection, silu(gate) * up in its epilogue
        {"name": "int4 prompt", "kind": "int4", "bf16": False, "M": 1024, "K": 4096, "N": 14336, "group": 128, "zero": False,
         "postop": 1, "f32": False},
        # routing of one decoding token: latency
        {"name": "topk one token", "kind": "topk", "bf16": True, "T": 1, "E": 128, "topk": 8, "ltype": "bf16", "score": "softmax",
         "bias": False, "n_group": 1, "topk_group": 1, "group_best": 1, "renorm": True, "scale": 1.0},
        # routing of a prompt, softmax weights as they are
        {"name": "topk prompt", "kind": "topk", "bf16": True, "T": 2048, "E": 64, "topk": 8, "ltype": "f32", "score": "softmax",
         "bias": False, "n_group": 1, "topk_group": 1, "group_best": 1, "renorm": False, "scale": 1.0},
        # routing of a large batch over groups of experts, sigmoid scores with a balance bias
        {"name": "topk groups", "kind": "topk", "bf16": True, "T": 16384, "E": 256, "topk": 8, "ltype": "f32", "score": "sigmoid",
         "bias": True, "n_group": 8, "topk_group": 4, "group_best": 2, "renorm": True, "scale": 2.5},
        # the answer's token of one sequence, with 20 alternatives
        {"name": "logprobs one row", "kind": "logprobs", "M": 1, "V": 151680, "pad": 0, "ltype": "f32", "topn": 20, "scale": 1.0},
        # a ragged batch of sequences, 16-bit logits at a temperature, a head padded past its vocabulary
        {"name": "logprobs batch", "kind": "logprobs", "M": 27, "V": 151643, "pad": 37, "ltype": "bf16", "topn": 5, "scale": 1.25},
        # scoring a prompt
        {"name": "logprobs prompt", "kind": "logprobs", "M": 512, "V": 151680, "pad": 0, "ltype": "f32", "topn": 20, "scale": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("int4", "int4", "topk", "logprobs"))
    if kind == "int4":
        K = 128 * _log(rng, 4, 112)
        N = 16 * min(_log(rng, 16, 9480), 4096 * 9480 // K)
        M = min(_log(rng, 1, 1024), max(1, 1024 * 4096 * 14336 // (K * N)))  # (no more than the largest listed)
        return {"kind": kind, "bf16": rng.random() < 0.5, "M": M, "K": K, "N": N, "group": rng.choice((32, 64, 128)),
                "zero": rng.random() < 0.5, "postop": rng.choice((0, 0, 1, 2, 3, 4, 5)), "f32": rng.random() < 0.25}
    if kind == "topk":
        n_group = rng.choice((1, 1, 2, 4, 8))
        E = n_group * _log(rng, 2, 512 // n_group)
        topk_group = rng.randint(1, n_group)
        return {"kind": kind, "bf16": rng.random() < 0.5, "T": _log(rng, 1, 16384), "E": E,
                "topk": min(_log(rng, 1, 16), topk_group * E // n_group), "ltype": rng.choice(("f16", "bf16", "f32")),
                "score": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.5, "n_group": n_group,
                "topk_group": topk_group, "group_best": rng.choice((1, 2)) if E // n_group > 1 else 1,
                "renorm": rng.random() < 0.6, "scale": rng.choice((1.0, 1.0, 2.5))}
    V = _log(rng, 1000, 262144)
    return {"kind": kind, "M": min(_log(rng, 1, 4096), 512 * 151680 // V), "V": V, "pad": rng.choice((0, 0, 1, 5, 64)),
            "ltype": rng.choice(("f16", "bf16", "f32")), "topn": rng.choice((1, 5, 20, 64)),
            "scale": rng.choice((1.0, 0.5, 1.25))}


# ---- inputs ----------------------------------------------------------------------

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _dt(case):
    return torch.bfloat16 if case["bf16"] else torch.float16


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)

    def normal(dt, *shape, sigma=1.0):
        return (torch.randn(shape, device=DEV, generator=g) * sigma).to(dt)

    s = dict(case)
    if case["kind"] == "int4":
        M, K, N, dt, p = case["M"], case["K"], case["N"], _dt(case), case["postop"]
        s["A"] = normal(dt, M, K)
        s["B"] = torch.randint(-2**31, 2**31, (K // 32, N, 4), dtype=torch.int32, device=DEV, generator=g)
        s["S"] = (torch.rand((K // case["group"], N), device=DEV, generator=g) * 0.004 + 0.002).to(dt)
        # (zero points in quarters about the codes' middle)
        s["Z"] = ((torch.randn((K // case["group"], N), device=DEV, generator=g) * 6).round() / 4).to(dt) if case["zero"] else None
        s["other"] = normal(dt, M, N) if p in (1, 2, 5) else None
        s["bias"] = normal(torch.float32 if case["f32"] else dt, N, sigma=0.1) if p in (3, 5) else None
        if own:
            import ternocl_amd as T
            s["C"] = torch.empty((M, N), dtype=torch.float32 if case["f32"] else dt, device=DEV)
            s["ws"] = _work(T, T.int4_gemm_ws_bytes(M, N, K, case["group"]))
    elif case["kind"] == "topk":
        s["logits"] = normal(_TYPES[case["ltype"]], case["T"], case["E"], sigma=1.5)
        s["bias"] = normal(torch.float32, case["E"], sigma=0.05) if case["bias"] else None
        if own:
            s["ids"] = torch.empty((case["T"], case["topk"]), dtype=torch.int32, device=DEV)
            s["RW"] = torch.empty((case["T"], case["topk"]), dtype=_dt(case), device=DEV)
    else:
        M, V, n = case["M"], case["V"], case["topn"]
        x = torch.randn((M, V + case["pad"]), device=DEV, generator=g) * 2.5
        # some likely tokens in each row
        hot = torch.randint(0, V, (M, 16), device=DEV, generator=g)
        x.scatter_add_(1, hot, torch.rand((M, 16), device=DEV, generator=g) * 12)
        # a tenth of the vocabulary is ruled out
        x = torch.where(torch.rand((1, V + case["pad"]), device=DEV, generator=g) < 0.1, -math.inf, x)
        s["logits"] = x.to(_TYPES[case["ltype"]])
        pick = torch.randint(0, 16, (M, 1), device=DEV, generator=g)
        tok = hot.gather(1, pick)[:, 0]
        any_ = torch.randint(0, V, (M,), device=DEV, generator=g)
        r = torch.rand((M,), device=DEV, generator=g)
        s["tokens"] = torch.where(r < 0.7, tok, torch.where(r < 0.95, any_, -1)).to(torch.int32)  # (-1: a padded row)
        if own:
            import ternocl_amd as T
            s["logp"] = torch.empty((M,), dtype=torch.float32, device=DEV)
            s["entropy"] = torch.empty((M,), dtype=torch.float32, device=DEV)
            s["top_ids"] = torch.empty((M, n), dtype=torch.int32, device=DEV)
            s["top_logp"] = torch.empty((M, n), dtype=torch.float32, device=DEV)
            s["ws"] = _work(T, T.logprobs_ws_bytes(M, V, n))
    return s


def _work(T, nbytes):
    """A workspace as the library wants it: zeroed once, None where a call uses none."""
    if not nbytes:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    T.workspace_zero(ws)
    return ws


# ---- one pass ----------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"int4": _plain_int4, "topk": _plain_topk, "logprobs": _plain_logprobs}[s["kind"]](s)


def _run_own(s):
    import ternocl_amd as T
    if s["kind"] == "int4":
        T.int4_gemm(s["A"], s["B"], s["S"], s["Z"], s["C"], s["other"], s["bias"], s["M"], s["N"], s["K"], s["group"],
                    s["postop"], s["f32"], ws=s["ws"])
        return s["C"]
    if s["kind"] == "topk":
        T.moe_topk(s["logits"], s["bias"], s["ids"], s["RW"], s["T"], s["E"], s["topk"], s["score"], s["n_group"],
                   s["topk_group"], s["group_best"], s["renorm"], s["scale"])
        return s["ids"], s["RW"]
    T.logprobs(s["logits"], s["tokens"], s["logp"], s["entropy"], s["top_ids"], s["top_logp"], s["M"], s["V"],
               s["V"] + s["pad"], s["topn"], s["scale"], ws=s["ws"])
    return s["logp"], s["entropy"], s["top_ids"], s["top_logp"]


# a word's nibble i holds row 2 i (i < 4) or 2 (i - 4) + 1 of its 8 rows
_SHIFTS = [4 * (r // 2 + 4 * (r % 2)) for r in range(8)]


def _plain_int4(s):
    M, K, N, g = s["M"], s["K"], s["N"], s["group"]
    sh = torch.tensor(_SHIFTS, dtype=torch.int32, device=DEV)
    q = (s["B"][..., None] >> sh) & 15                       # [K/32, N, 4, 8]
    q = torch.where(q > 7, q - 16, q).float()
    W = q.permute(0, 2, 3, 1).reshape(K // g, g, N)
    if s["Z"] is not None:
        W = W - s["Z"].float()[:, None, :]
    W = (W * s["S"].float()[:, None, :]).reshape(K, N)
    x = s["A"].float() @ W
    p = s["postop"]
    if p in (1, 4):
        y = torch.where(x <= -10, 0.0, 1 / (1 + torch.exp(-x)))  # the sigmoid of the library's epilogues
        x = x * y * s["other"].float() if p == 1 else y
    elif p == 2:
        x = x + s["other"].float()
    elif p == 3:
        x = x + s["bias"].float()
    elif p == 5:
        x = x + s["bias"].float() + s["other"].float()
    return x if s["f32"] else x.to(s["A"].dtype)


def _plain_topk(s):
    T, E, k, ng = s["T"], s["E"], s["topk"], s["n_group"]
    x = s["logits"].double()  # (64 bits: the choice between close scores)
    if s["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    sel = score if s["bias"] is None else score + s["bias"].double()
    if ng > 1 and s["topk_group"] < ng:
        best = sel.view(T, ng, E // ng).topk(s["group_best"], 2).values.sum(2)
        gi = _first(best, s["topk_group"])
        keep = torch.zeros((T, ng), dtype=torch.bool, device=DEV).scatter_(1, gi, True)
        sel = torch.where(keep[:, :, None], sel.view(T, ng, E // ng), -math.inf).view(T, E)
    ids = _first(sel, k)
    w = score.gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), (w * s["scale"]).to(_dt(s))


def _first(x, k):
    """The k largest of each row in order, ties to the lowest index."""
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]


def _plain_logprobs(s):
    V, n = s["V"], s["topn"]
    raw = s["logits"][:, :V].float()
    z = raw * s["scale"]
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(1)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * d, 0.0).sum(1) / total
    t = s["tokens"].long()
    logp = torch.where(t >= 0, d.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse, 0.0)
    # the alternatives by (logit, lowest index): whole numbers in that order
    b = raw.view(torch.int32)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long() * 2**32 + (2**31 - 1 - torch.arange(V, device=DEV))
    ids = torch.topk(key, n, 1).indices
    return logp, entropy, ids.to(torch.int32), d.gather(1, ids) - lse[:, None]


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "int4":
        return _exact_int4(s)
    return _exact_topk(s) if case["kind"] == "topk" else _exact_logprobs(s)


def _exact_int4(s):
    M, K, N, g = s["M"], s["K"], s["N"], s["group"]
    acc = torch.zeros((M, N), dtype=torch.float64, device=DEV)
    A = s["A"].double()
    step = max(1, 2**26 // (128 * N)) * 128  # rows of K at a time
    for k0 in range(0, K, step):
        k1 = min(K, k0 + step)
        words = s["B"][k0 // 32:k1 // 32].long() & 0xFFFFFFFF
        W = torch.empty((k1 - k0, N), dtype=torch.float64, device=DEV)
        for w in range(4):
            for pair in range(4):
                for odd in range(2):
                    c = (words[:, :, w] // 16 ** (pair + 4 * odd)) % 16
                    W[8 * w + 2 * pair + odd::32] = (c - 16 * (c // 8)).double()
        rows = torch.arange(k0, k1, device=DEV) // g
        if s["Z"] is not None:
            W -= s["Z"].double()[rows]
        W *= s["S"].double()[rows]
        acc += A[:, k0:k1] @ W
    o = None if s["other"] is None else s["other"].double()
    b = None if s["bias"] is None else s["bias"].double()
    p = s["postop"]
    if p == 0:
        return acc
    if p == 2:
        return acc + o
    if p == 3:
        return acc + b
    if p == 5:
        return acc + b + o
    sg = torch.exp(-acc).add_(1).reciprocal_().masked_fill_(acc <= -10, 0)
    return sg if p == 4 else acc * sg * o


def _exact_topk(s):
    T, E = s["T"], s["E"]
    x = s["logits"].double()
    if s["score"] == "softmax":
        score = torch.exp(x - torch.log(torch.exp(x - x.max()).sum(1, keepdim=True)) - x.max())
    else:
        score = torch.exp(-torch.log1p(torch.exp(-x)))
    # (softmax scores and plain sigmoids order as the logits do: without a bias the logits decide)
    order = x if s["bias"] is None else score + s["bias"].double()
    col = torch.arange(E, device=DEV)
    per = E // s["n_group"]
    allowed = torch.ones((T, E), dtype=torch.bool, device=DEV)
    if s["topk_group"] < s["n_group"]:
        sel = score if s["bias"] is None else order
        gs = sel.view(T, s["n_group"], per).sort(2, descending=True).values[:, :, :s["group_best"]].sum(2)
        if s["group_best"] == 1 and s["bias"] is None:
            gs = x.view(T, s["n_group"], per).amax(2)
        # a group is kept when fewer than topk_group others come before it
        gi = torch.arange(s["n_group"], device=DEV)
        before = (gs[:, None, :] > gs[:, :, None]) | ((gs[:, None, :] == gs[:, :, None]) & (gi[None, None, :] < gi[None, :, None]))
        allowed = (before.sum(2) < s["topk_group"])[:, col // per]
    ids = []
    for _ in range(s["topk"]):
        v = order.masked_fill(~allowed, -math.inf)
        i = torch.where((v == v.amax(1, keepdim=True)) & allowed, col, E).amin(1, keepdim=True)
        allowed = allowed.scatter(1, i, False)
        ids.append(i)
    ids = torch.cat(ids, 1)
    w = score.gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), w * s["scale"]


def _exact_logprobs(s):
    M, V, n = s["M"], s["V"], s["topn"]
    rows = max(1, 2**25 // V)
    out = []
    for r0 in range(0, M, rows):
        raw = s["logits"][r0:r0 + rows, :V].double()
        z = raw * s["scale"]
        top = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :max(n, 1)]
        z = z - z.gather(1, top[:, :1])
        e = torch.exp(z).scatter_(1, top[:, :1], 0.0)      # all but the largest, whose term is 1
        rest = e.sum(1)
        lse = torch.log1p(rest)
        entropy = lse - torch.where(e > 0, z * e, 0.0).sum(1) / (1 + rest)
        t = s["tokens"][r0:r0 + rows].long()
        logp = z.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse
        logp[t < 0] = 0
        out.append((logp, entropy, top[:, :n].to(torch.int32), z.gather(1, top[:, :n]) - lse[:, None]))
    return tuple(torch.cat(c) for c in zip(*out))


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if case["kind"] == "int4":
        M, K, N, p = case["M"], case["K"], case["N"], case["postop"]
        c = 4 if case["f32"] else 2
        scales = (2 if case["zero"] else 1) * (K // case["group"]) * N * 2
        nbytes = K * N // 2 + scales + M * K * 2 + M * N * c + (M * N * 2 if p in (1, 2, 5) else 0) + (N * c if p in (3, 5) else 0)
        return {"bytes": nbytes, "flops": 2 * M * N * K}
    if case["kind"] == "topk":
        T, E, k = case["T"], case["E"], case["topk"]
        return {"bytes": T * E * size[case["ltype"]] + (4 * E if case["bias"] else 0) + T * k * 6, "flops": T * E * (4 + k)}
    M, V, n = case["M"], case["V"], case["topn"]
    return {"bytes": M * V * size[case["ltype"]] + M * (4 + 8 + 8 * n), "flops": 6 * M * V}
