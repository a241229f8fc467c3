"""8-bit activations between a model's layers, as cases for timing and comparing.

  norm   root-mean-square norm of the residual stream with the residual's addition,
         its output as it is, as int8 with a scale for each row (for int8_gemm) or
         as int8 with a scale for each 128 (quant_a's, for int2_int8_gemm) (rmsnorm)
  quant  int8 with a scale for each row without a norm: what goes into a second
         projection (quant_rows)
  int8   products of 8-bit integers with a scale for each token and each channel
         (int8_gemm)

``run`` computes a case in its plain form, elementary torch operations in 32 bits (64
where a value is rounded to 8 bits), or, with ``own``, by the library's calls; ``exact``
is the definition in 64 bits, on its own.  What is held in 8 bits is returned as the
values it stands for, rounded to the activations' type.
"""
import math

import torch

own = False
DEV = "cuda:0"


def listed():
    return [
        # one decoding token before a projection of 8-bit integers: latency
        {"name": "norm one token", "kind": "norm", "bf16": False, "M": 1, "K": 4096, "pad": 0, "res": True, "quant": "rows",
         "y": False, "w32": False, "woff": 0.0},
        # one step of a ragged batch before a ternary product on int8 activations, the norm kept as well
        {"name": "norm batch", "kind": "norm", "bf16": True, "M": 27, "K": 5376, "pad": 0, "res": True, "quant": "groups",
         "y": True, "w32": False, "woff": 1.0},
        # a prompt before products on 16-bit activations
        {"name": "norm prompt", "kind": "norm", "bf16": True, "M": 1024, "K": 4096, "pad": 0, "res": True, "quant": "none",
         "y": True, "w32": True, "woff": 0.0},
        # several prompts together before a projection of 8-bit integers
        {"name": "norm long prompts", "kind": "norm", "bf16": True, "M": 8192, "K": 5120, "pad": 0, "res": True, "quant": "rows",
         "y": False, "w32": False, "woff": 0.0},
        # one decoding token between an MLP's projections
        {"name": "quant one token", "kind": "quant", "bf16": False, "M": 1, "K": 14336, "pad": 0},
        # a prompt between an MLP's projections, its rows in a wider tensor
        {"name": "quant prompt", "kind": "quant", "bf16": True, "M": 2047, "K": 14336, "pad": 64},
        # one token through a square projection: launch latency included
        {"name": "int8 one row", "kind": "int8", "bf16": False, "M": 1, "K": 4096, "N": 4096, "postop": 0, "f32": False},
        # the language-model head over four sequences, fp32 logits
        {"name": "int8 head", "kind": "int8", "bf16": False, "M": 4, "K": 4096, "N": 151680, "postop": 0, "f32": True},
        # one decode step of a batch through an MLP's second projection, residual added
        {"name": "int8 batch", "kind": "int8", "bf16": True, "M": 24, "K": 14336, "N": 4096, "postop": 2, "f32": False},
        # a short ragged prompt, bias added
        {"name": "int8 short prompt", "kind": "int8", "bf16": True, "M": 200, "K": 5120, "N": 5120, "postop": 3, "f32": False},
        # a prompt through an MLP's first projection, silu(gate) * up in its epilogue
        {"name": "int8 prompt", "kind": "int8", "bf16": False, "M": 1024, "K": 4096, "N": 14336, "postop": 1, "f32": False},
        # several prompts together through an MLP's widest projection
        {"name": "int8 long prompts", "kind": "int8", "bf16": True, "M": 4096, "K": 5120, "N": 34816, "postop": 0, "f32": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "quant", "int8", "int8", "int8"))
    bf16 = rng.random() < 0.5
    if kind == "int8":
        K = 128 * _log(rng, 2, 112)
        N = 16 * min(_log(rng, 4, 9480), 4096 * 9480 // K)
        M = min(_log(rng, 1, 4096), max(1, 4096 * 5120 * 34816 // (K * N)))  # (no more than the largest listed)
        return {"kind": kind, "bf16": bf16, "M": M, "K": K, "N": N, "postop": rng.choice((0, 0, 1, 2, 3, 4, 5)),
                "f32": rng.random() < 0.25}
    K = _log(rng, 64, 16384)
    quant = rng.choice(("none", "rows", "rows", "groups"))
    if kind == "quant" or quant != "groups":
        K = rng.choice((K, 8 * (K // 8), 64 * (K // 64)))  # odd sizes, whole vectors, a model's widths
    else:
        K = 128 * max(1, K // 128)
    M = min(_log(rng, 1, 8192), max(1, 8192 * 5120 // K))
    pad = rng.choice((0, 0, 0, 8, 64, 5))
    if kind == "quant":
        return {"kind": kind, "bf16": bf16, "M": M, "K": K, "pad": pad}
    return {"kind": kind, "bf16": bf16, "M": M, "K": K, "pad": pad, "res": rng.random() < 0.75, "quant": quant,
            "y": quant == "none" or rng.random() < 0.3, "w32": rng.random() < 0.3, "woff": rng.choice((0.0, 0.0, 1.0))}


# ---- inputs ----------------------------------------------------------------------

EPS = 1e-6


def _dt(case):
    return torch.bfloat16 if case["bf16"] else torch.float16


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)

    def normal(dt, *shape, sigma=1.0):
        return (torch.randn(shape, device=DEV, generator=g) * sigma).to(dt)

    s, dt, M, K = dict(case), _dt(case), case["M"], case["K"]
    if case["kind"] == "int8":
        N, p = case["N"], case["postop"]
        # (codes as they come out of a scaling by the largest: about normal, the ends rare)
        s["A"] = (torch.randn((M, K), device=DEV, generator=g) * 32).round().clamp(-127, 127).to(torch.int8)
        s["B"] = (torch.randn((K // 16, N, 16), device=DEV, generator=g) * 32).round().clamp(-128, 127).to(torch.int8)
        s["SA"] = torch.rand(M, device=DEV, generator=g) * 0.02 + 0.01
        s["SB"] = (torch.rand(N, device=DEV, generator=g) + 0.5) * (0.04 / math.sqrt(K))
        s["other"] = normal(dt, M, N) if p in (1, 2, 5) else None
        s["bias"] = normal(torch.float32 if case["f32"] else dt, N, sigma=0.1) if p in (3, 5) else None
        if own:
            import ternocl_amd as T
            s["C"] = torch.empty((M, N), dtype=torch.float32 if case["f32"] else dt, device=DEV)
            s["ws"] = _work(T, T.int8_gemm_ws_bytes(M, N, K))
        return s
    # a few channels are far larger than the rest, as in a model's residual stream
    chan = torch.exp(torch.randn(K + case["pad"], device=DEV, generator=g) * 0.5)
    chan = torch.where(torch.rand(K + case["pad"], device=DEV, generator=g) < 0.002, chan * 20, chan)
    s["X"] = (torch.randn((M, K + case["pad"]), device=DEV, generator=g) * chan).to(dt)[:, :K]
    if case["kind"] == "norm":
        s["R"] = normal(dt, M, K, sigma=3.0) if case["res"] else None
        w = torch.rand(K, device=DEV, generator=g) * 0.8 + (0.6 - case["woff"])
        s["W"] = w if case["w32"] else w.to(dt)
    if own:
        s["out"] = torch.empty((M, K), dtype=dt, device=DEV)  # the values that the codes stand for
        s["Q"] = torch.empty((M, K), dtype=torch.int8, device=DEV)
        s["SQ"] = torch.empty(M, device=DEV)
        if case["kind"] == "norm":
            s["H"] = torch.empty((M, K), dtype=dt, device=DEV) if case["res"] else None
            s["Y"] = torch.empty((M, K), dtype=dt, device=DEV) if case["y"] else None
            if case["quant"] == "groups":
                import ternocl_amd as T
                s["SQ"] = torch.empty((K // 128, T.ldsa(M)), dtype=dt, device=DEV)
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
    return {"norm": _plain_norm, "quant": _plain_quant, "int8": _plain_int8}[s["kind"]](s)


def _run_own(s):
    import ternocl_amd as T
    M, K = s["M"], s["K"]
    if s["kind"] == "int8":
        T.int8_gemm(s["A"], s["SA"], s["B"], s["SB"], s["C"], s["other"], s["bias"], M, s["N"], K, s["postop"], s["f32"],
                    ws=s["ws"])
        return s["C"]
    if s["kind"] == "quant":
        T.quant_rows(s["X"], s["Q"], s["SQ"], M, K, ld=K + s["pad"])
        return torch.mul(s["Q"], s["SQ"][:, None], out=s["out"]), s["SQ"]
    q = s["quant"]
    T.rmsnorm(s["X"], s["R"], s["W"], s["H"], s["Y"], s["Q"] if q != "none" else None, s["SQ"] if q != "none" else None,
              M, K, EPS, s["woff"], q, ldx=K + s["pad"])
    got = {"h": s["H"], "y": s["Y"]}
    if q == "rows":
        got["values"], got["scales"] = torch.mul(s["Q"], s["SQ"][:, None], out=s["out"]), s["SQ"]
    elif q == "groups":
        sa = s["SQ"][:, :M]
        inv = (1 / sa.float()).t().reshape(M, K // 128, 1)
        torch.mul(s["Q"].view(M, K // 128, 128), inv, out=s["out"].view(M, K // 128, 128))
        got["values"], got["scales"] = s["out"], sa
    return got


def _plain_rows(t, r):
    """int8 with a scale for each row of t * r: the values, and the scales."""
    top = t.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(127 * t / top), 0.0)  # (64 bits: quotients next to a half)
    scale = (top * r / 127).float()
    return q.float() * scale, scale[:, 0]


def _plain_norm(s):
    M, K, dt = s["M"], s["K"], _dt(s)
    h = s["X"].double()
    if s["R"] is not None:
        h = h + s["R"].double()
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    t = h * (s["W"].double() + s["woff"])
    y = (t * r).float().to(dt)
    got = {"h": h.float().to(dt) if s["R"] is not None else None, "y": y if s["y"] else None}
    if s["quant"] == "rows":
        v, got["scales"] = _plain_rows(t, r)
        got["values"] = v.to(dt)
    elif s["quant"] == "groups":
        a = y.float().view(M, K // 128, 128)
        sa = (127 / a.abs().amax(2).clamp(min=torch.finfo(torch.float32).eps)).to(dt)
        q = torch.round(a * sa.float()[:, :, None]).clamp(-128, 127)
        got["values"] = (q * (1 / sa.float())[:, :, None]).to(dt).view(M, K)
        got["scales"] = sa.t()
    return got


def _plain_quant(s):
    v, scale = _plain_rows(s["X"].double(), 1.0)
    return v.to(_dt(s)), scale


def _plain_int8(s):
    M, K, N = s["M"], s["K"], s["N"]
    W = s["B"].permute(0, 2, 1).reshape(K, N).float()
    x = (s["A"].float() @ W) * s["SA"][:, None] * s["SB"]
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
    return x if s["f32"] else x.to(_dt(s))


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "quant": _exact_quant, "int8": _exact_int8}[case["kind"]](s)


def _half_even(u):
    """The whole number next to each of u, the even one where two are as near."""
    low = torch.floor(u)
    d = u - low
    return low + ((d > 0.5) | ((d == 0.5) & (low % 2 != 0))).double()


def _chunks(s):
    step = max(1, 2**24 // s["K"])
    return [(i, min(s["M"], i + step)) for i in range(0, s["M"], step)]


def _codes(t):
    """(codes, largest magnitude) of rows."""
    top = torch.maximum(t.amax(1), -t.amin(1))[:, None]
    u = _half_even(t * 127 / torch.where(top == 0, 1.0, top))
    return u, top


def _exact_norm(s):
    K, dt, out = s["K"], _dt(s), []
    w = s["W"].double() + s["woff"]
    for i, j in _chunks(s):
        h = s["X"][i:j].double()
        if s["R"] is not None:
            h += s["R"][i:j]
        rms = (torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / K + EPS).sqrt()
        got = {"h": h if s["R"] is not None else None}
        t = h * w
        n = t / rms
        got["y"] = n if s["y"] else None
        if s["quant"] == "rows":
            u, top = _codes(t)
            step = top / (127 * rms)
            got["values"], got["scales"] = u * step, step[:, 0]
        elif s["quant"] == "groups":
            # by definition quant_a's of the norm in the activations' type
            a = n.float().to(dt).double().view(j - i, K // 128, 128)
            top = torch.maximum(a.amax(2), -a.amin(2)).clamp(min=2.0**-23)
            sa = (127 / top).float().to(dt).double()
            u = _half_even(a * sa[:, :, None]).clamp(-128, 127)
            got["values"], got["scales"] = (u / sa[:, :, None]).reshape(j - i, K), sa
        out.append(got)
    full = {k: None if out[0][k] is None else torch.cat([o[k] for o in out]) for k in out[0]}
    if s["quant"] == "groups":
        full["scales"] = full["scales"].t()
    return full


def _exact_quant(s):
    out = []
    for i, j in _chunks(s):
        u, top = _codes(s["X"][i:j].double())
        out.append((u * (top / 127), top[:, 0] / 127))
    return tuple(torch.cat(c) for c in zip(*out))


def _exact_int8(s):
    M, K, N = s["M"], s["K"], s["N"]
    acc = torch.zeros((M, N), dtype=torch.float64, device=DEV)
    step = max(1, 2**27 // (16 * N))  # blocks of 16 rows of K at a time
    for b in range(0, K // 16, step):
        part = s["B"][b:b + step].transpose(1, 2).reshape(-1, N).double()
        acc += s["A"][:, 16 * b:16 * b + part.shape[0]].double() @ part
    acc *= s["SB"].double()
    acc *= s["SA"].double()[:, None]
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


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    M, K = case["M"], case["K"]
    if case["kind"] == "int8":
        N, p, c = case["N"], case["postop"], 4 if case["f32"] else 2
        nbytes = K * N + M * K + 4 * (M + N) + M * N * c + (M * N * 2 if p in (1, 2, 5) else 0) + (N * c if p in (3, 5) else 0)
        return {"bytes": nbytes, "flops": 2 * M * N * K}
    if case["kind"] == "quant":
        return {"bytes": 3 * M * K + 4 * M, "flops": 4 * M * K}
    q = {"none": 0, "rows": M * K + 4 * M, "groups": M * K + M * K // 64}[case["quant"]]
    return {"bytes": M * K * (2 + (4 if case["res"] else 0) + (2 if case["y"] else 0)) + K * (4 if case["w32"] else 2) + q,
            "flops": 8 * M * K}
