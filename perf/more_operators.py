"""The W8A8 linear over experts: router, expert order, grouped products and their combination.

A layer with E experts sends each token to k of them.  The (token, choice) pairs, ordered by expert,
are the rows of the grouped products: expert e has the rows offsets[e] to offsets[e + 1].  The cases:

  route    moe_route: scores, the k best experts of each token, their weights, and the order
  order    moe_order: the order alone, of experts that were picked elsewhere
  mm       w8a8_grouped_mm: int8 activations, an int8 weight for each expert
  silu     w8a8_grouped_mm_silu_mul: the gate and up projections with silu(gate) * up
  combine  moe_combine: the weighted sum of a token's rows
"""

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "int8-linear_amd")

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# generic layers: hidden width, width of an expert, experts, experts a token takes
LAYERS = [(2048, 768, 128, 8), (2048, 1408, 60, 4), (4096, 14336, 8, 2), (1024, 512, 32, 8),
          (7168, 2048, 32, 8), (2880, 2880, 32, 4), (4096, 1792, 16, 2), (5120, 1024, 64, 6)]
MAX_FLOPS = 2.0 * 8192 * 4096 * 28672   # the largest listed product
MAX_WEIGHT = 8 * 4096 * 28672           # bytes of the largest listed weight


def listed():
    return [
        # one sequence's token: launch and latency
        {"name": "route 1 of 128", "kind": "route", "t": 1, "e": 128, "k": 8, "act": "bf16",
         "scoring": "softmax", "renorm": True, "masked": 0.0},
        # a full prompt, fp32 logits
        {"name": "route 8192 of 128", "kind": "route", "t": 8192, "e": 128, "k": 8, "act": "fp32",
         "scoring": "softmax", "renorm": True, "masked": 0.0},
        # a decode batch whose router stands elsewhere; a quarter of its pairs belong to other ranks
        {"name": "order 75 of 60", "kind": "order", "t": 75, "e": 60, "k": 4, "gone": 0.25},
        # a ragged prompt on one rank of several
        {"name": "order 5001 of 256", "kind": "order", "t": 5001, "e": 256, "k": 8, "gone": 0.5},
        # one sequence's token through eight experts' down projections
        {"name": "mm 1 down 768", "kind": "mm", "t": 1, "e": 128, "k": 8, "kk": 768, "n": 2048,
         "gather": False, "out": "bf16", "bias": False, "skew": 0.0, "gone": 0.0},
        # a decode batch through the gate and up projections of nearly every expert: all weights, few rows
        {"name": "mm 40 gate_up", "kind": "mm", "t": 40, "e": 128, "k": 8, "kk": 2048, "n": 1536,
         "gather": True, "out": "bf16", "bias": False, "skew": 0.5, "gone": 0.0},
        # a ragged prompt, K no whole number of steps, a bias, part of the experts on other ranks
        {"name": "mm 777 of 32 bias", "kind": "mm", "t": 777, "e": 32, "k": 4, "kk": 2880, "n": 5760,
         "gather": True, "out": "bf16", "bias": True, "skew": 0.5, "gone": 0.25},
        # a full prompt over few wide experts: arithmetic
        {"name": "mm 4096 of 8", "kind": "mm", "t": 4096, "e": 8, "k": 2, "kk": 4096, "n": 28672,
         "gather": True, "out": "bf16", "bias": False, "skew": 0.3, "gone": 0.0},
        # a small decode batch's gate and up projections with the activation
        {"name": "silu 4 of 60", "kind": "silu", "t": 4, "e": 60, "k": 4, "kk": 2048, "n": 2816,
         "gather": True, "out": "bf16", "bias": False, "skew": 0.5, "gone": 0.0},
        # a full prompt over many narrow experts
        {"name": "silu 4096 of 128", "kind": "silu", "t": 4096, "e": 128, "k": 8, "kk": 2048, "n": 1536,
         "gather": True, "out": "bf16", "bias": False, "skew": 0.5, "gone": 0.0},
        # a decode batch's rows back to its tokens
        {"name": "combine 40", "kind": "combine", "t": 40, "k": 8, "n": 2048, "act": "bf16",
         "base": False, "gone": 0.0},
        # a full prompt's, added to what an expert of all tokens gave
        {"name": "combine 8192 base", "kind": "combine", "t": 8192, "k": 8, "n": 2048, "act": "bf16",
         "base": True, "gone": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "order", "mm", "mm", "mm", "silu", "silu", "combine"])
    gone = rng.choice([0.0, 0.0, 0.25, 0.75])
    if kind in ("route", "order"):
        e = rng.choice([8, 16, 60, 64, 128, 160, 256, _log(rng, 2, 512)])
        case = {"kind": kind, "t": _log(rng, 1, 8192), "e": e, "k": rng.randint(1, min(8, e))}
        if kind == "order":
            return case | {"gone": gone}
        return case | {"act": rng.choice(["bf16", "fp16", "fp32"]), "scoring": rng.choice(["softmax", "sigmoid"]),
                       "renorm": rng.random() < 0.7, "masked": rng.choice([0.0, 0.0, 0.1, 0.9])}
    act = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "combine":
        k, n = rng.randint(1, 8), rng.choice([1024, 2048, 2880, 4096, 7168, _log(rng, 1, 8192)])
        return {"kind": kind, "t": _log(rng, 1, 8192 * 18 * 2048 // ((k + 2) * n * (2 if act == "fp32" else 1))),
                "k": k, "n": n, "act": act, "base": rng.random() < 0.5, "gone": gone}
    hidden, width, e, k = rng.choice(LAYERS)
    if rng.random() < 0.2:   # any whole 16s, with any other number of experts
        hidden, width = 16 * _log(rng, 1, 256), 8 * _log(rng, 1, 256)
        e = _log(rng, 1, 256)
        k = rng.randint(1, min(8, e))
    gather = kind == "silu" or rng.random() < 0.5
    kk, n = (hidden, 2 * width) if gather else (width, hidden)
    while e * kk * n > MAX_WEIGHT:
        e = (e + 1) // 2
    k = min(k, e)
    return {"kind": kind, "t": _log(rng, 1, min(8192, int(MAX_FLOPS / (2.0 * k * kk * n)))), "e": e, "k": k,
            "kk": kk, "n": n, "gather": gather, "out": act, "bias": rng.random() < 0.3,
            "skew": rng.choice([0.0, 0.5, 2.0]), "gone": gone}


# ------------------------------------------------------------------ inputs
def _randn(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _codes(shape, g):
    return _randn(shape, g, 32.0).round_().clamp_(-127, 127).to(torch.int8)


def _uniform(shape, g, lo, hi):
    return torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo


def _choices(case, g):
    """A router's experts [T, k], -1 where the expert is another rank's; some experts are picked more."""
    t, e, k = case["t"], case["e"], case["k"]
    score = _randn((t, e), g) + case.get("skew", 0.5) * _randn((e,), g)
    ids = score.topk(k, 1).indices.int()
    here = torch.rand((e,), generator=g, device="cuda") >= case["gone"]
    return torch.where(here[ids.long()], ids, -1)


def _sorted(ids, e):
    """(offsets [E + 1], token of each ordered row [T k], place of each pair [T, k])."""
    t, k = ids.shape
    flat = torch.where(ids < 0, e, ids).flatten()
    order = torch.sort(flat, stable=True).indices
    offsets = (flat[None, :] < torch.arange(e + 1, device=ids.device)[:, None]).sum(1).int()
    at = torch.arange(t * k, device=ids.device)
    tokens = torch.where(at < offsets[e], order // k, -1).int()
    places = torch.empty_like(at).scatter_(0, order, at)
    return offsets, tokens, torch.where(flat < e, places, -1).int().view(t, k)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, t, s = case["kind"], case["t"], {"case": case}
    if kind == "route":
        x = _randn((t, case["e"]), g, 1.5).to(DTYPE[case["act"]])
        if case["masked"]:   # experts that a token may not take; now and then none is left
            x = x.masked_fill(torch.rand(x.shape, generator=g, device="cuda") < case["masked"], -math.inf)
        return s | {"x": x}
    if kind == "order":
        return s | {"ids": _choices(case, g)}
    if kind == "combine":
        k, n = case["k"], case["n"]
        dt, rows = DTYPE[case["act"]], t * k
        places = torch.randperm(rows, generator=g, device="cuda").int()
        places = torch.where(torch.rand((rows,), generator=g, device="cuda") < case["gone"], -1, places).view(t, k)
        return s | {"y": _randn((rows, n), g).to(dt), "w": torch.softmax(_randn((t, k), g), 1), "places": places,
                    "base": _randn((t, n), g).to(dt) if case["base"] else None}
    e, k, kk, n = case["e"], case["k"], case["kk"], case["n"]
    offsets, tokens, _ = _sorted(_choices(case, g), e)
    rows = t * k
    m = t if case["gather"] else rows
    dt = DTYPE[case["out"]]
    w = torch.empty((e, n, kk), dtype=torch.int8, device="cuda")
    for i in range(e):
        w[i] = _codes((n, kk), g)
    # scales that give outputs of about one: 32 is the codes' deviation
    sb = _uniform((e, n), g, 0.5, 1.5) / (32.0 * math.sqrt(kk))
    return s | {"a": _codes((m, kk), g), "sa": _uniform((m, 1), g, 0.5, 1.5) / 32.0, "w": w, "sb": sb,
                "bias": _randn((e, n), g, 0.1).to(dt) if case["bias"] else None, "offsets": offsets,
                "rows": tokens if case["gather"] else None, "dtype": dt,
                "groups": offsets.tolist(),   # for the plain form, which needs them on the host
                "out": torch.zeros((rows, n // 2 if kind == "silu" else n), dtype=dt, device="cuda")}


# ------------------------------------------------------------------ plain forms
def _sigmoid(x):
    z = torch.exp(-x.abs())
    return torch.where(x >= 0, 1 / (1 + z), z / (1 + z))


def _plain_route(s):
    case, x = s["case"], s["x"].float()
    k, e = case["k"], case["e"]
    x = torch.where(torch.isnan(x), -math.inf, x)
    left, ids = x.clone(), []
    cols = torch.arange(e, device=x.device)
    for _ in range(k):   # the largest left, of equal ones the first
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, cols, e).amin(1, keepdim=True)
        ids.append(torch.where(best > -math.inf, first, -1))
        left = left.masked_fill(cols == first, -math.inf)
    ids = torch.cat(ids, 1)
    got = ids >= 0
    if case["scoring"] == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.where(x == -math.inf, 0.0, torch.where(x == top, 1.0, torch.exp(x - top)))
        total = p.sum(1, keepdim=True)
    else:
        p = _sigmoid(x)
        total = None
    w = torch.where(got, p.gather(1, ids.clamp(min=0)), 0.0)
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
    if total is not None:
        w = torch.where(total > 0, w / total, 0.0)
    offsets, tokens, places = _sorted(ids, e)
    return {"weights": w, "experts": ids.int(), "offsets": offsets, "tokens": tokens, "places": places}


def _plain_mm(s):
    a, out, at = s["a"].float(), s["out"], s["groups"]
    for e in range(len(at) - 1):
        lo, hi = at[e], at[e + 1]
        if lo == hi:
            continue
        r = slice(lo, hi) if s["rows"] is None else s["rows"][lo:hi].long()
        c = (a[r] @ s["w"][e].float().t()) * s["sa"][r] * s["sb"][e]
        if s["bias"] is not None:
            c = c + s["bias"][e].float()
        if s["case"]["kind"] == "silu":
            gate, up = c.chunk(2, 1)
            c = gate * _sigmoid(gate) * up
        out[lo:hi] = c.to(out.dtype)
    return {"out": out}


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        return _plain_route(s)
    if kind == "order":
        return dict(zip(("offsets", "tokens", "places"), _sorted(s["ids"], case["e"])))
    if kind == "combine":
        at = s["places"]
        total = None if s["base"] is None else s["base"].float()
        for j in range(case["k"]):
            row = torch.where((at[:, j] >= 0)[:, None], s["y"][at[:, j].clamp(min=0).long()].float(), 0.0)
            total = row * s["w"][:, j:j + 1] if total is None else total + row * s["w"][:, j:j + 1]
        return {"out": total.to(s["y"].dtype)}
    return _plain_mm(s)


# ------------------------------------------------------------------ one pass
def run(s):
    if not own:
        return _plain(s)
    moe, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "route":
        r = moe.moe_route(s["x"], case["k"], scoring=case["scoring"], renormalize=case["renorm"])
        return {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "tokens": r.tokens, "places": r.places}
    if kind == "order":
        offsets, tokens, places = moe.moe_order(s["ids"], case["e"])
        return {"offsets": offsets, "tokens": tokens, "places": places}
    if kind == "combine":
        return {"out": moe.moe_combine(s["y"], s["w"], s["places"], base=s["base"])}
    call = moe.w8a8_grouped_mm_silu_mul if kind == "silu" else moe.w8a8_grouped_mm
    # rows of experts elsewhere stay as they were: into the caller's output
    out = s["out"] if case["gone"] else None
    return {"out": call(s["a"], s["w"].transpose(1, 2), s["sa"], s["sb"], s["offsets"], s["dtype"], s["bias"],
                        rows=s["rows"], out=out)}


_module = None


def _package():
    global _module
    if _module is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from int8_linear import moe
        _module = moe
    return _module


def work(case):
    kind, t, k = case["kind"], case["t"], case["k"]
    pairs = t * k
    if kind == "route":
        return {"bytes": t * case["e"] * BYTES[case["act"]] + 16 * pairs + 4 * (case["e"] + 1),
                "flops": 6.0 * t * case["e"]}
    if kind == "order":
        return {"bytes": 12 * pairs + 4 * (case["e"] + 1), "flops": 4.0 * pairs}
    if kind == "combine":
        n, b = case["n"], BYTES[case["act"]]
        return {"bytes": pairs * (1 - case["gone"]) * n * b + t * n * b * (2 if case["base"] else 1) + 8 * pairs,
                "flops": 2.0 * pairs * n}
    e, kk, n = case["e"], case["kk"], case["n"]
    here = 1 - case["gone"]
    rows = pairs * here
    active = e * here * (1 - (1 - k / e) ** t)   # the experts that some token takes, as expected
    b = BYTES[case["out"]]
    return {"bytes": (t if case["gather"] else rows) * (kk + 4) + active * (n * (kk + 4 + (b if case["bias"] else 0)))
                     + rows * (n // 2 if kind == "silu" else n) * b, "flops": 2.0 * rows * n * kk}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_order(ids, e):
    """The same order by rank: a pair stands behind all of lower experts and its expert's earlier ones."""
    t, k = ids.shape
    ids = ids.cpu().flatten().tolist()
    rows = [[] for _ in range(e)]
    for i, x in enumerate(ids):
        if 0 <= x < e:
            rows[x].append(i)
    offsets, tokens, places = [0], [], [-1] * (t * k)
    for r in rows:
        for i in r:
            places[i] = len(tokens)
            tokens.append(i // k)
        offsets.append(len(tokens))
    tokens += [-1] * (t * k - len(tokens))
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return {"offsets": whole(offsets), "tokens": whole(tokens), "places": whole(places).view(t, k)}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "order":
        return _exact_order(s["ids"], case["e"])
    if kind == "route":
        x = s["x"].double()
        ranked = torch.sort(x, dim=1, descending=True, stable=True)
        got = ranked.values[:, :case["k"]] > -math.inf
        ids = torch.where(got, ranked.indices[:, :case["k"]], -1)
        if case["scoring"] == "softmax":
            p = torch.softmax(torch.where(got.any(1, keepdim=True), x, 0.0), 1)
        else:
            p = torch.sigmoid(x)
        w = torch.where(got, p.gather(1, ids.clamp(min=0)), 0.0)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        return {"weights": w, "experts": ids.int()} | _exact_order(ids, case["e"])
    if kind == "combine":
        y, places = s["y"], s["places"].long()
        out = torch.zeros((case["t"], case["n"]), dtype=torch.float64, device="cuda")
        if s["base"] is not None:
            out += s["base"].double()
        for j in range(case["k"]):
            some = (places[:, j] >= 0).nonzero().flatten()
            out[some] += y[places[some, j]].double() * s["w"][some, j].double()[:, None]
        return {"out": out}
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi == lo:
            continue
        at = torch.arange(lo, hi, device="cuda")
        at = at if s["rows"] is None else s["rows"][at].long()
        v = torch.matmul(s["a"][at].double() * s["sa"][at].double(), s["w"][e].double().t())
        v = v * s["sb"][e].double()
        if s["bias"] is not None:
            v = v + s["bias"][e].double()
        if kind == "silu":
            half = v.shape[1] // 2
            v = torch.nn.functional.silu(v[:, :half]) * v[:, half:]
        out[lo:hi] = v
    return {"out": out}
