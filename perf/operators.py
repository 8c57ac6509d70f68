"""The microscaled 4-bit (MXFP4) linear's operators and the query / key norm with its rotation.

An MXFP4 tensor holds E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte with
the even element in the low nibble, and one E8M0 scale (2^(byte - 127), 255 is NaN) for each 32
elements along K.  The cases:

  quant  mxfp4_quant of a tensor and mxfp4_dequant back to its values
  norm   add_rmsnorm_mxfp4_quant: the residual add, RMSNorm and quantizer before a projection
  silu   silu_mul_mxfp4_quant: the MLP's activation and quantizer before down_proj
  mm     mxfp4_mm over one projection: decode, batched decode, a chunk of a prompt, a full prompt
  qk     qk_norm_rope: the norms of the query and key heads and their rotation, read in place from
         the columns of a qkv output

The quantizers' codes come back as the values that they stand for, through mxfp4_dequant.
"""

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "int8-linear_amd")

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# (K, N) of the projections of the two models the benchmark runs, merged as a server runs them
QWEN = [(2048, 4096), (2048, 2048), (2048, 12288), (6144, 2048)]
LLAMA = [(4096, 6144), (4096, 4096), (4096, 28672), (14336, 4096)]
# generic: other hidden and MLP widths, and the shards of a tensor-parallel split
GENERIC = [(5120, 7680), (5120, 5120), (13824, 5120), (3584, 4608), (3584, 18944), (8192, 10240),
           (4096, 1536), (1792, 4096), (2560, 9728), (1024, 4096), (4096, 5504), (2752, 4096)]
HIDDEN = [1024, 2048, 2560, 3584, 4096, 5120, 8192]
MLP = [1536, 1792, 2752, 6144, 8960, 9728, 13824, 14336, 18944]
HEADS = [(16, 8), (32, 8), (8, 1), (4, 4), (5, 1), (28, 4), (64, 8)]

MAX_FLOPS = 2.0 * 4096 * 4096 * 28672   # the largest listed product
EPS = 1e-6


def listed():
    return [
        # a decode batch's attention output in front of o_proj
        {"name": "quant 7 x 2048", "kind": "quant", "m": 7, "k": 2048, "ld": 2048, "act": "bf16", "round": False},
        # a layer's weight (or a prompt's activations) laid out once, by the rounded scale
        {"name": "quant 4096 x 14336", "kind": "quant", "m": 4096, "k": 14336, "ld": 14336, "act": "bf16", "round": True},
        # one sequence's token in front of qkv_proj
        {"name": "norm 1 x 2048", "kind": "norm", "m": 1, "k": 2048, "act": "bf16", "residual": True, "round": False},
        # a full prompt in front of a projection of the 4096-wide model
        {"name": "norm 4096 x 4096", "kind": "norm", "m": 4096, "k": 4096, "act": "bf16", "residual": True, "round": False},
        # a decode batch in front of down_proj
        {"name": "silu 24 x 6144", "kind": "silu", "m": 24, "k": 6144, "act": "bf16", "round": False},
        # a ragged prompt in front of the wide model's down_proj
        {"name": "silu 3001 x 14336", "kind": "silu", "m": 3001, "k": 14336, "act": "bf16", "round": False},
        # one sequence's token through the smallest merged projection: launch and latency
        {"name": "mm qkv 1", "kind": "mm", "m": 1, "k": 2048, "n": 4096, "out": "bf16", "bias": False},
        # a ragged decode batch through the longest reduction
        {"name": "mm down 75", "kind": "mm", "m": 75, "k": 14336, "n": 4096, "out": "bf16", "bias": False},
        # a ragged chunk of a prompt, fp32 logits-style output with a bias
        {"name": "mm qkv 777 fp32 bias", "kind": "mm", "m": 777, "k": 4096, "n": 6144, "out": "fp32", "bias": True},
        # a full prompt through the widest projection
        {"name": "mm gate_up 4096", "kind": "mm", "m": 4096, "k": 4096, "n": 28672, "out": "bf16", "bias": False},
        # one sequence's token between qkv_proj and attention
        {"name": "qk 1", "kind": "qk", "m": 1, "hq": 16, "hk": 8, "d": 128, "rot": 128, "act": "bf16", "inter": False, "pos": "any"},
        # a prompt of the wider model
        {"name": "qk 4096 x 32+8", "kind": "qk", "m": 4096, "hq": 32, "hk": 8, "d": 128, "rot": 128, "act": "bf16", "inter": False, "pos": "run"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "norm", "silu", "mm", "mm", "mm", "qk", "qk"])
    act = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "mm":
        if rng.random() < 0.6:
            k, n = rng.choice(rng.choice([QWEN, LLAMA, GENERIC]))
        else:   # any whole number of blocks, any number of columns
            k, n = 32 * _log(rng, 1, 448), _log(rng, 1, 20000)
        return {"kind": kind, "m": _log(rng, 1, min(8192, int(MAX_FLOPS / (2.0 * k * n)))), "k": k, "n": n,
                "out": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "bias": rng.random() < 0.4}
    if kind == "quant":
        k = rng.choice(HIDDEN + [32 * _log(rng, 1, 400)])
        return {"kind": kind, "m": _log(rng, 1, 4096), "k": k, "ld": rng.choice([k, k + k // 2, k + 24]),
                "act": rng.choice(["bf16", "fp16", "fp32"]), "round": rng.random() < 0.5}
    if kind == "norm":
        return {"kind": kind, "m": _log(rng, 1, 8192), "k": rng.choice(HIDDEN + [32 * _log(rng, 1, 256)]), "act": act,
                "residual": rng.random() < 0.8, "round": rng.random() < 0.5}
    if kind == "silu":
        return {"kind": kind, "m": _log(rng, 1, 3000), "k": rng.choice(MLP + [32 * _log(rng, 1, 400)]), "act": act,
                "round": rng.random() < 0.5}
    hq, hk = rng.choice(HEADS)
    d = rng.choice([64, 80, 96, 128, 128, 256])
    return {"kind": kind, "m": _log(rng, 1, 8192 * 5120 // ((hq + hk) * d + 5120)), "hq": hq, "hk": hk, "d": d,
            "rot": rng.choice([d, d, d // 2, d // 4]), "act": act, "inter": rng.random() < 0.3,
            "pos": rng.choice(["any", "run"])}


# ------------------------------------------------------------------ inputs
def _randn(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, m, s = case["kind"], case["m"], {"case": case}
    if kind == "quant":
        x = _randn((m, case["ld"]), g).to(DTYPE[case["act"]])
        return s | {"x": x[:, :case["k"]]}
    if kind == "norm":
        k, dt = case["k"], DTYPE[case["act"]]
        return s | {"x": _randn((m, k), g).to(dt), "res": _randn((m, k), g).to(dt) if case["residual"] else None,
                    "w": (1 + _randn((k,), g, 0.1)).to(dt)}
    if kind == "silu":
        return s | {"x": _randn((m, 2 * case["k"]), g).to(DTYPE[case["act"]])}
    if kind == "mm":
        k, n = case["k"], case["n"]
        a_q, a_s = _pack(*_quant(_randn((m, k), g), False))
        w_q, w_s = _pack(*_quant(_randn((n, k), g, 0.02), False))
        bias = _randn((n,), g, 0.01).to(DTYPE[case["out"]]) if case["bias"] else None
        return s | {"a": a_q, "sa": a_s, "w": w_q.t(), "sw": w_s, "bias": bias, "out": DTYPE[case["out"]]}
    hq, hk, d, rot, dt = case["hq"], case["hk"], case["d"], case["rot"], DTYPE[case["act"]]
    qkv = _randn((m, (hq + 2 * hk) * d), g).to(dt)
    span = 40960
    if case["pos"] == "run":   # a prompt's positions, from somewhere in a sequence on
        first = torch.randint(0, span - m, (1,), generator=g, device="cuda")
        pos = first + torch.arange(m, device="cuda")
    else:                      # a decode batch's, each of its own sequence
        pos = torch.randint(0, span, (m,), generator=g, device="cuda")
    inv = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(span, device="cuda", dtype=torch.float64)[:, None] * inv
    return s | {"q": qkv[:, :hq * d].view(m, hq, d), "k": qkv[:, hq * d:(hq + hk) * d].view(m, hk, d),
                "qw": (1 + _randn((d,), g, 0.1)).to(dt), "kw": (1 + _randn((d,), g, 0.1)).to(dt),
                "cs": torch.cat([angle.cos(), angle.sin()], 1).float(), "pos": pos}


# ------------------------------------------------------------------ plain forms
def _quant(x, rounded):
    """E2M1 values of x / scale, and the scale's E8M0 codes, for each 32 along the last axis."""
    b = x.float().unflatten(-1, (-1, 32))
    peak = b.abs().amax(-1)
    part, e = torch.frexp(peak)
    e = e.int() - 1                                         # floor(log2(peak))
    if rounded:
        e = e + (part >= 0.875).int()                       # of peak rounded to E2M1's precision
    code = (e - 2 + 127).clamp(0, 254)
    code = torch.where(peak == 0, 0, code)
    v = b * ((254 - code) << 23).view(torch.float32)[..., None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = torch.copysign((torch.round(a / step) * step).clamp(max=6), v)
    bad = ~torch.isfinite(peak)
    return torch.where(bad[..., None], 0.0, v).flatten(-2), torch.where(bad, 255, code)


def _pack(v, code):
    """Values and scale codes as a checkpoint holds them: two codes a byte, bytes of E8M0."""
    a = v.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).int() | (torch.signbit(v).int() << 3)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), code.to(torch.uint8)


def _scale(code):
    s = torch.where(code == 0, 1 << 22, code.int() << 23).view(torch.float32)   # 2^(code - 127)
    return torch.where(code == 255, math.nan, s)


def _values(v, code):
    return (v.unflatten(-1, (-1, 32)) * _scale(code)[..., None]).flatten(-2)


def _unpack(q, code):
    c = torch.stack([q & 15, q >> 4], -1).flatten(-2).int()
    a = c & 7
    a = torch.where(a < 4, a * 0.5, torch.where(a < 6, a - 2.0, 2.0 * a - 8))
    return _values(torch.where(c >= 8, -a, a), code)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "quant":
        return {"values": _values(*_quant(s["x"], case["round"])).bfloat16()}
    if kind == "norm":
        x, w = s["x"], s["w"]
        v = x.float() if s["res"] is None else x.float() + s["res"].float()
        var = v.double().square().mean(1, keepdim=True).float()
        rs = (1 / (var + EPS).double().sqrt()).float()
        y = ((v * rs).to(w.dtype).float() * w.float()).to(x.dtype)
        out = {"values": _values(*_quant(y, case["round"])).bfloat16()}
        return out if s["res"] is None else out | {"residual": v.to(x.dtype)}
    if kind == "silu":
        g, u = s["x"].chunk(2, 1)
        a = (g.double() / (1 + (-g.double()).exp())).to(g.dtype)   # (in 64 bits: next to a rounding's border)
        return {"values": _values(*_quant((a.float() * u.float()).to(g.dtype), case["round"])).bfloat16()}
    if kind == "mm":
        c = _unpack(s["a"], s["sa"]) @ _unpack(s["w"].t(), s["sw"]).t()
        return {"out": (c if s["bias"] is None else c + s["bias"].float()).to(s["out"])}
    return {"q": _rotate(s, s["q"], s["qw"]), "k": _rotate(s, s["k"], s["kw"])}


def _rotate(s, x, w):
    rot, inter = s["case"]["rot"], s["case"]["inter"]
    h = x.float()
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.float()
    cos, sin = s["cs"][s["pos"]][:, None].chunk(2, -1)
    r = h[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else r.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([r, h[..., rot:]], -1).to(x.dtype)


# ------------------------------------------------------------------ one pass
def run(s):
    if not own:
        return _plain(s)
    mx, qk = _package()
    case = s["case"]
    kind = case["kind"]
    if kind == "quant":
        return {"values": mx.mxfp4_dequant(*mx.mxfp4_quant(s["x"], case["round"]))}
    if kind == "norm":
        q, e, res = mx.add_rmsnorm_mxfp4_quant(s["x"], s["res"], s["w"], EPS, case["round"])
        out = {"values": mx.mxfp4_dequant(q, e)}
        return out if res is None else out | {"residual": res}
    if kind == "silu":
        return {"values": mx.mxfp4_dequant(*mx.silu_mul_mxfp4_quant(s["x"], case["round"]))}
    if kind == "mm":
        return {"out": mx.mxfp4_mm(s["a"], s["w"], s["sa"], s["sw"], s["out"], s["bias"])}
    q, k = qk.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cs"], s["pos"], EPS, interleaved=case["inter"])
    return {"q": q, "k": k}


_modules = None


def _package():
    global _modules
    if _modules is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from int8_linear import mxfp4, qk_rope
        _modules = mxfp4, qk_rope
    return _modules


def work(case):
    kind, m = case["kind"], case["m"]
    if kind == "mm":
        k, n = case["k"], case["n"]
        return {"bytes": (m + n) * k * 17 / 32 + m * n * BYTES[case["out"]] + (n * BYTES[case["out"]] if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if kind == "qk":
        width = (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": m * (2 * width * BYTES[case["act"]] + 4 * case["rot"] + 8) + 4 * case["d"], "flops": 8.0 * m * width}
    k = case["k"]
    back = m * k * (17 / 32 + 2)   # the codes and scales, and the values that are made of them
    if kind == "quant":
        return {"bytes": m * k * BYTES[case["act"]] + back, "flops": 4.0 * m * k}
    if kind == "norm":
        return {"bytes": m * k * (6 if case["residual"] else 2) + 2 * k + back, "flops": 8.0 * m * k}
    return {"bytes": m * k * 4 + back, "flops": 12.0 * m * k}


# ------------------------------------------------------------------ the definitions in 64 bits
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_quant(y, rounded):
    """Nearest E2M1 value of y over its block's power of two, of two equally near ones the even code."""
    y = y.double()
    blocks = y.reshape(y.shape[0], -1, 32)
    peak = blocks.abs().max(-1, keepdim=True).values
    p = torch.floor(torch.log2(peak.clamp_min(1e-300)))
    p = torch.where(torch.exp2(p) > peak, p - 1, torch.where(torch.exp2(p + 1) <= peak, p + 1, p))
    if rounded:
        p = torch.where(peak >= 1.75 * torch.exp2(p), p + 1, p)
    scale = torch.exp2((p - 2).clamp(-127, 127))
    t = blocks.abs() / scale
    best, away = torch.zeros_like(t), t.clone()
    for i, grid in enumerate(_GRID[1:], 1):
        off = (t - grid).abs()
        nearer = (off < away) | ((off == away) & (i % 2 == 0))
        best, away = torch.where(nearer, grid, best), torch.where(nearer, off, away)
    return (torch.sign(blocks) * best * scale).reshape(y.shape)


def _exact_values(q, code):
    table = torch.tensor(_GRID + [-v for v in _GRID], dtype=torch.float64, device=q.device)
    v = torch.empty(q.shape[0], q.shape[1] * 2, dtype=torch.float64, device=q.device)
    v[:, 0::2], v[:, 1::2] = table[(q % 16).long()], table[(q // 16).long()]
    return v * torch.exp2(code.double() - 127).repeat_interleave(32, 1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quant":
        return {"values": _exact_quant(s["x"], case["round"])}
    if kind == "norm":
        v = s["x"].double()
        if s["res"] is not None:
            v = v + s["res"].double()
        h = v / (v.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS).sqrt()
        y = (h.to(s["w"].dtype).double() * s["w"].double()).to(s["x"].dtype)
        out = {"values": _exact_quant(y, case["round"])}
        return out if s["res"] is None else out | {"residual": v}
    if kind == "silu":
        half = s["x"].shape[1] // 2
        g, u = s["x"][:, :half].double(), s["x"][:, half:].double()
        return {"values": _exact_quant(((g * torch.sigmoid(g)).to(s["x"].dtype).double() * u).to(s["x"].dtype), case["round"])}
    if kind == "mm":
        c = torch.matmul(_exact_values(s["a"], s["sa"]), _exact_values(s["w"].t(), s["sw"]).t())
        return {"out": c if s["bias"] is None else c + s["bias"].double()}
    rot, table = case["rot"], s["cs"].double()
    turn = torch.complex(table[s["pos"], :rot // 2], table[s["pos"], rot // 2:])[:, None]
    out = {}
    for name, weight in (("q", "qw"), ("k", "kw")):
        x = s[name].double()
        h = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * s[weight].double()
        at = torch.arange(rot // 2, device=h.device)
        i, j = (2 * at, 2 * at + 1) if case["inter"] else (at, at + rot // 2)
        z = torch.complex(h[..., i], h[..., j]) * turn
        h[..., i], h[..., j] = z.real, z.imag
        out[name] = h
    return out
