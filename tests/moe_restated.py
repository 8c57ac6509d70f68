"""The operators of a layer over experts, restated in plain torch on the CPU from their definitions:
picks and order by Python's own sorting, products in float64 (exact for int8), the epilogue in the
float32 steps the definition names."""

from __future__ import annotations

import math

import torch


def picks(logits: torch.Tensor, k: int) -> torch.Tensor:
    """int32 [T, k]: the k largest, of equal ones the lower index; -1 where none is left."""
    out = []
    for row in logits.double().tolist():
        able = [e for e, x in enumerate(row) if x > -math.inf]       # (a NaN compares as false)
        able.sort(key=lambda e: (-row[e], e))
        out.append((able + [-1] * k)[:k])
    return torch.tensor(out, dtype=torch.int32).reshape(logits.shape[0], k)


def weights(logits: torch.Tensor, experts: torch.Tensor, scoring: str, renormalize: bool) -> torch.Tensor:
    """float64 [T, k]."""
    x = logits.double()
    able = x > -math.inf
    x = torch.where(able, x, -math.inf)
    if scoring == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.where(x == top, 1.0, torch.exp(x - torch.where(top.isinf(), 0.0, top)))
        p = torch.where(top == math.inf, (x == top).double(), p)
    elif renormalize:   # over the largest of the row, so that logits far below 0 keep their ratios
        log = torch.nn.functional.logsigmoid(x)
        p = torch.exp(log - log.amax(1, keepdim=True).clamp(min=-1e300))
    else:
        p = torch.sigmoid(x)
    p = torch.where(able, p, 0.0)
    got = experts >= 0
    w = torch.where(got, p.gather(1, experts.clamp(min=0).long()), 0.0)
    total = w.sum(1, keepdim=True) if renormalize else \
        p.sum(1, keepdim=True) if scoring == "softmax" else torch.ones(len(x), 1, dtype=torch.float64)
    return torch.where(total > 0, w / total, 0.0)


def order(experts: torch.Tensor, n_experts: int):
    """(offsets, tokens, places) by a stable sort of the pairs."""
    t, k = experts.shape
    flat = experts.flatten().tolist()
    rows = sorted((i for i, e in enumerate(flat) if 0 <= e < n_experts), key=lambda i: (flat[i], i))
    places, tokens = [-1] * (t * k), [-1] * (t * k)
    for at, i in enumerate(rows):
        places[i], tokens[at] = at, i // k
    offsets = [sum(1 for i in rows if flat[i] < e) for e in range(n_experts + 1)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32)
    return ints(offsets), ints(tokens), ints(places).reshape(t, k)


def grouped(a, w, sa, sb, offsets, bias=None, rows=None) -> torch.Tensor:
    """fp32 [R, N]: the epilogue's values before the last rounding; NaN in the rows of no expert."""
    a, w, sa, sb = a.cpu(), w.cpu(), sa.cpu().reshape(-1), sb.cpu().reshape(w.shape[0], w.shape[1])
    ends = offsets.tolist()
    r = a.shape[0] if rows is None else rows.numel()
    src = torch.arange(r) if rows is None else rows.cpu().long()
    out = torch.full((r, w.shape[1]), math.nan)
    for e in range(w.shape[0]):
        lo, hi = ends[e], ends[e + 1]
        if lo < hi:
            acc = a[src[lo:hi]].double() @ w[e].double().t()
            assert acc.abs().max() < 2 ** 31
            v = acc.float() * (sa[src[lo:hi]] if sa.numel() > 1 else sa.expand(hi - lo))[:, None]
            v = v * sb[e]
            out[lo:hi] = v if bias is None else v + bias[e].cpu().float()
    return out


def silu_mul(v: torch.Tensor) -> torch.Tensor:
    """float64 silu(gate) * up of the epilogue's fp32 values."""
    g, u = v.double().chunk(2, 1)
    return g * torch.sigmoid(g) * u


def combine(y, w, places, base=None):
    """(float64 sum, float64 sum of magnitudes) [T, N]."""
    y, w, places = y.cpu().double(), w.cpu().double(), places.cpu().long()
    out = torch.zeros(places.shape[0], y.shape[1], dtype=torch.float64)
    size = out.clone()
    if base is not None:
        out, size = out + base.cpu().double(), size + base.cpu().double().abs()
    for j in range(places.shape[1]):
        has = (places[:, j] >= 0) & (places[:, j] < y.shape[0])
        term = y[places[has, j]] * w[has, j, None]
        out[has] += term
        size[has] += term.abs()
    return out, size
