"""The MXFP4 operators and the q/k norm with its rotation from their definitions, in float64."""

from __future__ import annotations

import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_codes(peak: np.ndarray, rounded: bool) -> np.ndarray:
    """E8M0 codes of blocks with largest magnitudes `peak` (float64)."""
    with np.errstate(divide="ignore", invalid="ignore"):
        part, e = np.frexp(peak)                   # peak = part * 2^e, part in [1/2, 1)
    e = e.astype(np.int64) - 1 + (part >= 0.875) * bool(rounded)
    code = np.clip(e - 2 + 127, 0, 254)
    code[peak == 0] = 0
    code[~np.isfinite(peak)] = 255
    return code


def nearest_code(t: np.ndarray) -> np.ndarray:
    """E2M1 codes nearest to t (float64), of two equally near ones the even one; the sign in bit 3."""
    a = np.minimum(np.abs(t), 6.0)
    away = np.abs(a[..., None] - GRID)
    best = away.min(-1, keepdims=True)
    tie = away == best
    even = tie & (np.arange(8) % 2 == 0)
    pick = np.where(even.any(-1, keepdims=True), even, tie)
    return pick.argmax(-1) | (np.signbit(t) << 3)


def quant(x: np.ndarray, rounded: bool = False):
    """(codes [M, K/2], scales [M, K/32]) of float64 rows."""
    m, k = x.shape
    b = x.reshape(m, k // 32, 32)
    peak = np.where(np.isnan(b).any(-1), np.nan, np.abs(b).max(-1))
    s = scale_codes(peak, rounded)
    bad = (s == 255)[..., None]
    c = nearest_code(np.where(bad, 0.0, b) / np.exp2(np.where(bad, 127, s[..., None]) - 127.0))
    c = np.where(bad, 0, c).reshape(m, k).astype(np.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), s.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What codes and scales stand for, in float64."""
    t = np.concatenate([GRID, -GRID])
    v = np.empty((codes.shape[0], codes.shape[1] * 2))
    v[:, 0::2], v[:, 1::2] = t[codes & 15], t[codes >> 4]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return v * np.repeat(s, 32, 1)


def mm(a, sa, w, sw, bias=None):
    """(product, sum of the magnitudes of its terms), in float64."""
    x, y = values(a, sa), values(w, sw)
    out = x @ y.T
    return (out if bias is None else out + bias), np.abs(x) @ np.abs(y).T


def qk(x: torch.Tensor, w, cos_sin, positions, eps: float, interleaved: bool) -> torch.Tensor:
    """Normalized and rotated heads [T, H, D] in float64."""
    h = x.double()
    h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        h = h * w.double()
    rot = cos_sin.shape[1]
    inside = (positions >= 0) & (positions < cos_sin.shape[0])
    row = cos_sin.double()[torch.where(inside, positions, 0).long()]
    row = torch.where(inside[:, None], row, float("nan"))[:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out = h.clone()
    out[..., a] = h[..., a] * c - h[..., b] * s
    out[..., b] = h[..., b] * c + h[..., a] * s
    return out
