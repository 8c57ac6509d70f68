"""The norms of query and key heads with the position rotation, as one MI355X HIP kernel.

What stands between qkv_proj and the attention in the models of the Qwen3 family (and, without the
weights, in others): every head of the queries and keys is RMS-normalized over its own values, then
its first `rot` values are rotated in pairs by the token's position.

    qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps) -> (q, k)
    rope_cos_sin(max_positions, rot, base) -> the table of cosines and sines

The values are read in place from the columns of a qkv output.  Both steps are fp32 with one
rounding at the end.
"""

from __future__ import annotations

import torch

from int8_linear import _lib
from int8_linear.fused_quant import _act_code, _fast
from int8_linear.kernel import NotSupported, same_device

_FLOAT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


def rope_cos_sin(max_positions: int, rot: int, base: float = 1e6, *,
                 device: str | torch.device = "cuda",
                 dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[max_positions, rot]: the cosines of p * base^(-2i / rot) for i < rot / 2, then their sines.

    The angles are computed in float64: in float32 the angle of position 40960 is off by up to
    2e-3, which a bf16 result shows.
    """
    if rot <= 0 or rot % 2:
        raise ValueError(f"an even number of rotated values is needed, got {rot}")
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype)


def _heads(t: torch.Tensor, name: str, inplace: bool) -> int:
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head size], got {tuple(t.shape)}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise NotSupported(f"{name}: the values of a head must be contiguous")
    if inplace and t.numel():
        reach = 1   # the values that the inner dimensions span
        for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
            if size > 1 and stride < reach:
                raise ValueError(f"{name} overlaps itself (strides {t.stride()}): not in place")
            reach += (size - 1) * stride if size > 1 else 0
    return _act_code(t, name)


def _apart(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q and k share no memory: apart, or different columns of the same rows."""
    if not q.numel() or not k.numel():
        return True

    def span(t, dims):
        return t.element_size() * (sum((t.shape[d] - 1) * t.stride(d) for d in dims) + 1)

    a, b = sorted((q, k), key=lambda t: t.data_ptr())
    gap = b.data_ptr() - a.data_ptr()
    if gap >= span(a, (0, 1, 2)):
        return True
    row = a.stride(0) * a.element_size()
    return (a.shape[0] == b.shape[0] == 1 or a.stride(0) == b.stride(0)) and \
        gap >= span(a, (1, 2)) and (a.shape[0] == 1 or gap + span(b, (1, 2)) <= row)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                 k_weight: torch.Tensor | None, cos_sin: torch.Tensor, positions: torch.Tensor,
                 eps: float, *, interleaved: bool = False, inplace: bool = False):
    """Normalized and rotated (q [T, Hq, D], k [T, Hk, D]) of bf16 / fp16 heads.

    q and k may be views into a qkv output (any token and head strides, the values of a head
    contiguous).  q_weight and k_weight are the norms' [D] weights (bf16, fp16 or fp32, of one
    dtype), or None for a norm without.  cos_sin [positions, rot] (bf16, fp16 or fp32, contiguous) holds the
    cosines of the rot / 2 frequencies and then their sines; rot <= D is even, and the values past it
    are normalized only.  positions [T] (int32 or int64) picks the rows; a token whose position is
    outside the table gets NaN in its rotated values.  The pairs are (i, i + rot / 2), or
    (2i, 2i + 1) with interleaved.  With inplace, q and k are written over and returned.  There is no
    backward: heads, weights or a table that require a gradient are refused where gradients are
    recorded.
    """
    r = _fast("qk_norm_rope", q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, inplace)
    if r is not None:
        return r
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad
                                       for x in (q, k, q_weight, k_weight, cos_sin)):
        raise NotSupported("qk_norm_rope has no gradient: call it under torch.no_grad()")
    act = _heads(q, "q", inplace)
    if _heads(k, "k", inplace) != act:
        raise NotSupported(f"q and k must have one dtype, got {q.dtype} and {k.dtype}")
    if q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} are not heads of the same tokens")
    t, hq, d = q.shape
    hk = k.shape[1]
    same_device(q.device, k=k, q_weight=q_weight, k_weight=k_weight, cos_sin=cos_sin,
                positions=positions)
    w_code = _lib.DTYPE_NONE
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if tuple(w.shape) != (d,):
                raise ValueError(f"{name} must have shape ({d},), got {tuple(w.shape)}")
            code = _FLOAT.get(w.dtype)
            if code is None or w_code not in (_lib.DTYPE_NONE, code):
                raise NotSupported(f"{name}: bf16, fp16 or fp32 weights of one dtype, got {w.dtype}")
            w_code = code
            w = w.contiguous()
        weights.append(w)
    if cos_sin.dim() != 2 or cos_sin.shape[1] % 2 or not 2 <= cos_sin.shape[1] <= d:
        raise ValueError(f"cos_sin must be [positions, rot] with an even rot up to {d}, got "
                         f"{tuple(cos_sin.shape)}")
    cs_code = _FLOAT.get(cos_sin.dtype)
    if cs_code is None or not cos_sin.is_contiguous():
        raise NotSupported("cos_sin must be contiguous bf16, fp16 or fp32")
    if tuple(positions.shape) != (t,):
        raise ValueError(f"positions must have shape ({t},), got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise NotSupported(f"positions must be int32 or int64, got {positions.dtype}")
    positions = positions.contiguous()
    if inplace:
        if not _apart(q, k):
            raise ValueError("q and k overlap: they cannot be written in place")
        qo, ko = q, k
    else:
        qo = torch.empty((t, hq, d), dtype=q.dtype, device=q.device)
        ko = torch.empty((t, hk, d), dtype=q.dtype, device=q.device)

    def heads(x):
        return x.data_ptr(), x.stride(0), x.stride(1)

    with torch.cuda.device(q.device):
        status = _lib.lib().i8l_qk_norm_rope(
            *heads(q), *heads(k), *heads(qo), *heads(ko),
            *(w.data_ptr() if w is not None else None for w in weights), w_code, float(eps),
            cos_sin.data_ptr(), cs_code, cos_sin.shape[0], positions.data_ptr(),
            positions.element_size() * 8, t, hq, hk, d, cos_sin.shape[1], int(bool(interleaved)),
            act, _lib.stream_of(q))
    _lib.check(status, NotSupported)
    if inplace:   # the kernel writes past autograd, which counts the writes to what it saved
        torch.autograd.graph.increment_version((q, k))
    return qo, ko


@torch.library.custom_op("int8_linear::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                    k_weight: torch.Tensor | None, cos_sin: torch.Tensor, positions: torch.Tensor,
                    eps: float, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved=interleaved)


@qk_norm_rope_op.register_fake
def _(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)
