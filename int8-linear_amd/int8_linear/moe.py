"""The W8A8 linear over experts, as MI355X HIP kernels.

A layer with E experts sends each of T tokens to k of them.  Its (token, choice) pairs, ordered by
expert, are the rows of grouped products, in which every row is multiplied by its expert's weight:

    moe_route(logits, top_k) -> Routing(weights, experts, offsets, tokens, places)
    moe_order(experts, n_experts) -> (offsets, tokens, places)      of experts picked elsewhere
    w8a8_grouped_mm(a_q, b_q, scale_a, scale_b, offsets) -> [R, N]
    w8a8_grouped_mm_silu_mul(a_q, b_q, scale_a, scale_b, offsets) -> [R, N / 2]
    moe_combine(y, weights, places) -> [T, N]

so that the MLP of such a layer, with the per-token quantizers of fused_quant, is

    q, s = quant_per_token(x)
    r = moe_route(logits, 8)
    y = w8a8_grouped_mm_silu_mul(q, w13.transpose(1, 2), s, s13, r.offsets, rows=r.tokens)
    q, s = quant_per_token(y)
    y = w8a8_grouped_mm(q, w2.transpose(1, 2), s, s2, r.offsets)
    out = moe_combine(y, r.weights, r.places)

A token's row is quantized once and read by each of its experts in place (rows=), and nothing is
copied into expert order.  All sizes that the router decides stay on the device: no call waits for
them, and a captured graph can be replayed with other choices.  A rank that holds some of the experts
orders its own with moe_order (any expert outside [0, n_experts) is elsewhere); the rows from
offsets[n_experts] on are then not computed, and moe_combine leaves those pairs out.

Launches go on the caller's current stream and allocate nothing but the outputs and, for more than
64 tokens, the ordering's counts (up to 516 KiB).  There is no backward and no forward mode: what would
carry a gradient is refused where gradients are recorded, and what has a tangent in forward mode.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from int8_linear import _lib
from int8_linear.fused_quant import _fast
from int8_linear.kernel import NotSupported, same_device
from int8_linear.mxfp4 import _float_code, _ld, _no_gradient

SCORING = ("softmax", "sigmoid")


class Routing(NamedTuple):
    """What moe_route returns.  Row i of the grouped products belongs to token tokens[i] and to the
    expert e with offsets[e] <= i < offsets[e + 1]."""
    weights: torch.Tensor   # fp32 [T, k]
    experts: torch.Tensor   # int32 [T, k], -1 where none was left to pick
    offsets: torch.Tensor   # int32 [E + 1]
    tokens: torch.Tensor    # int32 [T * k], -1 from row offsets[E] on
    places: torch.Tensor    # int32 [T, k]: the row of each pair, -1 where it has no expert


def _order_outputs(t: int, e: int, k: int, need: int, device: torch.device):
    """The order's outputs and its workspace of `need` bytes (None of 0)."""
    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=device)
    return ints(e + 1), ints(t * k), ints(t, k), ints(need // 4) if need else None


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def moe_route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax",
              renormalize: bool = True) -> Routing:
    """The top_k experts of each token by its logits [T, E] (bf16, fp16 or fp32), and their order.

    The largest logits are picked, largest first, of equal ones the lower expert; one of -inf (an
    expert that the token may not take) or NaN is never picked, and where fewer than top_k are left
    the expert is -1 and the weight 0.  The weights, in fp32, are the picked experts' softmax over all
    experts, or their sigmoids; with renormalize they are divided by their sum.  The logits' rows may be any distance apart.  Up to 512 experts and 64 picks.
    """
    r = _fast("moe_route", logits, top_k, scoring, renormalize)
    if r is not None:
        return Routing(*r)
    _no_gradient("moe_route", logits)
    code = _float_code(logits.dtype, "logits")
    if not logits.is_cuda:
        raise NotSupported("logits must be on a HIP device")
    if scoring not in SCORING:
        raise ValueError(f"scoring must be one of {SCORING}, got {scoring!r}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got {tuple(logits.shape)}")
    t, e = logits.shape
    if not 1 <= top_k <= e:
        raise ValueError(f"cannot pick {top_k} of {e} experts")
    if e > 1 and logits.stride(1) != 1:
        raise NotSupported("logits need a unit column stride")
    if t > 1 and logits.stride(0) < e:
        logits = logits.contiguous()   # rows that share memory (an expanded matrix)
    weights = torch.empty((t, top_k), dtype=torch.float32, device=logits.device)
    experts = torch.empty((t, top_k), dtype=torch.int32, device=logits.device)
    need = _lib.lib().i8l_moe_route_workspace_bytes(t, e, top_k)
    offsets, tokens, places, ws = _order_outputs(t, e, top_k, need, logits.device)
    with torch.cuda.device(logits.device):
        status = _lib.lib().i8l_moe_route(
            logits.data_ptr(), _ld(logits), code, t, e, top_k, SCORING.index(scoring),
            int(bool(renormalize)), weights.data_ptr(), experts.data_ptr(), offsets.data_ptr(),
            tokens.data_ptr(), places.data_ptr(), _ptr(ws), need, _lib.stream_of(logits))
    _lib.check(status, NotSupported)
    return Routing(weights, experts, offsets, tokens, places)


def moe_order(experts: torch.Tensor, n_experts: int):
    """(offsets, tokens, places) of Routing for experts int32 [T, k] that were picked elsewhere.

    A value outside [0, n_experts) is a pair without an expert here: its place is -1.  (For experts
    [a, b) of more, pass experts - a and b - a.)  Pairs of one expert keep their order.
    """
    r = _fast("moe_order", experts, n_experts)
    if r is not None:
        return r
    if experts.dtype != torch.int32:
        raise NotSupported(f"experts must be int32, got {experts.dtype}")
    if not experts.is_cuda:
        raise NotSupported("experts must be on a HIP device")
    if experts.dim() != 2:
        raise ValueError(f"experts must be [tokens, choices], got {tuple(experts.shape)}")
    t, k = experts.shape
    if n_experts < 1 or k < 1:
        raise ValueError(f"{k} choices of {n_experts} experts")
    experts = experts.contiguous()
    need = _lib.lib().i8l_moe_order_workspace_bytes(t, n_experts, k)
    offsets, tokens, places, ws = _order_outputs(t, n_experts, k, need, experts.device)
    with torch.cuda.device(experts.device):
        status = _lib.lib().i8l_moe_order(experts.data_ptr(), t, n_experts, k, offsets.data_ptr(),
                                          tokens.data_ptr(), places.data_ptr(), _ptr(ws), need,
                                          _lib.stream_of(experts))
    _lib.check(status, NotSupported)
    return offsets, tokens, places


def _grouped(who: str, silu: bool, a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows, out):
    r = _fast("w8a8_grouped_mm", a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows, out, silu)
    if r is not None:
        return r
    _no_gradient(who, scale_a, scale_b, bias, out)
    out_code = _float_code(out_dtype, "the output")
    if a_q.dtype != torch.int8 or b_q.dtype != torch.int8:
        raise NotSupported(f"int8 operands only, got {a_q.dtype} and {b_q.dtype}")
    if scale_a.dtype != torch.float32 or scale_b.dtype != torch.float32:
        raise NotSupported(f"fp32 scales only, got {scale_a.dtype} and {scale_b.dtype}")
    if offsets.dtype != torch.int32 or (rows is not None and rows.dtype != torch.int32):
        raise NotSupported("offsets and rows must be int32")
    if not a_q.is_cuda:
        raise NotSupported("a_q must be on a HIP device")
    if a_q.dim() != 2 or b_q.dim() != 3 or a_q.shape[1] != b_q.shape[1]:
        raise ValueError(f"cannot multiply {tuple(a_q.shape)} by experts' {tuple(b_q.shape)}")
    m, k = a_q.shape
    e, n = b_q.shape[0], b_q.shape[2]
    if not e or not k:
        raise ValueError(f"{e} experts, K of {k}")
    if silu and n % 2:
        raise ValueError(f"{n} columns are not gate and up halves")
    if tuple(offsets.shape) != (e + 1,):
        raise ValueError(f"offsets must have shape ({e + 1},), got {tuple(offsets.shape)}")
    if rows is not None and rows.dim() != 1:
        raise ValueError(f"rows must be a vector, got {tuple(rows.shape)}")
    if tuple(scale_a.shape) not in ((m,), (m, 1), (1,), (1, 1), ()):
        raise ValueError(f"scale_a must have {m} values or one, got {tuple(scale_a.shape)}")
    if tuple(scale_b.shape) not in ((e, n), (e, n, 1)):
        raise ValueError(f"scale_b must have shape ({e}, {n}), got {tuple(scale_b.shape)}")
    if (k > 1 and a_q.stride(1) != 1) or (k > 1 and b_q.stride(1) != 1):
        raise NotSupported("a_q and b_q must be contiguous along K")
    same_device(a_q.device, b_q=b_q, scale_a=scale_a, scale_b=scale_b, offsets=offsets, bias=bias,
                rows=rows, out=out)
    bias_code = _lib.DTYPE_NONE
    if bias is not None:
        if tuple(bias.shape) != (e, n):
            raise ValueError(f"bias must have shape ({e}, {n}), got {tuple(bias.shape)}")
        bias = bias.contiguous()
        bias_code = _float_code(bias.dtype, "bias")
    scale_a, scale_b, offsets = scale_a.contiguous(), scale_b.contiguous(), offsets.contiguous()
    if rows is not None:
        rows = rows.contiguous()
    r, width = m if rows is None else rows.shape[0], n // 2 if silu else n
    if out is None:
        out = torch.empty((r, width), dtype=out_dtype, device=a_q.device)
    else:
        if tuple(out.shape) != (r, width) or out.dtype != out_dtype:
            raise ValueError(f"out must be {out_dtype} ({r}, {width}), got {out.dtype} "
                             f"{tuple(out.shape)}")
        if (width > 1 and out.stride(1) != 1) or (r > 1 and out.stride(0) < width):
            raise NotSupported("out needs a unit column stride and rows that do not overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise NotSupported("out requires a gradient")
    with torch.cuda.device(a_q.device):
        status = _lib.lib().i8l_w8a8_grouped_mm(
            a_q.data_ptr(), _ld(a_q), m, _ptr(rows), b_q.data_ptr(), b_q.stride(0),
            b_q.stride(2) if n > 1 else k, scale_a.data_ptr(), scale_a.numel(), scale_b.data_ptr(),
            _ptr(bias), bias_code, offsets.data_ptr(), out.data_ptr(), _ld(out), out_code, int(silu),
            r, e, n, k, _lib.stream_of(a_q))
    _lib.check(status, NotSupported)
    return out


def _written(out: torch.Tensor | None) -> None:
    """The kernel writes past autograd, which counts the writes to what it saved."""
    if out is not None:
        torch.autograd.graph.increment_version(out)


def w8a8_grouped_mm(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor,
                    scale_b: torch.Tensor, offsets: torch.Tensor,
                    out_dtype: torch.dtype = torch.bfloat16, bias: torch.Tensor | None = None, *,
                    rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """w8a8_mm of each row with its expert's weight: [R, N] in out_dtype (bf16, fp16 or fp32).

    a_q int8 [M, K] and scale_a fp32 ([M], [M, 1] or one value) as for w8a8_mm; b_q = w_q.transpose(1, 2)
    int8 [E, K, N] of a weight w_q [E, N, K], scale_b fp32 [E, N] or [E, N, 1], bias [E, N].  Expert
    e's rows are offsets[e] to offsets[e + 1] - 1 (int32 [E + 1]); row i reads a_q[rows[i]] with its
    scale, or a_q[i] without rows.  The arithmetic is w8a8_mm's, bit for bit.  `out` [R, N] (unit
    column stride) takes the result; rows of no expert (before offsets[0], from offsets[E] on) are left as
    they were there, and in a new output hold anything.  A row outside a_q gives NaN; an offset outside [0, R] or below an earlier
    one is held to those.  There is no backward: scales, a bias or an out that require a gradient are refused
    where gradients are recorded.
    """
    o = _grouped("w8a8_grouped_mm", False, a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows, out)
    _written(out)
    return o


def w8a8_grouped_mm_silu_mul(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor,
                             scale_b: torch.Tensor, offsets: torch.Tensor,
                             out_dtype: torch.dtype = torch.bfloat16,
                             bias: torch.Tensor | None = None, *, rows: torch.Tensor | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """w8a8_grouped_mm of gate and up weights with silu(gate) * up: [R, N / 2] in out_dtype.

    b_q [E, K, N] holds the gate columns and then the up columns.  The products, the SiLU and its
    product with up stay in fp32 and are rounded once (w8a8_mm_silu_mul rounds each to bf16 on the
    way).  Everything else is as in w8a8_grouped_mm.
    """
    o = _grouped("w8a8_grouped_mm_silu_mul", True, a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias,
                 rows, out)
    _written(out)
    return o


def moe_combine(y: torch.Tensor, weights: torch.Tensor, places: torch.Tensor, *,
                base: torch.Tensor | None = None) -> torch.Tensor:
    """(base[t] +) sum_j weights[t, j] * y[places[t, j]]: [T, N] in y's dtype (bf16, fp16 or fp32).

    y [R, N] are the grouped product's rows (unit column stride), weights fp32 and places int32
    [T, k]; base [T, N], of y's dtype, what is added to (a shared expert's output, the residual).
    Summed in fp32 in the order of j, rounded once.  A place outside [0, R) adds nothing, whatever
    stands there.  There is no backward: inputs that require a gradient are refused where gradients
    are recorded.
    """
    r = _fast("moe_combine", y, weights, places, base)
    if r is not None:
        return r
    _no_gradient("moe_combine", y, weights, base)
    code = _float_code(y.dtype, "y")
    if not y.is_cuda:
        raise NotSupported("y must be on a HIP device")
    if weights.dtype != torch.float32 or places.dtype != torch.int32:
        raise NotSupported(f"fp32 weights and int32 places, got {weights.dtype} and {places.dtype}")
    if y.dim() != 2 or places.dim() != 2 or weights.shape != places.shape or not places.shape[1]:
        raise ValueError(f"y {tuple(y.shape)}, weights {tuple(weights.shape)} and places "
                         f"{tuple(places.shape)} do not belong together")
    t, k = places.shape
    rows, n = y.shape
    if base is not None:
        if tuple(base.shape) != (t, n):
            raise ValueError(f"base must have shape ({t}, {n}), got {tuple(base.shape)}")
        if base.dtype != y.dtype:
            raise NotSupported(f"base must be {y.dtype}, got {base.dtype}")
    same_device(y.device, weights=weights, places=places, base=base)

    def spaced(x):   # unit column stride, rows that do not overlap
        if (n > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < n):
            return x.contiguous()
        return x

    y, base = spaced(y), spaced(base) if base is not None else None
    weights, places = weights.contiguous(), places.contiguous()
    out = torch.empty((t, n), dtype=y.dtype, device=y.device)
    with torch.cuda.device(y.device):
        status = _lib.lib().i8l_moe_combine(
            y.data_ptr(), _ld(y), rows, weights.data_ptr(), places.data_ptr(), _ptr(base),
            _ld(base) if base is not None else n, out.data_ptr(), t, k, n, code, _lib.stream_of(y))
    _lib.check(status, NotSupported)
    return out


@torch.library.custom_op("int8_linear::moe_route", mutates_args=())
def moe_route_op(logits: torch.Tensor, top_k: int, scoring: str, renormalize: bool) -> tuple[
        torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(moe_route(logits, top_k, scoring=scoring, renormalize=renormalize))


@moe_route_op.register_fake
def _(logits, top_k, scoring, renormalize):
    t, e = logits.shape
    pairs = logits.new_empty((t, top_k), dtype=torch.int32)
    return (logits.new_empty((t, top_k), dtype=torch.float32), pairs,
            pairs.new_empty((e + 1,)), pairs.new_empty((t * top_k,)), torch.empty_like(pairs))


@torch.library.custom_op("int8_linear::moe_order", mutates_args=())
def moe_order_op(experts: torch.Tensor, n_experts: int) -> tuple[torch.Tensor, torch.Tensor,
                                                                 torch.Tensor]:
    return moe_order(experts, n_experts)


@moe_order_op.register_fake
def _(experts, n_experts):
    return (experts.new_empty((n_experts + 1,)), experts.new_empty((experts.numel(),)),
            experts.new_empty(experts.shape))


@torch.library.custom_op("int8_linear::w8a8_grouped_mm", mutates_args=())
def w8a8_grouped_mm_op(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor,
                       scale_b: torch.Tensor, offsets: torch.Tensor, out_dtype: torch.dtype,
                       bias: torch.Tensor | None, rows: torch.Tensor | None) -> torch.Tensor:
    return w8a8_grouped_mm(a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows=rows)


@w8a8_grouped_mm_op.register_fake
def _(a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows):
    m = a_q.shape[0] if rows is None else rows.shape[0]
    return a_q.new_empty((m, b_q.shape[2]), dtype=out_dtype)


@torch.library.custom_op("int8_linear::w8a8_grouped_mm_silu_mul", mutates_args=())
def w8a8_grouped_mm_silu_mul_op(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor,
                                scale_b: torch.Tensor, offsets: torch.Tensor,
                                out_dtype: torch.dtype, bias: torch.Tensor | None,
                                rows: torch.Tensor | None) -> torch.Tensor:
    return w8a8_grouped_mm_silu_mul(a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows=rows)


@w8a8_grouped_mm_silu_mul_op.register_fake
def _(a_q, b_q, scale_a, scale_b, offsets, out_dtype, bias, rows):
    m = a_q.shape[0] if rows is None else rows.shape[0]
    return a_q.new_empty((m, b_q.shape[2] // 2), dtype=out_dtype)


@torch.library.custom_op("int8_linear::moe_combine", mutates_args=())
def moe_combine_op(y: torch.Tensor, weights: torch.Tensor, places: torch.Tensor,
                   base: torch.Tensor | None) -> torch.Tensor:
    return moe_combine(y, weights, places, base=base)


@moe_combine_op.register_fake
def _(y, weights, places, base):
    return y.new_empty((places.shape[0], y.shape[1]))
