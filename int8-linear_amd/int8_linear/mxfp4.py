"""The microscaled 4-bit (MXFP4) form of the linear path, as MI355X HIP kernels.

An MXFP4 matrix [R, K] is two uint8 tensors, as the OCP microscaling format lays them out: codes
[R, K/2], two E2M1 elements a byte (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; the even element
in the low nibble), and scales [R, K/32], one E8M0 byte for each 32 elements (2^(byte - 127), 255 is
NaN).  K is a multiple of 32.

    mxfp4_quant(x) -> (codes, scales)                    any bf16 / fp16 / fp32 matrix
    mxfp4_dequant(codes, scales) -> values
    add_rmsnorm_mxfp4_quant(x, residual, w, eps) -> (codes, scales, residual_out)
    silu_mul_mxfp4_quant(gate_up) -> (codes, scales)
    mxfp4_mm(a_q, b_q, scale_a, scale_b, out_dtype, bias) -> [M, N]

A weight [N, K] is quantized once, by mxfp4_quant or by whoever wrote the checkpoint, and passed as
the transposed view w_q.t() [K/2, N], as w8a8_mm takes an int8 one; the activations are quantized
for each call.  Both operands' scales enter the matrix instructions themselves
(v_mfma_scale_f32_*_f8f6f4), which accumulate in fp32.  A linear reads 17/32 of a byte a weight,
0.53 of the int8 path's, and the instruction does twice the int8 one's operations.

Launches go on the caller's current stream and allocate nothing but the outputs, and where a product
of 33 to 4096 tokens has too few tiles for the card and its K is cut into parts, the parts' sums (up to
64 MiB; 14336 -> 4096: from 81 to 640 tokens).

There is no backward.  Codes and scales are integers and carry no gradient; a call whose floating
output would lose one is refused.
"""

from __future__ import annotations

import torch

from int8_linear import _lib
from int8_linear.fused_quant import _act_code, _fast
from int8_linear.kernel import NotSupported, same_device

BLOCK = 32

_FLOAT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_CODES = tuple(t for t in (torch.uint8, getattr(torch, "float4_e2m1fn_x2", None)) if t)
_SCALES = tuple(t for t in (torch.uint8, getattr(torch, "float8_e8m0fnu", None)) if t)


def _float_code(dtype: torch.dtype, what: str) -> int:
    code = _FLOAT.get(dtype)
    if code is None:
        raise NotSupported(f"{what} must be bfloat16, float16 or float32, got {dtype}")
    return code


def _matrix(codes: torch.Tensor, scales: torch.Tensor, what: str):
    """codes [R, K/2] and scales [R, K/32] as uint8, checked against each other."""
    if codes.dtype not in _CODES or scales.dtype not in _SCALES:
        raise NotSupported(f"{what}: uint8 codes and scales only, got {codes.dtype} and {scales.dtype}")
    if not codes.is_cuda:
        raise NotSupported(f"{what} must be on a HIP device")
    if codes.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"{what}: codes and scales are matrices, got {codes.dim()} and "
                         f"{scales.dim()} dimensions")
    rows, k = codes.shape[0], 2 * codes.shape[1]
    if k == 0 or k % BLOCK:
        raise ValueError(f"{what}: rows of {k} values are not whole blocks of {BLOCK}")
    if tuple(scales.shape) != (rows, k // BLOCK):
        raise ValueError(f"{what}: codes of {rows} rows of {k} need scales ({rows}, {k // BLOCK}), "
                         f"got {tuple(scales.shape)}")
    if codes.stride(1) != 1 or (scales.stride(1) != 1 and scales.shape[1] > 1):
        raise NotSupported(f"{what}: codes and scales must be contiguous along K")
    return codes.view(torch.uint8), scales.view(torch.uint8)


def _no_gradient(who: str, *inputs: torch.Tensor | None) -> None:
    """Refuses inputs whose gradient a floating output of `who` would lose."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        raise NotSupported(f"{who} has no gradient: call it under torch.no_grad()")


def _ld(t: torch.Tensor) -> int:
    """The row stride; of one row, its length."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _outputs(m: int, k: int, device: torch.device):
    if k == 0 or k % BLOCK:
        raise ValueError(f"rows of {k} values are not whole blocks of {BLOCK}")
    return (torch.empty((m, k // 2), dtype=torch.uint8, device=device),
            torch.empty((m, k // BLOCK), dtype=torch.uint8, device=device))


def mxfp4_quant(x: torch.Tensor, round_scale: bool = False):
    """(codes uint8 [M, K/2], scales uint8 [M, K/32]) of a bf16 / fp16 / fp32 matrix [M, K].

    The scale of a block whose largest magnitude is p is 2^(floor(log2 p) - 2) (the OCP rule:
    p / scale lies in [4, 8) and what is past 6 saturates); with round_scale, p is first rounded to
    E2M1's one mantissa bit, so peaks from 1.75 * 2^e take the next scale.  Elements are rounded
    to nearest even.  A block that holds an infinity or a NaN gets the NaN scale.  x may be a
    column slice of a wider matrix (unit column stride, any row stride).
    """
    r = _fast("mxfp4_quant", x, round_scale)
    if r is not None:
        return r
    code = _float_code(x.dtype, "x")
    if not x.is_cuda:
        raise NotSupported("x must be on a HIP device")
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, got {x.dim()} dimensions")
    m, k = x.shape
    q, s = _outputs(m, k, x.device)
    if x.stride(1) != 1:
        raise NotSupported("x needs a unit column stride")
    if m > 1 and x.stride(0) < k:
        x = x.contiguous()   # rows that share memory (an expanded matrix)
    with torch.cuda.device(x.device):
        status = _lib.lib().i8l_mxfp4_quant(x.data_ptr(), _ld(x), q.data_ptr(), s.data_ptr(), m, k,
                                            code, int(bool(round_scale)), _lib.stream_of(x))
    _lib.check(status, NotSupported)
    return q, s


def mxfp4_dequant(codes: torch.Tensor, scales: torch.Tensor,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [M, K] that codes [M, K/2] and scales [M, K/32] stand for: exact in bf16 and fp32,
    but for 2^128 and more, which is infinite (fp16 rounds below its range and overflows above it);
    NaN where the scale is."""
    r = _fast("mxfp4_dequant", codes, scales, out_dtype)
    if r is not None:
        return r
    code = _float_code(out_dtype, "the output")
    codes, scales = _matrix(codes, scales, "mxfp4_dequant")
    same_device(codes.device, scales=scales)
    m, k = codes.shape[0], 2 * codes.shape[1]
    if m > 1 and codes.stride(0) < k // 2:
        codes = codes.contiguous()
    if m > 1 and scales.stride(0) < k // BLOCK:
        scales = scales.contiguous()
    out = torch.empty((m, k), dtype=out_dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        status = _lib.lib().i8l_mxfp4_dequant(codes.data_ptr(), _ld(codes), scales.data_ptr(),
                                              _ld(scales), out.data_ptr(), m, k, code,
                                              _lib.stream_of(codes))
    _lib.check(status, NotSupported)
    return out


def add_rmsnorm_mxfp4_quant(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                            eps: float, round_scale: bool = False):
    """mxfp4_quant of add_rmsnorm's row, as one kernel: (codes, scales, residual_out or None).

    The values that are quantized are those of fused_quant.add_rmsnorm_quant bit for bit: the
    residual add and the norm in fp32, the normalized value rounded to the weight's dtype, times the
    weight, rounded to x's dtype.  x and residual are contiguous bf16 / fp16 [M, K], weight [K].
    There is no backward: where gradients are recorded, an x or a residual that requires one is
    refused with a residual, whose sum with x is returned (codes are integers and have none).
    """
    r = _fast("add_rmsnorm_mxfp4_quant", x, residual, weight, eps, round_scale)
    if r is not None:
        return r
    if residual is not None:
        _no_gradient("add_rmsnorm_mxfp4_quant", x, residual)
    act, wcode = _act_code(x, "x"), _act_code(weight, "weight")
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, got {x.dim()} dimensions")
    m, k = x.shape
    if weight.numel() != k:
        raise ValueError(f"weight has {weight.numel()} values for rows of {k}")
    if not x.is_contiguous():
        raise NotSupported("x must be contiguous")
    weight = weight.contiguous()
    same_device(x.device, weight=weight, residual=residual)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} for x {tuple(x.shape)}")
        if residual.dtype != x.dtype or not residual.is_contiguous():
            raise NotSupported("residual must be contiguous and of x's dtype")
    q, s = _outputs(m, k, x.device)
    rout = torch.empty_like(x) if residual is not None else None
    with torch.cuda.device(x.device):
        status = _lib.lib().i8l_add_rmsnorm_mxfp4_quant(
            x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(),
            float(eps), q.data_ptr(), s.data_ptr(), rout.data_ptr() if rout is not None else None,
            m, k, act, wcode, int(bool(round_scale)), _lib.stream_of(x))
    _lib.check(status, NotSupported)
    return q, s, rout


def silu_mul_mxfp4_quant(gate_up: torch.Tensor, round_scale: bool = False):
    """mxfp4_quant of silu(gate) * up, as one kernel: (codes [M, I/2], scales [M, I/32]).

    The values that are quantized are those of fused_quant.silu_mul_quant with round_silu bit for
    bit: the SiLU rounded to gate_up's dtype, as the served models compute it, and its product with
    up rounded again.  gate_up is contiguous bf16 / fp16 [M, 2I], the gate values first.
    """
    r = _fast("silu_mul_mxfp4_quant", gate_up, round_scale)
    if r is not None:
        return r
    act = _act_code(gate_up, "gate_up")
    if gate_up.dim() != 2 or gate_up.shape[1] % 2:
        raise ValueError(f"gate_up must be a matrix of gate and up halves, got {tuple(gate_up.shape)}")
    if not gate_up.is_contiguous():
        raise NotSupported("gate_up must be contiguous")
    m, i = gate_up.shape[0], gate_up.shape[1] // 2
    q, s = _outputs(m, i, gate_up.device)
    with torch.cuda.device(gate_up.device):
        status = _lib.lib().i8l_silu_mul_mxfp4_quant(gate_up.data_ptr(), q.data_ptr(), s.data_ptr(),
                                                     m, i, act, int(bool(round_scale)),
                                                     _lib.stream_of(gate_up))
    _lib.check(status, NotSupported)
    return q, s


def mxfp4_mm(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
             out_dtype: torch.dtype = torch.bfloat16,
             bias: torch.Tensor | None = None) -> torch.Tensor:
    """A @ W^T (+ bias) of two MXFP4 matrices: [M, N] in out_dtype (bf16, fp16 or fp32).

    a_q [M, K/2] and scale_a [M, K/32] are the activations', scale_b [N, K/32] and b_q = w_q.t()
    [K/2, N] the weight's (codes contiguous along K).  Accumulated in fp32, the bias [N] added in
    fp32, rounded once.  There is no backward: a bias that requires a gradient is refused where
    gradients are recorded.

    Which kernel runs goes by the sizes and the alignment (the same results up to the order of the
    fp32 sums).  Prompts are fast where K is a multiple of 512 from 1024 on, N of 8 from 128 on, and
    the codes, the scales, the bias and their rows start on 16 bytes; elsewhere they take the kernels
    for few tokens, at 4096 tokens 6 to 13 times as long.  Rows of codes that do not start on 16 bytes
    take a slow kernel without matrix instructions.
    """
    r = _fast("mxfp4_mm", a_q, b_q, scale_a, scale_b, out_dtype, bias)
    if r is not None:
        return r
    _no_gradient("mxfp4_mm", bias)
    out_code = _float_code(out_dtype, "the output")
    if a_q.dim() != 2 or b_q.dim() != 2 or a_q.shape[1] != b_q.shape[0]:
        raise ValueError(f"cannot multiply codes {tuple(a_q.shape)} by {tuple(b_q.shape)}")
    a_q, scale_a = _matrix(a_q, scale_a, "a_q")
    w_q, scale_b = _matrix(b_q.t(), scale_b, "b_q")
    same_device(a_q.device, b_q=w_q, scale_a=scale_a, scale_b=scale_b, bias=bias)
    m, n, k = a_q.shape[0], w_q.shape[0], 2 * a_q.shape[1]
    bias_code = _lib.DTYPE_NONE
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
        bias_code = _float_code(bias.dtype, "bias")
    # rows that share memory (expanded operands) are read through a copy
    a_q, w_q, scale_a, scale_b = (t if t.shape[0] <= 1 or t.stride(0) >= t.shape[1] else t.contiguous()
                                  for t in (a_q, w_q, scale_a, scale_b))
    out = torch.empty((m, n), dtype=out_dtype, device=a_q.device)
    # the fp32 sums of a split of K, from the caching allocator (the graph's pool under capture)
    need = _lib.lib().i8l_mxfp4_mm_workspace_bytes(m, n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=a_q.device) if need else None
    with torch.cuda.device(a_q.device):
        status = _lib.lib().i8l_mxfp4_mm_ws(
            a_q.data_ptr(), _ld(a_q), w_q.data_ptr(), _ld(w_q), scale_a.data_ptr(), _ld(scale_a),
            scale_b.data_ptr(), _ld(scale_b), bias.data_ptr() if bias is not None else None,
            bias_code, out.data_ptr(), n, out_code, m, n, k, ws.data_ptr() if need else None, need,
            _lib.stream_of(a_q))
    _lib.check(status, NotSupported)
    return out


@torch.library.custom_op("int8_linear::mxfp4_quant", mutates_args=())
def mxfp4_quant_op(x: torch.Tensor, round_scale: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return mxfp4_quant(x.contiguous(), round_scale)


def _fake_pair(x: torch.Tensor, k: int):
    return (x.new_empty((x.shape[0], k // 2), dtype=torch.uint8),
            x.new_empty((x.shape[0], k // BLOCK), dtype=torch.uint8))


@mxfp4_quant_op.register_fake
def _(x, round_scale):
    return _fake_pair(x, x.shape[1])


@torch.library.custom_op("int8_linear::add_rmsnorm_mxfp4_quant", mutates_args=())
def add_rmsnorm_mxfp4_quant_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                               eps: float, round_scale: bool) -> tuple[torch.Tensor, torch.Tensor,
                                                                       torch.Tensor]:
    return add_rmsnorm_mxfp4_quant(x.contiguous(), residual.contiguous(), weight, eps, round_scale)


@add_rmsnorm_mxfp4_quant_op.register_fake
def _(x, residual, weight, eps, round_scale):
    return (*_fake_pair(x, x.shape[1]), x.new_empty(x.shape))


@torch.library.custom_op("int8_linear::silu_mul_mxfp4_quant", mutates_args=())
def silu_mul_mxfp4_quant_op(gate_up: torch.Tensor, round_scale: bool) -> tuple[torch.Tensor,
                                                                               torch.Tensor]:
    return silu_mul_mxfp4_quant(gate_up.contiguous(), round_scale)


@silu_mul_mxfp4_quant_op.register_fake
def _(gate_up, round_scale):
    return _fake_pair(gate_up, gate_up.shape[1] // 2)


@torch.library.custom_op("int8_linear::mxfp4_mm", mutates_args=())
def mxfp4_mm_op(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                out_dtype: torch.dtype, bias: torch.Tensor | None) -> torch.Tensor:
    return mxfp4_mm(a_q, b_q, scale_a, scale_b, out_dtype, bias)


@mxfp4_mm_op.register_fake
def _(a_q, b_q, scale_a, scale_b, out_dtype, bias):
    return a_q.new_empty((a_q.shape[0], b_q.shape[1]), dtype=out_dtype)
