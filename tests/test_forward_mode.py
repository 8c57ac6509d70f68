"""Under forward differentiation a floating output that depends on an input with a tangent is refused, as
there is no rule to carry it: the value alone would read as a derivative of zero."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from int8_linear import NotSupported, moe, mxfp4, qk_rope


def _i8(*shape):
    return torch.ones(shape, dtype=torch.int8)


def _grouped(call):
    def run(a, b, sa, sb, off, bias, out):
        return call(a, b.transpose(1, 2), sa, sb, off, torch.float32, bias, out=out)
    width = 16 if call is moe.w8a8_grouped_mm_silu_mul else 32
    args = (_i8(6, 64), _i8(2, 32, 64), torch.ones(6, 1), torch.ones(2, 32),
            torch.tensor([0, 2, 6], dtype=torch.int32), torch.zeros(2, 32), torch.zeros(6, width))
    return run, args, (2, 3, 5, 6)


def _combine():
    places = torch.tensor([[0, 3], [2, -1]], dtype=torch.int32)
    return (lambda y, w, p, base: moe.moe_combine(y, w, p, base=base),
            (torch.ones(4, 8), torch.ones(2, 2), places, torch.ones(2, 8)), (0, 1, 3))


def _mx_mm():
    q, s = torch.full((4, 32), 0x22, dtype=torch.uint8), torch.full((4, 2), 127, dtype=torch.uint8)
    return (lambda q, s, bias: mxfp4.mxfp4_mm(q, q.t(), s, s, torch.float32, bias),
            (q, s, torch.zeros(4)), (2,))


def _mx_norm():
    x = torch.ones(4, 64).bfloat16()
    return (lambda x, r, w: mxfp4.add_rmsnorm_mxfp4_quant(x, r, w, 1e-6),
            (x, x.clone(), torch.ones(64).bfloat16()), (0, 1))


def _rope():
    h, pos = torch.ones(2, 3, 64).bfloat16(), torch.arange(2)
    return (lambda q, k, qw, kw, cs, pos: qk_rope.qk_norm_rope(q, k, qw, kw, cs, pos, 1e-6),
            (h, h[:, :1].clone(), torch.ones(64), torch.ones(64), torch.ones(8, 64), pos), (0, 1, 2, 3, 4))


CALLS = {"route": (lambda x: moe.moe_route(x, 2), (torch.arange(12.0).view(3, 4),), (0,)),
         "combine": _combine(), "mm": _grouped(moe.w8a8_grouped_mm),
         "silu": _grouped(moe.w8a8_grouped_mm_silu_mul), "mxfp4 mm": _mx_mm(), "mxfp4 norm": _mx_norm(),
         "rope": _rope()}
EACH = [(name, i) for name, (_, _, which) in CALLS.items() for i in which]


def _dual(args, i):
    return [forward_ad.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]


@pytest.mark.parametrize("name,i", EACH)
def test_a_lost_tangent_is_refused(name, i):
    run, args, _ = CALLS[name]
    with forward_ad.dual_level():
        duals = _dual(args, i)
        with pytest.raises(NotSupported, match="gradient"):
            run(*duals)
        with torch.no_grad(), pytest.raises(NotSupported, match="gradient"):   # (tangents go on there)
            run(*duals)
        with torch.inference_mode(), pytest.raises(NotSupported, match="HIP device"):   # (but not there)
            run(*duals)


def test_a_call_under_jvp_is_refused():
    with pytest.raises(NotSupported, match="gradient"):
        torch.func.jvp(lambda x: moe.moe_route(x, 2).weights, (torch.ones(3, 4),), (torch.ones(3, 4),))


def test_codes_have_no_tangent_to_lose():
    """Quantizers give integers: the call goes on to its other checks."""
    with forward_ad.dual_level():
        x, = _dual([torch.ones(4, 64)], 0)
        with pytest.raises(NotSupported, match="HIP device"):
            mxfp4.mxfp4_quant(x)


@pytest.mark.gpu
@pytest.mark.parametrize("name,i", EACH)
def test_the_binding_refuses_it_too(name, i):
    run, args, _ = CALLS[name]
    args = [a.cuda() for a in args]
    want = [t.clone() for t in _tensors(run(*args))]
    with forward_ad.dual_level():
        duals = _dual(args, i)
        with pytest.raises(NotSupported, match="gradient"):
            run(*duals)
        with torch.inference_mode():
            _same(run(*duals), want)
        _same(run(*args), want)
    _same(run(*duals), want)


def _tensors(out):
    return [out] if isinstance(out, torch.Tensor) else [t for t in out if t is not None]


def _same(out, want):
    assert all(torch.equal(a, b) for a, b in zip(_tensors(out), want, strict=True))


@pytest.mark.gpu
def test_a_level_without_tangents_keeps_the_binding():
    from int8_linear import _lib
    y, w = torch.ones(4, 8, device="cuda"), torch.ones(2, 2, device="cuda")
    places = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    before = _lib.fast().launches()
    with forward_ad.dual_level():
        moe.moe_combine(y, w, places)
    assert _lib.fast().launches() == before + 1


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
def test_the_custom_ops_refuse_it(wide):
    """Also where the op copies its input before it calls (rows of a wider matrix)."""
    ops = torch.ops.int8_linear
    x = torch.ones(4, 128, device="cuda").bfloat16()
    r, w = torch.ones(4, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda").bfloat16()
    with forward_ad.dual_level():
        d, = _dual([x], 0)
        d = d[:, :64] if wide else d[:, :64].contiguous()
        assert forward_ad.unpack_dual(d).tangent is not None
        with pytest.raises(NotSupported, match="gradient"):
            ops.add_rmsnorm_mxfp4_quant(d, r, w, 1e-6, False)
        with pytest.raises(NotSupported, match="gradient"):
            ops.moe_combine(d, torch.ones(2, 2, device="cuda"),
                            torch.zeros(2, 2, dtype=torch.int32, device="cuda"), None)
