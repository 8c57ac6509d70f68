"""A floating output that depends on an input which requires a gradient is refused where gradients are
recorded, as there is no backward; codes, which are integers, have none to lose."""

from __future__ import annotations

import pytest
import torch

from int8_linear import NotSupported, mxfp4, qk_rope


def _norm_args():
    return [torch.ones(4, 64).bfloat16(), torch.ones(4, 64).bfloat16(), torch.ones(64).bfloat16()]


def _mm_args():
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.full((4, 2), 127, dtype=torch.uint8)
    return q, q.t(), s, s


@pytest.mark.parametrize("which", [0, 1])
def test_the_residual_stream(which):
    args = _norm_args()
    args[which].requires_grad_()
    with pytest.raises(NotSupported, match="gradient"):
        mxfp4.add_rmsnorm_mxfp4_quant(*args, 1e-6)


def test_the_bias_of_a_product():
    bias = torch.zeros(4, requires_grad=True)
    with pytest.raises(NotSupported, match="gradient"):
        mxfp4.mxfp4_mm(*_mm_args(), torch.float32, bias)


def test_the_table_of_a_rotation():
    h, cs = torch.zeros(2, 3, 64).bfloat16(), torch.zeros(8, 64, requires_grad=True)
    with pytest.raises(NotSupported, match="gradient"):
        qk_rope.qk_norm_rope(h, h[:, :1], None, None, cs, torch.zeros(2, dtype=torch.int64), 1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["residual", "x", "bias", "table"])
def test_the_binding_refuses_them_too(call):
    args = [t.cuda() for t in _norm_args()]
    mm = [t.cuda() for t in _mm_args()]
    bias = torch.ones(4, device="cuda")
    h, cs = torch.ones(2, 3, 64).bfloat16().cuda(), torch.ones(8, 64, device="cuda")
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    leaf = {"residual": args[1], "x": args[0], "bias": bias, "table": cs}[call]

    def run():
        if call in ("residual", "x"):
            return mxfp4.add_rmsnorm_mxfp4_quant(*args, 1e-6)
        if call == "bias":
            return (mxfp4.mxfp4_mm(*mm, torch.float32, bias),)
        return qk_rope.qk_norm_rope(h, h[:, :1], None, None, cs, pos, 1e-6)
    want = run()
    leaf.requires_grad_()
    with pytest.raises(NotSupported, match="gradient"):
        run()
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(run(), want))


@pytest.mark.gpu
def test_codes_are_made_of_trained_weights():
    """A weight of a model that could be trained is quantized as it is: its codes are integers."""
    w = torch.nn.Parameter(torch.randn(64, 128, device="cuda"))
    q, s = mxfp4.mxfp4_quant(w)
    assert not q.requires_grad and not s.requires_grad
    want = mxfp4.mxfp4_quant(w.detach())
    assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    gamma = torch.nn.Parameter(torch.ones(128, device="cuda").bfloat16())
    x = torch.randn(5, 128, device="cuda").bfloat16()
    got = mxfp4.add_rmsnorm_mxfp4_quant(x, x, gamma, 1e-6)
    want = mxfp4.add_rmsnorm_mxfp4_quant(x, x, gamma.detach(), 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["residual", "bias", "heads"])
def test_the_custom_ops_have_no_silent_backward(call):
    """torch records them and raises when the backward comes to them."""
    ops = torch.ops.int8_linear
    args = [t.cuda() for t in _norm_args()]
    if call == "residual":
        out = ops.add_rmsnorm_mxfp4_quant(args[0], args[1].requires_grad_(), args[2], 1e-6, False)[2]
    elif call == "bias":
        bias = torch.ones(4, device="cuda", requires_grad=True)
        out = ops.mxfp4_mm(*(t.cuda() for t in _mm_args()), torch.float32, bias)
    else:
        h = torch.ones(2, 3, 64, device="cuda").bfloat16().requires_grad_()
        out = ops.qk_norm_rope(h, h[:, :1], None, None, torch.ones(8, 64, device="cuda"),
                               torch.zeros(2, dtype=torch.int64, device="cuda"), 1e-6, False)[0]
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="autograd"):
        out.float().sum().backward()
