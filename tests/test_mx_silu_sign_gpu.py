"""silu_mul_mxfp4_quant and the sign of a zero: E2M1 has a negative zero (code 8), and a gate of -0 has
one in its SiLU.  Codes are compared bit for bit with the definition in float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_restated as mx
from helpers import np_, say
from int8_linear import mxfp4

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _check(gu: torch.Tensor, dev: torch.Tensor):
    g, u = gu.double().chunk(2, 1)
    a = (g / (1 + (-g).exp())).to(gu.dtype)
    y = (a.float() * u.float()).to(gu.dtype)
    q0, s0 = mx.quant(y.double().numpy())
    q, s = mxfp4.silu_mul_mxfp4_quant(dev)
    assert np.array_equal(np_(s), s0) and np.array_equal(np_(q), q0)
    return q0


def _gates(m, i, seed, dtype):
    """Gates in steps of 1/8 (none within an fp32 rounding of a border of its SiLU's), a third of them
    zeros of both signs; ups of both signs, zeros among them."""
    g = torch.Generator().manual_seed(seed)
    gate = torch.round(torch.randn(m, i, generator=g) * 16) / 8
    zero = torch.rand(m, i, generator=g)
    gate[zero < 0.2] = -0.0
    gate[zero > 0.9] = 0.0
    up = torch.randn(m, i, generator=g)
    up[torch.rand(m, i, generator=g) < 0.1] = -0.0
    return torch.cat([gate, up], 1).to(dtype)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,i", [(1, 32), (3, 96), (24, 6144), (2100, 2048), (1700, 2080)])
def test_gates_of_minus_zero(m, i, dtype, far):
    """far: some gates lie below -87, whose waves take their values another way."""
    say(f"silu_mul_mxfp4_quant {m}x{i} {dtype} far={far}")
    gu = _gates(m, i, m + i, DT[dtype])
    if far:
        gu[::2, 5] = -100.0
    q0 = _check(gu, gu.cuda())
    assert ((q0 & 15) == 8).any() and ((q0 >> 4) == 8).any()


@pytest.mark.parametrize("dtype", DT)
def test_gates_of_minus_zero_from_an_odd_pointer(dtype):
    gu = _gates(40, 96, 7, DT[dtype])
    dev = torch.empty(gu.numel() + 1, dtype=gu.dtype, device="cuda")[1:].view(gu.shape)
    _check(gu, dev.copy_(gu))


def test_a_code_does_not_depend_on_the_other_gates_of_its_row():
    gu = torch.ones(2, 1024, dtype=torch.bfloat16)
    gu[:, :32] = -0.0
    gu[1, 500] = -100.0
    q, s = mxfp4.silu_mul_mxfp4_quant(gu.cuda())
    assert torch.equal(q[0, :16], q[1, :16]) and (q[0, :16] == 0x88).all()


def test_a_gate_next_to_a_rounding_is_rounded_as_the_served_models_round_it():
    """fp16 -2.724609375: its SiLU in fp32, as torch computes it, rounds to -0.16760254 where the exact
    one rounds to -0.16772461.  The ups make the two fall on different sides of an E2M1 border."""
    gu = torch.zeros(1, 64, dtype=torch.float16)
    gu[0, :32], gu[0, 32:] = -2.724609375, 1.0
    gu[0, 32:48] = 0.93212890625
    y = torch.nn.functional.silu(gu[:, :32]) * gu[:, 32:]
    exact = gu[:, :32].double() * torch.sigmoid(gu[:, :32].double())
    q0, s0 = mx.quant(y.double().numpy())
    assert not np.array_equal(q0, mx.quant((exact.half() * gu[:, 32:]).double().numpy())[0])
    q, s = mxfp4.silu_mul_mxfp4_quant(gu.cuda())
    assert np.array_equal(np_(q), q0) and np.array_equal(np_(s), s0)
