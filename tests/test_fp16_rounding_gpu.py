"""fp16 roundings of the quantizers: to fp32 first, then to fp16, as their definitions say.

A compiler may make one instruction of a product and its cast to fp16, which rounds once; over the
rows below that changes codes and residuals in places.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import bits, np_, randn, say
from int8_linear import fused_quant as fq
from oracle import oracle as o

pytestmark = pytest.mark.gpu

CODE = {torch.bfloat16: o.BF16, torch.float16: o.F16}


@pytest.mark.parametrize("m,k", [(257, 4096), (64, 1000), (2100, 2048)])
@pytest.mark.parametrize("act,wdt", [(torch.bfloat16, torch.float16), (torch.float16, torch.float16),
                                     (torch.float16, torch.bfloat16)])
def test_add_rmsnorm_quant(m, k, act, wdt):
    say(f"add_rmsnorm_quant {m}x{k} {act} {wdt}")
    x, r = randn((m, k), m, dtype=act), randn((m, k), m + 1, 300.0, dtype=act)
    w = (randn((k,), 3, 0.1, dtype=torch.float32) + 1).to(wdt)
    for res in (None, r):
        q, s, ro = fq.add_rmsnorm_quant(x, res, w, 1e-6)
        want = o.add_rmsnorm_quant(bits(x), bits(res) if res is not None else None, bits(w), 1e-6,
                                   CODE[act], CODE[wdt])
        assert np.array_equal(np_(q), want[0]) and np.array_equal(np_(s), want[1])
        assert res is None or np.array_equal(bits(ro), want[2])


@pytest.mark.parametrize("round_silu", [False, True])
def test_silu_mul_quant(round_silu):
    say(f"silu_mul_quant fp16 round={round_silu}")
    gu = randn((300, 2 * 4096), 5, 2.0, dtype=torch.float16)
    q, s = fq.silu_mul_quant(gu, True, round_silu)
    want = o.silu_mul_quant(bits(gu), o.F16, round_silu, True)
    assert np.array_equal(np_(q), want[0]) and np.array_equal(np_(s), want[1])
