"""fp16 through the shared conversions: the int8 products' fp16 outputs against the oracle over enough
values that a product and its cast rounded as one would show (one value in 2^13 lies where the two
roundings of the definition meet a border), and the time of the fp16 quantizers beside the bf16 ones."""

from __future__ import annotations

import statistics

import numpy as np
import pytest
import torch

from helpers import bits, ints, np_, randn, say
from int8_linear import fused_quant as fq
from int8_linear import w8a8_mm
from oracle import oracle as o
from test_gemm_gpu import oracle_out

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(16, 12288, 256), (64, 4096, 512), (300, 2048, 256), (1024, 1024, 512),
                                   (129, 4100, 320), (2048, 520, 256)])
@pytest.mark.parametrize("bias", [None, torch.float16, torch.float32])
def test_fp16_outputs_are_rounded_twice(m, n, k, bias):
    say(f"w8a8_mm fp16 m={m} n={n} k={k} bias={bias}")
    g = torch.Generator().manual_seed(m + n)
    a, w = ints((m, k), 1), ints((n, k), 2)
    sa = (torch.rand((m, 1), generator=g) * 1e-2 + 1e-3).cuda()
    sb = (torch.rand((n, 1), generator=g) * 1e-2 + 1e-3).cuda()
    b = torch.randn(n, generator=g).to(bias).cuda() if bias else None
    out = w8a8_mm(a, w.t(), sa, sb, torch.float16, b)
    assert np.array_equal(bits(out), oracle_out(a, w, sa, sb, b, torch.float16))


def _us(call) -> float:
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(20):
            call()
    times = []
    for _ in range(9):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        graph.replay()
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / 20)
    return statistics.median(times)


@pytest.mark.parametrize("round_silu,most", [(False, 1.2), (True, 1.4)])
def test_silu_mul_quant_takes_about_as_long_as_in_bf16(round_silu, most):
    """3001 x 14336 as many bytes as in bf16: 41.7 / 39.7 us unrounded and 40.8 / 33.8 rounded (fp16 /
    bf16), where a conversion for each value and both ways to the quotient kept apart take 53 and 54."""
    say(f"silu_mul_quant fp16 and bf16 times, round_silu={round_silu}")
    us = {}
    for dtype in (torch.bfloat16, torch.float16):
        gu = randn((3001, 2 * 14336), 1, dtype=dtype)
        us[dtype] = _us(lambda: fq.silu_mul_quant(gu, True, round_silu))
    assert us[torch.float16] < most * us[torch.bfloat16], us


@pytest.mark.parametrize("m,i", [(5, 6144), (300, 2080)])
@pytest.mark.parametrize("round_silu", [False, True])
def test_silu_mul_quant_of_subnormal_products(m, i, round_silu):
    """SiLU times up below fp16's smallest normal value, 2^-14, down to its last bit."""
    gu = randn((m, 2 * i), m, 2.0 ** -9, dtype=torch.float16)
    q, s = fq.silu_mul_quant(gu, True, round_silu)
    want = o.silu_mul_quant(bits(gu), o.F16, round_silu, True)
    assert np.array_equal(np_(q), want[0]) and np.array_equal(np_(s), want[1])
    assert np_(s).max() * 127 < 2.0 ** -14


@pytest.mark.parametrize("m,k", [(3, 2048), (5, 2080), (600, 4096), (40, 1000)])
def test_add_rmsnorm_quant_of_subnormal_products(m, k):
    x, w = randn((m, k), m, dtype=torch.float16), randn((k,), 3, 2.0 ** -17, dtype=torch.float16)
    q, s, _ = fq.add_rmsnorm_quant(x, None, w, 1e-6)
    want = o.add_rmsnorm_quant(bits(x), None, bits(w), 1e-6, o.F16, o.F16)
    assert np.array_equal(np_(q), want[0]) and np.array_equal(np_(s), want[1])
    assert np_(s).max() * 127 < 2.0 ** -12
