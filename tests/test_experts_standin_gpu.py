"""The decoder stand-in with experts: a layer's calls in a row against their definitions, a split over
two ranks, and the whole step eager and as a graph."""

from __future__ import annotations

import pytest
import torch

import moe_restated as ref
from helpers import say
from int8_linear import fused_quant as fq
from int8_linear import moe, standin

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 13, 150])
def test_a_layer_call_by_call(m):
    """Each operator against its definition, on the inputs that the step gives it."""
    say(f"experts layer, {m} tokens")
    st = standin.ExpertsStandIn(m, layers=1)
    layer = st.layers[0]
    q, s, _ = fq.add_rmsnorm_quant(st.x, st.x, st.norm, standin.EPS)
    logits = st.mm(layer, "router", q, s, torch.float32)
    weights, offsets, tokens, places = st.route(logits)
    experts = ref.picks(logits.cpu(), st.TOP_K)
    for got, want in zip((offsets, tokens, places), ref.order(experts, st.EXPERTS)):
        assert torch.equal(got.cpu(), want)
    w, ws = layer["gate_up"]
    y = moe.w8a8_grouped_mm_silu_mul(q, w.transpose(1, 2), s, ws, offsets, rows=tokens)
    v = ref.grouped(q, w, s, ws, offsets, None, tokens)
    want = ref.silu_mul(v)
    # (test_moe_gpu.py derives it: the exponential's argument, its function and half a bf16 step)
    g, u = v.double().abs().chunk(2, 1)
    rel = 2.0 ** -20 + g * 2.0 ** -23 + 2.0 ** -8 * (1 + 2.0 ** -9)
    assert ((y.cpu().double() - want).abs() <= want.abs() * rel + g * u * 2.0 ** -126 + 1e-38).all()
    q2, s2 = fq.quant_per_token(y)
    w, ws = layer["down"]
    o = moe.w8a8_grouped_mm(q2, w.transpose(1, 2), s2, ws, offsets)
    assert torch.equal(o.cpu(), ref.grouped(q2, w, s2, ws, offsets).bfloat16())
    out = st.experts(layer, q, s, (weights, offsets, tokens, places))
    want, size = ref.combine(o, weights, places)
    # 8 products and sums in fp32, half a bf16 step
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -20 * size + 2.0 ** -8 * want.abs() + 1e-38).all()


@pytest.mark.parametrize("m", [1, 60])
def test_ranks_sum_to_the_whole(m):
    whole = standin.ExpertsStandIn(m, layers=1)
    parts = [standin.ExpertsStandIn(m, layers=1, first_expert=a, local_experts=n) for a, n in ((0, 24), (24, 40))]
    q, s, _ = fq.add_rmsnorm_quant(whole.x, whole.x, whole.norm, standin.EPS)
    logits = whole.mm(whole.layers[0], "router", q, s, torch.float32)
    want = whole.experts(whole.layers[0], q, s, whole.route(logits)).double()
    got = sum(p.experts(p.layers[0], q, s, p.route(logits)).double() for p in parts)
    # the parts and the whole are rounded to bf16: half a step each, of values that may be larger
    # than their sum
    assert (got - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_the_step_in_a_graph():
    st = standin.ExpertsStandIn(9, layers=2)
    eager = st.forward()
    seen = []
    us = standin.per_layer_us(st, windows=1, min_window_ms=1.0, check=lambda h: seen.append(torch.equal(h, eager)))
    assert seen == [True] and us > 0
    assert torch.equal(st.forward(), eager)
