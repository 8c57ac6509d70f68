"""The MXFP4 decoder stand-in: a layer's calls in a row, each against its definition in float64 on the
inputs it had, and the whole step eager and as a graph.

Tolerances: as for the operators one by one (test_mxfp4_gpu.py, test_qk_rope_gpu.py).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_restated as mx
from helpers import np_, say
from int8_linear import mxfp4, standin

pytestmark = pytest.mark.gpu


def _norm(x, res, w):
    v = x.float() if res is None else x.float() + res.float()
    var = v.double().square().mean(1, keepdim=True).float()
    rs = (1 / (var + torch.tensor(standin.EPS, dtype=torch.float32)).double().sqrt()).float()
    return ((v * rs).to(w.dtype).float() * w.float()).to(x.dtype), v.to(x.dtype)


def _check_codes(q, s, y):
    q0, s0 = mx.quant(y.double().numpy())
    assert np.array_equal(np_(s), s0) and np.array_equal(np_(q), q0)


def _check_mm(out, q, s, w, ws):
    want, terms = mx.mm(np_(q), np_(s), np_(w), np_(ws))
    off = 2 * q.shape[1] / 32 * 2.0 ** -23 * terms
    assert (np.abs(out.cpu().double().numpy() - want) <= off + 2.0 ** -8 * (np.abs(want) + off)).all()


@pytest.mark.parametrize("m", [1, 7, 100])
def test_a_layer_call_by_call(m):
    say(f"MXFP4 layer, {m} tokens")
    st = standin.Mxfp4StandIn(m, layers=1)
    layer, ones = st.layers[0], torch.ones(standin.HIDDEN, dtype=torch.bfloat16)
    q, s, rout = mxfp4.add_rmsnorm_mxfp4_quant(st.x, None, st.norm, standin.EPS)
    assert rout is None
    _check_codes(q, s, _norm(st.x.cpu(), None, ones)[0])
    qkv = st.mm(layer, "qkv_proj", q, s)
    _check_mm(qkv, q, s, *layer["qkv_proj"])
    qh, kh = st.heads(qkv)
    cs, pos = st.cos_sin.cpu(), st.positions.cpu()
    first = 0
    for heads, n in ((qh, standin.Q_HEADS), (kh, standin.KV_HEADS)):
        x = qkv[:, first:first + n * 128].unflatten(1, (n, 128)).cpu()
        first += n * 128
        want = mx.qk(x, None, cs, pos, standin.EPS, False)
        h = x.double().abs() / (x.double().square().mean(-1, keepdim=True) + standin.EPS).sqrt()
        pair = h[..., :64] + h[..., 64:]
        off = 2.0 ** -19 * torch.cat([pair, pair], -1)
        assert ((heads.cpu().double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()
    q, s = mxfp4.mxfp4_quant(qh.flatten(1))
    _check_codes(q, s, qh.flatten(1).cpu())
    o = st.mm(layer, "o_proj", q, s)
    _check_mm(o, q, s, *layer["o_proj"])
    q, s, res = mxfp4.add_rmsnorm_mxfp4_quant(o, st.x, st.norm, standin.EPS)
    y, rout = _norm(o.cpu(), st.x.cpu(), ones)
    _check_codes(q, s, y)
    assert torch.equal(res.cpu(), rout)
    gu = st.mm(layer, "gate_up_proj", q, s)
    _check_mm(gu, q, s, *layer["gate_up_proj"])
    q, s = mxfp4.silu_mul_mxfp4_quant(gu)
    g, u = gu.cpu().chunk(2, 1)
    _check_codes(q, s, ((g.double() / (1 + (-g.double()).exp())).bfloat16().float() * u.float()).bfloat16())
    out = st.mm(layer, "down_proj", q, s)
    _check_mm(out, q, s, *layer["down_proj"])
    h, keys = st.forward(with_keys=True)
    assert torch.equal(h, out) and torch.equal(keys[0], kh)


@pytest.mark.parametrize("m", [1, 33, 200])
def test_the_step_as_a_graph(m):
    st = standin.Mxfp4StandIn(m, layers=3)
    assert st.weight_bytes() == 3 * sum(k * n * 17 // 32 for k, n in standin.SHAPES.values())
    st.forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = st.forward()
    for i in range(3):
        st.x.copy_(torch.randn((m, standin.HIDDEN), generator=torch.Generator().manual_seed(i)))
        want = st.forward()
        h.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(h, want)


def test_per_layer_time_takes_the_stand_in():
    assert 0 < standin.per_layer_us(standin.Mxfp4StandIn(1, layers=2), windows=1, min_window_ms=1.0) < 1e4
