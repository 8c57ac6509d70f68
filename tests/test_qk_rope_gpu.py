"""The q/k norm with its rotation on the GPU against its definition in float64.

Tolerance: half a step of the output's type, and 2^-19 (|h_a| + |h_b|) of the pair for fp32: the sum
of squares of up to 64 lanes' up to 16 values each and its mean, root and reciprocal (fewer than 24
roundings, halved by the root), the two products of the norm, the products and the sum of the
rotation come to less than 32 steps of 2^-24.
"""

from __future__ import annotations

import pytest
import torch

import mx_restated as mx
from helpers import say
from int8_linear import NotSupported, _lib, qk_rope

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _rand(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _case(t, hq, hk, d, rot, dtype=torch.bfloat16, wdtype=None, csdtype=torch.float32, span=5000,
          pos_dtype=torch.int64, pad=0):
    """A qkv output (pad values more a row), the views of q and k, and the rest, on the CPU."""
    qkv = _rand((t, (hq + 2 * hk) * d + pad), t + d, dtype, 2.0)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    wdtype = wdtype or dtype
    return dict(qkv=qkv, q=q, k=k, qw=1 + _rand((d,), 1, scale=0.2).to(wdtype),
                kw=1 + _rand((d,), 2, scale=0.2).to(wdtype),
                cs=qk_rope.rope_cos_sin(span, rot, 1e6, device="cpu", dtype=csdtype),
                pos=torch.randint(0, span, (t,), generator=torch.Generator().manual_seed(t)).to(pos_dtype))


def _views(c, dev):
    hq, hk, d = c["q"].shape[1], c["k"].shape[1], c["q"].shape[2]
    return dev[:, :hq * d].unflatten(1, (hq, d)), dev[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))


def _check(got, x, w, c, interleaved):
    want = mx.qk(x, w, c["cs"], c["pos"], EPS, interleaved)
    h = x.double()
    h = (h / (h.square().mean(-1, keepdim=True) + EPS).sqrt()).abs()
    if w is not None:
        h = h * w.double().abs()
    rot = c["cs"].shape[1]
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    pair = h[..., a] + h[..., b]
    h[..., a], h[..., b] = pair, pair
    off = 2.0 ** -19 * h
    tol = off + torch.finfo(x.dtype).eps / 2 * (want.abs() + off) + 2.0 ** -24   # (fp16 subnormals)
    g = got.cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert ((g - want).abs() <= tol)[~torch.isnan(want)].all()


def _run(c, interleaved=False, weights=True, inplace=False):
    dev = c["qkv"].cuda()
    q, k = _views(c, dev)
    qw, kw = (c["qw"], c["kw"]) if weights else (None, None)
    qo, ko = qk_rope.qk_norm_rope(q, k, qw.cuda() if weights else None, kw.cuda() if weights else None,
                                  c["cs"].cuda(), c["pos"].cuda(), EPS, interleaved=interleaved,
                                  inplace=inplace)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == q.dtype
    _check(qo, c["q"], qw, c, interleaved)
    _check(ko, c["k"], kw, c, interleaved)
    return dev, q, k, qo, ko


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (128, 64), (96, 96), (96, 24),
                                   (80, 80), (80, 40), (80, 20), (512, 512), (192, 64), (32, 32),
                                   (1024, 1024), (2, 2), (6, 4), (17, 16), (100, 50), (2048, 128)])
def test_head_sizes(d, rot, interleaved):
    say(f"qk_norm_rope heads of {d}, {rot} rotated, interleaved={interleaved}")
    _run(_case(9, 5, 2, d, rot), interleaved)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("t,hq,hk", [(1, 16, 8), (1, 1, 1), (3, 32, 8), (7, 5, 1), (130, 28, 4),
                                     (1031, 16, 8), (4099, 4, 4), (5, 64, 8)])
def test_tokens_and_heads(t, hq, hk, dtype):
    say(f"qk_norm_rope {t} tokens {hq}+{hk} {dtype}")
    _run(_case(t, hq, hk, 128, 128, DT[dtype]))


@pytest.mark.parametrize("wdtype", DT)
@pytest.mark.parametrize("csdtype", DT)
def test_table_and_weight_types(csdtype, wdtype):
    for d, rot in ((128, 128), (80, 20)):
        _run(_case(5, 4, 2, d, rot, torch.bfloat16, DT[wdtype], DT[csdtype], pos_dtype=torch.int32))


@pytest.mark.parametrize("pad", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("d,rot", [(128, 128), (80, 40)])
def test_row_strides(d, rot, pad):
    _run(_case(6, 3, 2, d, rot, pad=pad))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,pad", [(128, 128, 0), (128, 64, 4), (80, 20, 1)])
def test_in_place_writes_the_heads_and_nothing_else(d, rot, pad, interleaved):
    c = _case(70, 6, 2, d, rot, pad=pad)
    dev, q, k, qo, ko = _run(c, interleaved, inplace=True)
    assert qo.data_ptr() == q.data_ptr() and ko.data_ptr() == k.data_ptr()
    out = _run(c, interleaved)
    assert torch.equal(q, out[3]) and torch.equal(k, out[4])
    rest = (c["q"].shape[1] + c["k"].shape[1]) * d
    assert torch.equal(dev[:, rest:].cpu(), c["qkv"][:, rest:])


def test_no_weights():
    for d, rot in ((128, 128), (80, 20)):
        _run(_case(5, 4, 2, d, rot), weights=False)


def test_far_positions():
    c = _case(64, 4, 1, 128, 128, span=40960)
    c["pos"] = torch.arange(40960 - 64, 40960)
    _run(c)


def test_positions_outside_the_table_are_nan():
    for d, rot in ((128, 64), (80, 20)):
        c = _case(8, 3, 1, d, rot, span=100)
        c["pos"][1], c["pos"][4], c["pos"][6] = -1, 100, 1 << 40
        _, _, _, qo, _ = _run(c)
        assert torch.isnan(qo[4, :, :rot]).all() and torch.isfinite(qo[4, :, rot:]).all()


def test_zero_and_non_finite_heads():
    c = _case(4, 3, 1, 128, 128)
    c["qkv"][0] = 0
    c["qkv"][1, 5] = float("nan")
    c["qkv"][2, 128 + 3] = float("inf")
    dev = c["qkv"].cuda()
    q, k = _views(c, dev)
    qo, _ = qk_rope.qk_norm_rope(q, k, c["qw"].cuda(), c["kw"].cuda(), c["cs"].cuda(), c["pos"].cuda(), EPS)
    assert (qo[0] == 0).all()
    assert torch.isnan(qo[1, 0]).all() and torch.isfinite(qo[1, 1:]).all()
    assert torch.isfinite(qo[2, 0]).all() and torch.isnan(qo[2, 1]).any()
    assert torch.isfinite(qo[3]).all()


def test_no_tokens_and_no_key_heads():
    c = _case(3, 2, 1, 64, 64)
    cs, qw = c["cs"].cuda(), c["qw"].cuda()
    q, k = _views(c, c["qkv"].cuda())
    pos = c["pos"].cuda()
    qo, ko = qk_rope.qk_norm_rope(q[:0], k[:0], qw, qw, cs, pos[:0], EPS)
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 1, 64)
    qo, ko = qk_rope.qk_norm_rope(q, k[:, :0], qw, qw, cs, pos, EPS)
    _check(qo, c["q"], c["qw"], c, False)
    assert ko.shape == (3, 0, 64)


def test_in_a_graph():
    c = _case(33, 16, 8, 128, 128)
    dev, cs, pos = c["qkv"].cuda(), c["cs"].cuda(), c["pos"].cuda()
    q, k = _views(c, dev)
    qw, kw = c["qw"].cuda(), c["kw"].cuda()
    qk_rope.qk_norm_rope(q, k, qw, kw, cs, pos, EPS)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = qk_rope.qk_norm_rope(q, k, qw, kw, cs, pos, EPS)
    for i in range(4):
        dev.copy_(_rand(dev.shape, 40 + i, torch.bfloat16))
        pos.copy_((pos + 7) % 5000)
        want = qk_rope.qk_norm_rope(q, k, qw, kw, cs, pos, EPS)
        qo.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_binding_and_ctypes_paths_agree(monkeypatch):
    f = _lib.fast()
    if f is None:
        pytest.skip("the C++ binding is not built")
    c = _case(5, 16, 8, 128, 128)
    before = f.launches()
    a = _run(c)
    assert f.launches() == before + 1
    monkeypatch.setattr(qk_rope, "_fast", lambda *x: None)
    b = _run(c)
    assert torch.equal(a[3], b[3]) and torch.equal(a[4], b[4]) and f.launches() == before + 1
    op = torch.ops.int8_linear.qk_norm_rope(a[1], a[2], c["qw"].cuda(), c["kw"].cuda(), c["cs"].cuda(),
                                            c["pos"].cuda(), EPS, False)
    assert torch.equal(op[0], a[3])


def test_refusals():
    c = _case(4, 2, 1, 64, 64)
    q, k = _views(c, c["qkv"].cuda())
    w, cs, pos = c["qw"].cuda(), c["cs"].cuda(), c["pos"].cuda()

    def call(q=q, k=k, qw=w, kw=w, cs=cs, pos=pos, **kw2):
        return lambda: qk_rope.qk_norm_rope(q, k, qw, kw, cs, pos, EPS, **kw2)
    wide = torch.zeros(4, 8, 64, dtype=torch.bfloat16, device="cuda")
    for err, f in [
            (ValueError, call(q=q[0])), (ValueError, call(q=q[:3])), (ValueError, call(k=k[..., :32])),
            (NotSupported, call(q=q.float(), k=k.float())), (NotSupported, call(k=k.half())),
            (NotSupported, call(q=wide.transpose(1, 2))),
            (ValueError, call(qw=w[:32])), (NotSupported, call(qw=w.float())),
            (NotSupported, call(qw=w.double(), kw=w.double())),
            (ValueError, call(cs=cs[:, :63])), (ValueError, call(cs=cs[:, :0])),
            (ValueError, call(cs=torch.zeros(9, 66, device="cuda"))),
            (NotSupported, call(cs=cs.double())), (NotSupported, call(cs=cs[:, ::2])),
            (ValueError, call(pos=pos[:3])), (NotSupported, call(pos=pos.short())),
            (ValueError, call(pos=pos.cpu())), (ValueError, call(cs=cs.cpu())),
            (ValueError, call(q=wide[:, :2], k=wide[:, 1:3], inplace=True)),
            (ValueError, call(q=wide[:1].expand(4, 8, 64), k=k, inplace=True))]:
        with pytest.raises(err):
            f()


@pytest.mark.parametrize("which", ["q", "q_weight"])
def test_a_lost_gradient_is_refused_by_the_binding_too(which):
    c = _case(4, 2, 1, 64, 64)
    q, k = _views(c, c["qkv"].cuda())
    w, rest = c["qw"].cuda(), (c["cs"].cuda(), c["pos"].cuda(), EPS)
    want = qk_rope.qk_norm_rope(q, k, w, w, *rest)
    if which == "q":
        q = q.detach().requires_grad_()
    else:
        w = w.clone().requires_grad_()
    with pytest.raises(NotSupported, match="gradient"):
        qk_rope.qk_norm_rope(q, k, w, w, *rest)
    with torch.no_grad():
        got = qk_rope.qk_norm_rope(q, k, w, w, *rest)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
