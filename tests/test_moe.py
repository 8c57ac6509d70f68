"""The operators over experts without a GPU: the restatement, the refusals, the custom ops' shapes."""

from __future__ import annotations

import ctypes

import pytest
import torch

import moe_restated as ref
from int8_linear import NotSupported, _lib, moe

P = ctypes.c_void_p(0x1000)   # never read: every call below is refused before a launch
OK, BAD, INV = _lib.OK, _lib.UNSUPPORTED, _lib.INVALID_ARG


def test_restated_order_agrees_with_counting():
    g = torch.Generator().manual_seed(0)
    experts = torch.randint(-2, 9, (50, 4), generator=g, dtype=torch.int32)
    offsets, tokens, places = ref.order(experts, 7)
    flat = experts.flatten()
    here = (flat >= 0) & (flat < 7)
    assert torch.equal(offsets[1:] - offsets[:-1], torch.bincount(flat[here], minlength=7).int())
    assert offsets[-1] == here.sum() and (tokens[offsets[-1]:] == -1).all()
    assert torch.equal((places.flatten() >= 0), here)
    for i in here.nonzero().flatten().tolist():
        at = places.flatten()[i].item()
        assert tokens[at] == i // 4 and offsets[flat[i]] <= at < offsets[flat[i] + 1]


def test_restated_weights_are_torchs():
    x = torch.randn(20, 12, generator=torch.Generator().manual_seed(1))
    e = ref.picks(x, 5)
    assert torch.equal(e.long(), x.topk(5).indices)
    soft = torch.softmax(x.double(), 1).gather(1, e.long())
    assert torch.allclose(ref.weights(x, e, "softmax", False), soft)
    assert torch.allclose(ref.weights(x, e, "softmax", True), soft / soft.sum(1, keepdim=True))
    assert torch.allclose(ref.weights(x, e, "sigmoid", False), torch.sigmoid(x.double()).gather(1, e.long()))


def _status(status: int) -> int:
    assert _lib.last_error()
    return status


def test_route_entry_refuses():
    L = _lib.lib()

    def call(logits=P, ldl=8, dt=_lib.BF16, T=4, E=8, k=2, scoring=0, out=P, ws=None, nbytes=0):
        return _status(L.i8l_moe_route(logits, ldl, dt, T, E, k, scoring, 1, out, out, out, out, out,
                                       ws, nbytes, None))
    assert call(T=-1) == INV and call(E=0) == INV and call(k=0) == INV and call(k=9) == INV
    assert call(ldl=7) == INV and call(logits=None) == INV and call(out=None) == INV
    assert call(dt=_lib.I32) == BAD and call(scoring=2) == BAD and call(scoring=-1) == BAD
    assert call(E=513, ldl=513) == BAD and call(E=100, ldl=100, k=65) == BAD
    assert call(T=2 ** 25, k=2) == BAD
    need = L.i8l_moe_route_workspace_bytes(2000, 8, 2)
    assert need > 0 and L.i8l_moe_route_workspace_bytes(1, 8, 2) == 0
    assert call(T=2000) == INV and call(T=2000, ws=P, nbytes=need - 1) == INV
    assert call(T=2000, ws=ctypes.c_void_p(0x1002), nbytes=need) == INV


def test_order_entry_refuses():
    L = _lib.lib()

    def call(experts=P, T=4, E=8, k=2, out=P):
        return _status(L.i8l_moe_order(experts, T, E, k, out, out, out, None, 0, None))
    assert call(T=-1) == INV and call(E=0) == INV and call(k=0) == INV
    assert call(experts=None) == INV and call(out=None) == INV
    assert call(E=513) == BAD and call(k=65) == BAD and call(T=2 ** 24 + 1) == BAD
    assert call(T=2000) == INV                                        # no workspace
    for sizes in ((-1, 8, 2), (2000, 0, 2), (2000, 8, 0), (2000, 513, 2), (2000, 8, 65)):
        assert L.i8l_moe_order_workspace_bytes(*sizes) == 0 == L.i8l_moe_route_workspace_bytes(*sizes)


def test_grouped_entry_refuses():
    L = _lib.lib()

    def call(a=P, lda=64, M=4, rows=P, b=P, eb=512, ldb=64, sa=P, sa_len=4, sb=P, bias=None, bias_dt=0,
             offsets=P, out=P, ldc=8, dt=_lib.BF16, silu=0, R=8, E=2, N=8, K=64):
        return _status(L.i8l_w8a8_grouped_mm(a, lda, M, rows, b, eb, ldb, sa, sa_len, sb, bias, bias_dt,
                                             offsets, out, ldc, dt, silu, R, E, N, K, None))
    assert call(M=-1) == INV and call(R=-1) == INV and call(E=0) == INV and call(N=-1) == INV
    assert call(K=0) == INV and call(rows=None) == INV                # 8 ordered rows, 4 to read
    assert call(silu=1, N=7) == INV and call(sa_len=3) == INV and call(ldc=7) == INV
    assert call(silu=1, ldc=3) == INV and call(lda=-64) == INV and call(eb=-1) == INV
    assert call(M=0, sa_len=1) == INV
    for name in ("a", "b", "sa", "sb", "offsets", "out"):
        assert call(**{name: None}) == INV
    assert call(dt=_lib.I32) == BAD and call(bias=P, bias_dt=_lib.I32) == BAD
    assert call(E=513) == BAD and call(R=2 ** 25 + 1) == BAD and call(K=2 ** 17) == BAD
    assert call(N=2 ** 24 + 1, ldc=2 ** 24 + 1) == BAD


def test_combine_entry_refuses():
    L = _lib.lib()

    def call(y=P, ldy=16, R=8, w=P, places=P, base=None, ldb=16, out=P, T=4, k=2, N=16, dt=_lib.BF16):
        return _status(L.i8l_moe_combine(y, ldy, R, w, places, base, ldb, out, T, k, N, dt, None))
    assert call(T=-1) == INV and call(k=0) == INV and call(N=-1) == INV and call(R=-1) == INV
    assert call(ldy=15) == INV and call(base=P, ldb=15) == INV
    for name in ("y", "w", "places", "out"):
        assert call(**{name: None}) == INV
    assert call(dt=_lib.I32) == BAD and call(T=2 ** 24) == BAD and call(k=1025) == BAD
    assert call(N=2 ** 24, ldy=2 ** 24) == BAD and call(R=2 ** 31) == BAD


def _mm_args(t=4, e=2, k=64, n=8):
    return dict(a_q=torch.zeros(t, k, dtype=torch.int8), b_q=torch.zeros(e, n, k, dtype=torch.int8).transpose(1, 2),
                scale_a=torch.ones(t, 1), scale_b=torch.ones(e, n), offsets=torch.zeros(e + 1, dtype=torch.int32))


def test_python_layer_refuses_host_tensors():
    with pytest.raises(NotSupported):
        moe.moe_route(torch.zeros(2, 4), 2)
    with pytest.raises(NotSupported):
        moe.moe_order(torch.zeros(2, 4, dtype=torch.int32), 4)
    with pytest.raises(NotSupported):
        moe.w8a8_grouped_mm(**_mm_args())
    with pytest.raises(NotSupported):
        moe.moe_combine(torch.zeros(2, 4), torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.int32))


def test_types_are_refused():
    with pytest.raises(NotSupported, match="logits"):
        moe.moe_route(torch.zeros(2, 4, dtype=torch.float64), 2)
    with pytest.raises(NotSupported, match="int32"):
        moe.moe_order(torch.zeros(2, 4, dtype=torch.int64), 4)
    for name, dt in (("a_q", torch.uint8), ("b_q", torch.uint8), ("scale_a", torch.float64),
                     ("scale_b", torch.bfloat16), ("offsets", torch.int64)):
        args = _mm_args()
        args[name] = args[name].to(dt)
        with pytest.raises(NotSupported, match="only|int32"):
            moe.w8a8_grouped_mm(**args)
    with pytest.raises(NotSupported, match="output"):
        moe.w8a8_grouped_mm(**_mm_args(), out_dtype=torch.int32)


@pytest.mark.parametrize("which", ["scale_a", "scale_b", "bias"])
def test_a_lost_gradient_is_refused(which):
    args = _mm_args() | {"bias": torch.zeros(2, 8)}
    args[which].requires_grad_()
    for call in (moe.w8a8_grouped_mm, moe.w8a8_grouped_mm_silu_mul):
        with pytest.raises(NotSupported, match="no gradient"):
            call(**args)
        with torch.no_grad(), pytest.raises(NotSupported, match="HIP device"):
            call(**args)


def test_a_lost_gradient_of_the_router_and_the_sum_is_refused():
    with pytest.raises(NotSupported, match="no gradient"):
        moe.moe_route(torch.zeros(2, 4, requires_grad=True), 2)
    places = torch.zeros(1, 2, dtype=torch.int32)
    for i in range(3):
        ts = [torch.zeros(2, 4), torch.zeros(1, 2), torch.zeros(1, 4)]
        ts[i].requires_grad_()
        with pytest.raises(NotSupported, match="no gradient"):
            moe.moe_combine(ts[0], ts[1], places, base=ts[2])


def test_custom_ops_have_shapes_without_running():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        ops = torch.ops.int8_linear
        w, e, offsets, tokens, places = ops.moe_route(torch.empty(5, 16, dtype=torch.bfloat16), 3, "softmax", True)
        assert (w.shape, e.shape, offsets.shape, tokens.shape, places.shape) == ((5, 3), (5, 3), (17,), (15,), (5, 3))
        assert w.dtype == torch.float32 and {x.dtype for x in (e, offsets, tokens, places)} == {torch.int32}
        assert [x.shape for x in ops.moe_order(e, 7)] == [(8,), (15,), (5, 3)]
        a, b = torch.empty(5, 64, dtype=torch.int8), torch.empty(16, 64, 32, dtype=torch.int8)
        args = (a, b, torch.empty(5, 1), torch.empty(16, 32), offsets, torch.float16, None)
        assert ops.w8a8_grouped_mm(*args, tokens).shape == (15, 32)
        y = ops.w8a8_grouped_mm_silu_mul(*args, tokens)
        assert y.shape == (15, 16) and y.dtype == torch.float16
        assert ops.moe_combine(y, w, places, None).shape == (5, 16)
