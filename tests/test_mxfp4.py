"""MXFP4 without a GPU: the restatement against first principles, and the refusals."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import mx_restated as mx
from int8_linear import NotSupported, _lib, mxfp4, qk_rope

P = ctypes.c_void_p(0x1000)   # never read: every call below is refused before a launch


def test_every_code_is_its_own_nearest_and_ties_go_to_the_even_code():
    t = np.concatenate([mx.GRID, -mx.GRID])
    assert np.array_equal(mx.nearest_code(t), np.arange(16))
    mid = (mx.GRID[:-1] + mx.GRID[1:]) / 2
    assert np.array_equal(mx.nearest_code(mid), [0, 2, 2, 4, 4, 6, 6])
    assert np.array_equal(mx.nearest_code(np.nextafter(mid, 9)), [1, 2, 3, 4, 5, 6, 7])
    assert np.array_equal(mx.nearest_code(np.nextafter(mid, 0)), [0, 1, 2, 3, 4, 5, 6])
    assert mx.nearest_code(np.array([1e9]))[0] == 7


@pytest.mark.parametrize("rounded", [False, True])
def test_the_scale_puts_the_peak_at_the_top_of_the_grid(rounded):
    peak = np.exp2(np.arange(-120, 120, dtype=np.float64))[:, None] * np.linspace(1, 2, 257)[:-1]
    t = peak / np.exp2(mx.scale_codes(peak, rounded) - 127.0)
    assert t.min() >= (3.5 if rounded else 4) and t.max() < (7 if rounded else 8)


def test_round_trip_is_within_half_a_step():
    x = np.random.default_rng(0).standard_normal((64, 256))
    q, s = mx.quant(x, True)
    scale = np.repeat(np.exp2(s - 127.0), 32, 1)
    off = np.abs(mx.values(q, s) - x) / scale
    assert off.max() <= 1.0                                  # half of the largest step, 2
    assert off[np.abs(x) < 2 * scale].max() <= 0.25


def _status(status: int) -> int:
    assert _lib.last_error()
    return status


@pytest.mark.parametrize("k", [0, -32, 16, 33, 63])
def test_entry_points_refuse_broken_blocks(k):
    L = _lib.lib()
    for st in (L.i8l_mxfp4_quant(P, 64, P, P, 4, k, _lib.BF16, 0, None),
               L.i8l_mxfp4_dequant(P, 64, P, 2, P, 4, k, _lib.BF16, None),
               L.i8l_add_rmsnorm_mxfp4_quant(P, None, P, 1e-6, P, P, None, 4, k, _lib.BF16,
                                             _lib.BF16, 0, None),
               L.i8l_silu_mul_mxfp4_quant(P, P, P, 4, k, _lib.BF16, 0, None),
               L.i8l_mxfp4_mm(P, 64, P, 64, P, 2, P, 2, None, 0, P, 8, _lib.BF16, 4, 8, k, None)):
        assert _status(st) == _lib.INVALID_ARG


def test_entry_points_refuse_types_strides_and_null():
    L = _lib.lib()
    bad, inv = _lib.UNSUPPORTED, _lib.INVALID_ARG
    assert _status(L.i8l_mxfp4_quant(P, 64, P, P, 4, 64, _lib.I32, 0, None)) == bad
    assert _status(L.i8l_mxfp4_quant(P, 32, P, P, 4, 64, _lib.BF16, 0, None)) == inv
    assert _status(L.i8l_mxfp4_quant(None, 64, P, P, 4, 64, _lib.BF16, 0, None)) == inv
    assert _status(L.i8l_mxfp4_quant(P, 64, P, P, -1, 64, _lib.BF16, 0, None)) == inv
    assert _status(L.i8l_mxfp4_dequant(P, 16, P, 2, P, 4, 64, _lib.BF16, None)) == inv
    assert _status(L.i8l_mxfp4_dequant(P, 32, P, 2, ctypes.c_void_p(0x1002), 4, 64, _lib.BF16,
                                       None)) == bad
    assert _status(L.i8l_add_rmsnorm_mxfp4_quant(P, P, P, 1e-6, P, P, None, 4, 64, _lib.BF16,
                                                 _lib.BF16, 0, None)) == inv
    assert _status(L.i8l_add_rmsnorm_mxfp4_quant(P, None, P, 1e-6, P, P, None, 4, 65536, _lib.BF16,
                                                 _lib.BF16, 0, None)) == bad
    assert _status(L.i8l_silu_mul_mxfp4_quant(P, P, P, 4, 64, _lib.F32, 0, None)) == bad

    def mm(lda=32, ldb=32, ldsa=2, ldsb=2, ldc=8, out=_lib.BF16, bias=None, bias_dt=0, a=P):
        return _status(L.i8l_mxfp4_mm(a, lda, P, ldb, P, ldsa, P, ldsb, bias, bias_dt, P, ldc, out,
                                      4, 8, 64, None))
    assert mm(lda=31) == inv and mm(ldb=16) == inv and mm(ldsa=1) == inv and mm(ldsb=1) == inv
    assert mm(ldc=7) == inv and mm(a=None) == inv
    assert mm(out=_lib.I32) == bad and mm(bias=P, bias_dt=_lib.I32) == bad


def test_qk_norm_rope_refuses():
    L = _lib.lib()

    def call(T=4, hq=2, hk=1, d=64, r=64, act=_lib.BF16, cs=_lib.F32, w=_lib.BF16, bits=64, q=P,
             pos=P):
        return _status(L.i8l_qk_norm_rope(q, 192, 64, P, 192, 64, P, 128, 64, P, 64, 64, P, P, w,
                                          1e-6, P, cs, 100, pos, bits, T, hq, hk, d, r, 0, act, None))
    inv, bad = _lib.INVALID_ARG, _lib.UNSUPPORTED
    assert call(T=-1) == inv and call(r=65) == inv and call(r=66) == inv and call(r=0) == inv
    assert call(d=0, r=0) == inv and call(bits=16) == inv and call(q=None) == inv
    assert call(pos=None) == inv
    assert call(act=_lib.F32) == bad and call(cs=_lib.I32) == bad and call(w=_lib.I32) == bad
    assert call(T=1 << 30, hq=64) == bad


def test_python_layer_refuses_host_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    h = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: mxfp4.mxfp4_quant(x), lambda: mxfp4.mxfp4_dequant(q, s),
                 lambda: mxfp4.add_rmsnorm_mxfp4_quant(x, None, x[0], 1e-6),
                 lambda: mxfp4.silu_mul_mxfp4_quant(x),
                 lambda: mxfp4.mxfp4_mm(q, q.t(), s, s),
                 lambda: qk_rope.qk_norm_rope(h, h, None, None, torch.zeros(9, 64),
                                              torch.zeros(4, dtype=torch.int64), 1e-6)):
        with pytest.raises(NotSupported):
            call()


@pytest.mark.parametrize("d,t,hk", [(64, (1 << 26) - 3, 0), (6, 1 << 24, 4)])
def test_qk_norm_rope_refuses_more_waves_than_a_grid_counts(d, t, hk):
    status = _status(_lib.lib().i8l_qk_norm_rope(P, d, d, P, d * hk, d, P, d, d, P, d * hk, d, None,
                                                 None, _lib.DTYPE_NONE, 1e-6, P, _lib.F32, 100, P, 64,
                                                 t, 1, hk, d, d, 0, _lib.BF16, None))
    assert status == _lib.UNSUPPORTED


@pytest.mark.parametrize("which", range(4))
def test_qk_norm_rope_refuses_to_lose_a_gradient(which):
    args = [torch.zeros(2, 3, 64).bfloat16(), torch.zeros(2, 1, 64).bfloat16(),
            torch.ones(64).bfloat16(), torch.ones(64).bfloat16()]
    args[which].requires_grad_()
    rest = (torch.zeros(8, 64), torch.zeros(2, dtype=torch.int64), 1e-6)
    for inplace in (False, True):
        with pytest.raises(NotSupported, match="gradient"):
            qk_rope.qk_norm_rope(*args, *rest, inplace=inplace)


def test_rope_cos_sin_is_exact_far_out():
    t = qk_rope.rope_cos_sin(40960, 64, 1e4, device="cpu")
    assert t.shape == (40960, 64) and t.dtype == torch.float32
    p, i = 40959, 3
    angle = p * 1e4 ** (-2 * i / 64)
    assert abs(t[p, i].item() - np.cos(angle)) <= 2 ** -24 and \
        abs(t[p, 32 + i].item() - np.sin(angle)) <= 2 ** -24
    with pytest.raises(ValueError):
        qk_rope.rope_cos_sin(16, 7)


def test_shared_memory_is_seen_before_writing_in_place():
    buf = torch.zeros(6, 4 * 16)
    cols = lambda a, n: buf[:, a * 16:(a + n) * 16].unflatten(1, (n, 16))   # noqa: E731
    assert qk_rope._apart(cols(0, 2), cols(2, 1)) and qk_rope._apart(cols(3, 1), cols(0, 2))
    assert not qk_rope._apart(cols(0, 2), cols(1, 1))
    assert qk_rope._apart(cols(0, 2)[:3], cols(0, 2)[3:])
    assert not qk_rope._apart(buf[0:3].unflatten(1, (4, 16)), buf[1:4].unflatten(1, (4, 16)))


def test_custom_ops_have_shapes_without_running():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.int8_linear
    with FakeTensorMode():
        x = torch.empty(5, 128, dtype=torch.bfloat16)
        q, s = ops.mxfp4_quant(x, False)
        assert q.shape == (5, 64) and s.shape == (5, 4)
        q, s, r = ops.add_rmsnorm_mxfp4_quant(x, x, x[0], 1e-6, False)
        assert r.shape == x.shape
        q, s = ops.silu_mul_mxfp4_quant(x, False)
        assert q.shape == (5, 32) and s.shape == (5, 2)
        w, ws = torch.empty(9, 32, dtype=torch.uint8), torch.empty(9, 2, dtype=torch.uint8)
        assert ops.mxfp4_mm(q, w.t(), s, ws, torch.float16, None).shape == (5, 9)
        h = torch.empty(5, 3, 64, dtype=torch.bfloat16)
        a, b = ops.qk_norm_rope(h, h[:, :1], None, None, torch.empty(8, 64),
                                torch.empty(5, dtype=torch.int64), 1e-6, False)
        assert a.shape == h.shape and b.shape == (5, 1, 64)
