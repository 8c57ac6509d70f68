"""MXFP4 quantizers and product on the GPU against their definitions in float64.

Codes and scales are compared bit for bit.  Products are compared exactly where every partial sum is
exact in fp32 (the operands are built so: multiples of a power of two u with the magnitudes of the
terms summing below 2^23 u, checked), else within half a step of the output's type plus
K/32 * 2^-23 of the sum of the magnitudes of the terms: a block's 32 products sum exactly, and each
of the K/32 additions of a block is off by at most a step of fp32.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import mx_restated as mx
from helpers import bits, np_, say
from int8_linear import NotSupported, _lib, mxfp4

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _x(shape, seed, dtype, spread=4.0):
    """Values whose blocks lie at many powers of two."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    return (x * torch.exp2(torch.randn((shape[0], shape[1] // 32), generator=g) * spread
                           ).repeat_interleave(32, 1)).to(dtype)


def _same(q, s, x: torch.Tensor, rounded=False):
    q0, s0 = mx.quant(x.double().numpy(), rounded)
    assert np.array_equal(np_(s), s0)
    assert np.array_equal(np_(q), q0)


# ------------------------------------------------------------------ quantizer
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (3, 96), (5, 2080), (64, 512), (65, 544),
                                 (700, 1056), (1025, 2048), (300, 14336)])
def test_quant_bits(m, k, dtype):
    say(f"mxfp4_quant {m}x{k} {dtype}")
    x = _x((m, k), m * 7 + k, DT[dtype])
    for rounded in (False, True):
        _same(*mxfp4.mxfp4_quant(x.cuda(), rounded), x, rounded)


@pytest.mark.parametrize("dtype", DT)
def test_quant_special_blocks(dtype):
    t = DT[dtype]
    x = _x((40, 64), 3, t)
    top = torch.finfo(t).max
    tiny = torch.finfo(t).smallest_normal
    x[0] = 0
    x[1, :32] = -0.0
    x[2, 5], x[3, 40], x[4, 3] = float("nan"), float("inf"), float("-inf")
    x[5, 0], x[5, 1], x[5, 40] = float("nan"), float("inf"), top
    x[6], x[7] = top, -top
    x[8], x[9, 3] = tiny, tiny
    x[10] = tiny * torch.finfo(t).eps                       # the smallest subnormal
    x[11] = torch.linspace(0, 1, 64).to(t) * tiny           # subnormals
    x[12] = torch.linspace(-8, 8, 64).to(t)
    for i, peak in enumerate((4.0, 5.0, 6.0, 6.9, 7.0, 7.1, 7.9, 3.5, 1.75)):
        x[13 + i] = (torch.linspace(0, 1, 64) * peak).to(t)
        x[13 + i, 0] = peak
    if dtype != "fp16":
        x[25:30] = (_x((5, 64), 4, torch.float32).double() * 2.0 ** -124).to(t)
        x[30:35] = (_x((5, 64), 5, torch.float32).double() * 2.0 ** 118).to(t)
    for rounded in (False, True):
        q, s = mxfp4.mxfp4_quant(x.cuda(), rounded)
        _same(q, s, x, rounded)
        v = mxfp4.mxfp4_dequant(q, s, torch.float32)
        assert np.array_equal(np_(v), mx.values(np_(q), np_(s)).astype(np.float32), equal_nan=True)


def test_quant_every_bf16_value():
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x.view(-1, 32)
    q, s = mxfp4.mxfp4_quant(x.cuda())
    _same(q, s, x)
    # each magnitude as its block's only value, so that it is the peak
    alone = torch.zeros(1 << 15, 32, dtype=torch.bfloat16)
    alone[:, 7] = x.reshape(-1)[:1 << 15]
    q, s = mxfp4.mxfp4_quant(alone.cuda(), True)
    _same(q, s, alone, True)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("first,ld", [(0, 192), (8, 136), (1, 131), (64, 256)])
def test_quant_reads_slices_in_place(first, ld, dtype):
    wide = _x((37, 320), 11, DT[dtype]).reshape(-1)[:37 * ld].view(37, ld)
    dev = wide.cuda()
    x = dev[:, first:first + 64]
    _same(*mxfp4.mxfp4_quant(x), wide[:, first:first + 64])
    _same(*mxfp4.mxfp4_quant(dev[:1, first:first + 64]), wide[:1, first:first + 64])


def test_quant_of_shared_rows_and_no_rows():
    x = _x((1, 64), 2, torch.bfloat16)
    _same(*mxfp4.mxfp4_quant(x.cuda().expand(5, 64)), x.expand(5, 64))
    q, s = mxfp4.mxfp4_quant(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 32) and s.shape == (0, 2)
    assert mxfp4.mxfp4_dequant(q, s).shape == (0, 64)


@pytest.mark.parametrize("m,k", [(3, 544), (300, 2080)])
def test_quantizers_leave_what_lies_behind(m, k):
    """One byte past the codes and scales, and the pad before them, stay as they were."""
    x, L = _x((m, 2 * k), 5, torch.bfloat16).cuda(), _lib.lib()
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    for kind in ("quant", "norm", "silu"):
        q = torch.full((m * k // 2 + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        s = torch.full((m * k // 32 + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        qp, sp = ctypes.c_void_p(q.data_ptr() + 32), ctypes.c_void_p(s.data_ptr() + 32)
        stream = _lib.stream_of(x)
        if kind == "quant":
            st = L.i8l_mxfp4_quant(x.data_ptr(), 2 * k, qp, sp, m, k, _lib.BF16, 0, stream)
        elif kind == "norm":
            st = L.i8l_add_rmsnorm_mxfp4_quant(x.data_ptr(), None, w.data_ptr(), 1e-6, qp, sp, None,
                                               m, k, _lib.BF16, _lib.BF16, 0, stream)
        else:
            st = L.i8l_silu_mul_mxfp4_quant(x.data_ptr(), qp, sp, m, k, _lib.BF16, 0, stream)
        assert st == _lib.OK
        for t in (q, s):
            assert (t[:32] == 0xA5).all() and (t[-32:] == 0xA5).all()


# ------------------------------------------------------------------ dequantizer
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (7, 96, 0), (33, 544, 16), (33, 544, 3), (2049, 2048, 0)])
def test_dequant(m, k, pad, dtype):
    g = torch.Generator().manual_seed(m + k)
    q = torch.randint(0, 256, (m, k // 2 + pad), dtype=torch.uint8, generator=g)[:, :k // 2]
    s = torch.randint(100, 140, (m, k // 32 + pad), dtype=torch.uint8, generator=g)[:, :k // 32]
    s[0, 0] = 255
    out = mxfp4.mxfp4_dequant(q.cuda(), s.cuda(), DT[dtype])
    qd, sd = torch.empty(m, k // 2 + pad, dtype=torch.uint8, device="cuda"), \
        torch.empty(m, k // 32 + pad, dtype=torch.uint8, device="cuda")
    qd[:, :k // 2], sd[:, :k // 32] = q.cuda(), s.cuda()
    strided = mxfp4.mxfp4_dequant(qd[:, :k // 2], sd[:, :k // 32], DT[dtype])
    want = torch.from_numpy(mx.values(q.numpy(), s.numpy())).to(DT[dtype])
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    assert torch.equal(torch.nan_to_num(out, nan=77.0), torch.nan_to_num(strided, nan=77.0))


def test_dequant_every_code_and_scale():
    q = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat(256, 1)
    s = torch.arange(256, dtype=torch.uint8).repeat_interleave(16)[:, None]
    # 2^127 times 2 and more is past the largest fp32 and bf16: infinite, as the casts have it
    want = torch.from_numpy(mx.values(q.numpy(), s.numpy()))
    for dt in (torch.bfloat16, torch.float32):
        out = mxfp4.mxfp4_dequant(q.cuda(), s.cuda(), dt).cpu()
        assert np.array_equal(out.double().numpy(), want.to(dt).double().numpy(), equal_nan=True)


# ------------------------------------------------------------------ fused quantizers
def _norm_rows(x, res, w, eps):
    """add_rmsnorm's values: the sum of squares in float64, every rounding where the norm has it."""
    v = x.float() if res is None else x.float() + res.float()
    var = v.double().square().mean(1, keepdim=True).float()
    rs = (1 / (var + torch.tensor(eps, dtype=torch.float32)).double().sqrt()).float()
    return ((v * rs).to(w.dtype).float() * w.float()).to(x.dtype), v.to(x.dtype)


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp16"),
                                          ("fp16", "bf16")])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 2048), (3, 96), (8, 2080), (257, 4096), (1030, 512),
                                 (600, 5120), (2, 32768)])
def test_add_rmsnorm_quant(m, k, dtype, wdtype):
    say(f"add_rmsnorm_mxfp4_quant {m}x{k} {dtype} {wdtype}")
    x = _x((m, k), m + k, DT[dtype], 0.5)
    res = _x((m, k), m + k + 1, DT[dtype], 0.5)
    w = (1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(1))).to(DT[wdtype])
    for r in (None, res):
        y, rout = _norm_rows(x, r, w, 1e-6)
        q, s, ro = mxfp4.add_rmsnorm_mxfp4_quant(x.cuda(), r.cuda() if r is not None else None,
                                                 w.cuda(), 1e-6, r is None)
        _same(q, s, y, r is None)
        assert ro is None if r is None else np.array_equal(bits(ro), bits(rout))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,i", [(1, 32), (1, 6144), (3, 96), (24, 6144), (130, 2080), (700, 8960),
                                 (9, 14336)])
def test_silu_mul_quant(m, i, dtype):
    say(f"silu_mul_mxfp4_quant {m}x{i} {dtype}")
    gu = _x((m, 2 * i), m + i, DT[dtype], 0.5)
    g, u = gu[:, :i], gu[:, i:]
    # the one fp16 gate whose SiLU lies within a step of fp32 of a rounding's border
    g[g == -2.724609375] = -2.72265625
    a = (g.double() / (1 + (-g.double()).exp())).to(DT[dtype])
    y = (a.float() * u.float()).to(DT[dtype])
    for rounded in (False, True):
        _same(*mxfp4.silu_mul_mxfp4_quant(gu.cuda(), rounded), y, rounded)


def test_silu_of_far_gates():
    gu = torch.ones(2, 128)
    gu[0, :64] = torch.linspace(-80, 80, 64)
    gu[1, :64] = torch.tensor([float("inf"), -200.0, -100.0, float("nan")] * 16)
    gu[1, 0:64:2] = 3.0
    gu = gu.bfloat16()
    g = gu[:, :64].double()
    y = ((g / (1 + (-g).exp())).bfloat16().float() * gu[:, 64:].float()).bfloat16()
    _same(*mxfp4.silu_mul_mxfp4_quant(gu.cuda()), y)


@pytest.mark.parametrize("kind", ["norm", "silu"])
def test_fused_quantizers_take_odd_pointers(kind):
    flat = _x((1, 40 * 192 + 32), 9, torch.bfloat16, 0.5).reshape(-1)
    x = flat[1:1 + 40 * 192].view(40, 192)
    dev = flat.cuda()[1:1 + 40 * 192].view(40, 192)
    if kind == "norm":
        w = torch.ones(192, dtype=torch.bfloat16)
        q, s, _ = mxfp4.add_rmsnorm_mxfp4_quant(dev, None, w.cuda(), 1e-6)
        _same(q, s, _norm_rows(x, None, w, 1e-6)[0])
    else:
        g = x[:, :96].double()
        y = ((g / (1 + (-g).exp())).bfloat16().float() * x[:, 96:].float()).bfloat16()
        _same(*mxfp4.silu_mul_mxfp4_quant(dev), y)


# ------------------------------------------------------------------ product
def _operand(r, k, seed, scales=(126, 129), ld=0, lds=0, offset=0):
    """Codes and scales on the GPU (row strides ld and lds, offset bytes into their buffers)."""
    g = torch.Generator().manual_seed(seed)
    ld, lds = max(ld, k // 2), max(lds, k // 32)
    q = torch.randint(0, 256, (r * ld + offset,), dtype=torch.uint8, generator=g)
    s = torch.randint(*scales, (r * lds + offset,), dtype=torch.uint8, generator=g)
    cut = lambda t, w, n: t[offset:].view(r, w)[:, :n]   # noqa: E731
    qd, sd = q.cuda(), s.cuda()
    return (cut(q, ld, k // 2).numpy(), cut(s, lds, k // 32).numpy(), cut(qd, ld, k // 2),
            cut(sd, lds, k // 32))


def _check_exact(m, n, k, dtype=torch.float32, bias=False, **kw):
    say(f"mxfp4_mm {m}x{n}x{k} {dtype} {kw}")
    a, sa, ad, sad = _operand(m, k, m + 3 * k, **kw)
    w, sw, wd, swd = _operand(n, k, n + 5 * k, **kw)
    b = torch.randint(-64, 64, (n,), generator=torch.Generator().manual_seed(n)).float()
    want, terms = mx.mm(a, sa, w, sw, b.numpy() if bias else None)
    unit = 2.0 ** (int(sa.min()) + int(sw.min()) - 254 - 2)
    assert terms.max() + 64 < unit * 2 ** 23
    out = mxfp4.mxfp4_mm(ad, wd.t(), sad, swd, dtype, b.cuda() if bias else None)
    assert out.dtype == dtype and out.shape == (m, n)
    assert torch.equal(out.cpu(), torch.from_numpy(want).float().to(dtype))


MS = [1, 2, 7, 16, 17, 33, 64, 65, 100, 128, 129, 257, 300]


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(64, 32), (1, 64), (5, 96), (130, 160), (257, 512), (96, 1056),
                                 (512, 1024), (320, 2048), (192, 4096), (96, 384), (4112, 128),
                                 (64, 12544)])
def test_mm_exact(m, n, k):
    _check_exact(m, n, k)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (5, 2048, 6144), (24, 12288, 2048), (75, 4096, 7168),
                                   (513, 1024, 2048), (777, 1536, 4096), (1000, 520, 1536),
                                   (2049, 256, 1024), (100, 1024, 14336), (300, 512, 8192),
                                   (129, 2048, 6144), (640, 392, 6144), (40, 28672, 1024),
                                   (90, 12288, 1536)])
def test_mm_exact_served_sizes(m, n, k):
    _check_exact(m, n, k)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 96, 512), (40, 100, 1024), (200, 256, 1024), (300, 320, 1536)])
def test_mm_output_and_bias_types(m, n, k, dtype):
    for bias in (False, True):
        _check_exact(m, n, k, DT[dtype], bias)


@pytest.mark.parametrize("m,n,k", [(3, 64, 512), (40, 130, 1024), (200, 256, 1024)])
@pytest.mark.parametrize("kw", [{"ld": 1024, "lds": 64}, {"ld": 1040, "lds": 41},
                                {"ld": 1037, "lds": 33}, {"offset": 16}, {"offset": 1}])
def test_mm_strides_and_alignment(m, n, k, kw):
    _check_exact(m, n, k, **kw)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 256, 14336), (33, 512, 4096), (75, 128, 14336),
                                   (300, 1024, 2048), (700, 512, 8192)])
def test_mm_real_values(m, n, k, dtype):
    """Quantized normal values (scales differ from block to block), with a bias of the output's type."""
    say(f"mxfp4_mm values {m}x{n}x{k} {dtype}")
    g = torch.Generator().manual_seed(m + n + k)
    x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * 0.02
    b = (torch.randn(n, generator=g) * 0.1).to(DT[dtype])
    a, sa = mxfp4.mxfp4_quant(x.cuda())
    wq, sw = mxfp4.mxfp4_quant(w.cuda())
    out = mxfp4.mxfp4_mm(a, wq.t(), sa, sw, DT[dtype], b.cuda()).cpu().double().numpy()
    want, terms = mx.mm(np_(a), np_(sa), np_(wq), np_(sw), b.double().numpy())
    off = k / 32 * 2.0 ** -23 * terms + 2.0 ** -23 * np.abs(b.double().numpy())
    step = torch.finfo(DT[dtype]).eps / 2
    assert (np.abs(out - want) <= off + step * (np.abs(want) + off)).all()


@pytest.mark.parametrize("m,n,k", [(2, 32, 64), (20, 64, 512), (130, 128, 1024)])
def test_mm_scales_of_both_ends(m, n, k):
    a, sa, ad, sad = _operand(m, k, 1)
    w, sw, wd, swd = _operand(n, k, 2)
    for ea, eb in ((254, 1), (0, 254), (127, 3), (200, 60)):   # uniform scales: the sums stay exact
        sad.fill_(ea)
        swd.fill_(eb)
        want, terms = mx.mm(a, np.full_like(sa, ea), w, np.full_like(sw, eb))
        assert terms.max() < 2.0 ** (ea + eb - 256 + 23)
        out = mxfp4.mxfp4_mm(ad, wd.t(), sad, swd, torch.float32).cpu().double().numpy()
        assert np.array_equal(out, want), (ea, eb)


@pytest.mark.parametrize("m,n,k", [(2, 32, 64), (20, 64, 512), (130, 128, 1024), (3, 5, 96)])
def test_mm_nan_scales_reach_their_rows_and_columns_only(m, n, k):
    a, sa, ad, sad = _operand(m, k, 1)
    w, sw, wd, swd = _operand(n, k, 2)
    sad[m - 1, k // 32 - 1] = 255
    swd[1, 0] = 255
    out = mxfp4.mxfp4_mm(ad, wd.t(), sad, swd, torch.float32).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[m - 1], bad[:, 1] = True, True
    assert torch.equal(torch.isnan(out), bad)
    want = torch.from_numpy(mx.mm(a, sa, w, sw)[0]).float()
    assert torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("m,n,k", [(100, 1024, 14336), (200, 136, 6144)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_mm_with_and_without_a_workspace(m, n, k, dt):
    """The split of K, with its workspace NULL, too small, misaligned or given; nothing is written
    past what it needs."""
    a, sa, ad, sad = _operand(m, k, 1)
    w, sw, wd, swd = _operand(n, k, 2)
    bias = torch.arange(n).to(DT[dt]).cuda()
    # (the bias as its type holds it: bf16 has no 257)
    want, terms = mx.mm(a, sa, w, sw, bias.double().cpu().numpy())
    assert terms.max() + n < 2.0 ** (int(sa.min()) + int(sw.min()) - 256 + 23)
    L = _lib.lib()
    need = L.i8l_mxfp4_mm_workspace_bytes(m, n, k)
    assert need >= 2 * m * n * 4 and need % (m * n * 4) == 0
    ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    for ptr, size in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 4, need + 32),
                      (ws.data_ptr(), need)):
        out = torch.full((m + 1, n), 7.0, dtype=DT[dt], device="cuda")
        st = L.i8l_mxfp4_mm_ws(ad.data_ptr(), k // 2, wd.data_ptr(), k // 2, sad.data_ptr(), k // 32,
                               swd.data_ptr(), k // 32, bias.data_ptr(), _lib.DTYPE_CODE[DT[dt]],
                               out.data_ptr(), n, _lib.DTYPE_CODE[DT[dt]], m, n, k, ptr, size,
                               _lib.stream_of(ad))
        assert st == _lib.OK
        used = ptr == ws.data_ptr() and size == need
        assert bool((ws[:need] == 0xA5).all()) != used and (ws[need:] == 0xA5).all()
        assert torch.equal(out[:m].cpu(), torch.from_numpy(want).float().to(DT[dt]))
        assert (out[m] == 7).all()


def test_mm_of_nothing_and_shared_rows():
    _, _, wd, swd = _operand(64, 512, 2)
    _, _, ad, sad = _operand(1, 512, 1)
    none = mxfp4.mxfp4_mm(ad[:0], wd.t(), sad[:0], swd)
    assert none.shape == (0, 64)
    assert mxfp4.mxfp4_mm(ad, wd[:0].t(), sad, swd[:0]).shape == (1, 0)
    five = mxfp4.mxfp4_mm(ad.expand(5, -1), wd.t(), sad.expand(5, -1), swd)
    assert torch.equal(five, mxfp4.mxfp4_mm(ad, wd.t(), sad, swd).expand(5, -1))


@pytest.mark.parametrize("m,n,k", [(3, 100, 512), (40, 130, 1056), (200, 256, 1024), (130, 130, 2048)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_mm_leaves_what_lies_behind(m, n, k, dt):
    """Columns between the output's rows and rows past the last stay as they were."""
    a, sa, ad, sad = _operand(m, k, 1)
    w, sw, wd, swd = _operand(n, k, 2)
    ldc = n + 24
    out = torch.full((m + 3, ldc), 7.0, dtype=DT[dt], device="cuda")
    st = _lib.lib().i8l_mxfp4_mm(ad.data_ptr(), k // 2, wd.data_ptr(), k // 2, sad.data_ptr(), k // 32,
                                 swd.data_ptr(), k // 32, None, 0, out.data_ptr(), ldc,
                                 _lib.DTYPE_CODE[DT[dt]], m, n, k, _lib.stream_of(ad))
    assert st == _lib.OK
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()
    want = torch.from_numpy(mx.mm(a, sa, w, sw)[0]).float().to(DT[dt])
    assert torch.equal(out[:m, :n].cpu(), want)


def test_mm_takes_the_4_and_8_bit_dtypes():
    if not hasattr(torch, "float4_e2m1fn_x2") or not hasattr(torch, "float8_e8m0fnu"):
        pytest.skip("this torch has no such dtypes")
    _, _, ad, sad = _operand(4, 512, 1)
    _, _, wd, swd = _operand(64, 512, 2)
    want = mxfp4.mxfp4_mm(ad, wd.t(), sad, swd)
    e8, e2 = torch.float8_e8m0fnu, torch.float4_e2m1fn_x2
    out = mxfp4.mxfp4_mm(ad.view(e2), wd.view(e2).t(), sad.view(e8), swd.view(e8))
    assert torch.equal(out, want)


# ------------------------------------------------------------------ streams, graphs, refusals
@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_calls_in_a_graph_replay_as_eager_ones(m):
    """quantizer, product, norm and SiLU captured together; inputs change between the replays."""
    k, n = 512, 1024
    w = mxfp4.mxfp4_quant(_x((n, k), 1, torch.bfloat16, 0.5).cuda())
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    x = _x((m, k), 2, torch.bfloat16, 0.5).cuda()

    def step(x):
        q, s, r = mxfp4.add_rmsnorm_mxfp4_quant(x, x, gamma, 1e-6)
        gu = mxfp4.mxfp4_mm(q, w[0].t(), s, w[1])
        q, s = mxfp4.silu_mul_mxfp4_quant(gu)
        return r, mxfp4.mxfp4_mm(*(t for t in (q, w[0].t(), s, w[1])), torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, out = step(x)
    for i in range(4):
        x.copy_(_x((m, k), 10 + i, torch.bfloat16, 0.5))
        want = step(x.clone())
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r, want[0]) and torch.equal(out, want[1])


def test_a_split_of_k_in_a_graph():
    """Two graphs of one split product each, replayed on two streams at once: each has its own sums."""
    w = mxfp4.mxfp4_quant(_x((512, 8192), 1, torch.bfloat16, 0.5).cuda())
    assert _lib.lib().i8l_mxfp4_mm_workspace_bytes(200, 512, 8192) > 0
    cases = []
    for i in range(2):
        x = mxfp4.mxfp4_quant(_x((200, 8192), 5 + i, torch.bfloat16, 0.5).cuda())
        call = lambda x=x: mxfp4.mxfp4_mm(x[0], w[0].t(), x[1], w[1], torch.float32)   # noqa: E731
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        cases.append((graph, out, want, torch.cuda.Stream()))
    for _ in range(5):
        for graph, out, _, stream in cases:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, _, _, stream in cases:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _ in cases)


def test_calls_on_another_stream():
    x = _x((64, 512), 2, torch.bfloat16, 0.5).cuda()
    w = mxfp4.mxfp4_quant(_x((256, 512), 1, torch.bfloat16, 0.5).cuda())
    want = mxfp4.mxfp4_mm(*(lambda q, s: (q, w[0].t(), s, w[1]))(*mxfp4.mxfp4_quant(x)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        big = big @ big   # keeps the stream busy: the calls below must queue behind it
        x2 = x + 0 * big[0, 0].to(torch.bfloat16).nan_to_num()
        q, s = mxfp4.mxfp4_quant(x2)
        out = mxfp4.mxfp4_mm(q, w[0].t(), s, w[1])
    side.synchronize()
    assert torch.equal(out, want)


def test_results_do_not_change_from_call_to_call():
    for m in (1, 40, 300):
        x = mxfp4.mxfp4_quant(_x((m, 2048), m, torch.bfloat16).cuda())
        w = mxfp4.mxfp4_quant(_x((512, 2048), 1, torch.bfloat16).cuda())
        first = mxfp4.mxfp4_mm(x[0], w[0].t(), x[1], w[1], torch.float32)
        for _ in range(5):
            assert torch.equal(mxfp4.mxfp4_mm(x[0], w[0].t(), x[1], w[1], torch.float32), first)


def test_custom_ops_are_the_calls():
    ops = torch.ops.int8_linear
    x = _x((5, 128), 1, torch.bfloat16, 0.5).cuda()
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    for got, want in ((ops.mxfp4_quant(x, True), mxfp4.mxfp4_quant(x, True)),
                      (ops.add_rmsnorm_mxfp4_quant(x, x, w, 1e-6, False),
                       mxfp4.add_rmsnorm_mxfp4_quant(x, x, w, 1e-6)),
                      (ops.silu_mul_mxfp4_quant(x, False), mxfp4.silu_mul_mxfp4_quant(x))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, s = mxfp4.mxfp4_quant(x)
    assert torch.equal(ops.mxfp4_mm(q, q.t(), s, s, torch.float32, None),
                       mxfp4.mxfp4_mm(q, q.t(), s, s, torch.float32))


def test_binding_and_ctypes_paths_agree(monkeypatch):
    f = _lib.fast()
    if f is None:
        pytest.skip("the C++ binding is not built")
    x = _x((5, 256), 1, torch.bfloat16, 0.5).cuda()
    gamma = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    q, s = mxfp4.mxfp4_quant(x)
    bias = torch.randn(5, device="cuda")

    def every():
        return (*mxfp4.mxfp4_quant(x, True), mxfp4.mxfp4_dequant(q, s, torch.float16),
                *mxfp4.add_rmsnorm_mxfp4_quant(x, x, gamma, 1e-6), *mxfp4.silu_mul_mxfp4_quant(x),
                mxfp4.mxfp4_mm(q, q.t(), s, s, torch.float16, bias))
    before = f.launches()
    fast = every()
    assert f.launches() == before + 5
    monkeypatch.setattr(mxfp4, "_fast", lambda *a: None)
    assert all(torch.equal(a, b) for a, b in zip(fast, every()))
    assert f.launches() == before + 5


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    q, s = mxfp4.mxfp4_quant(x)
    w, sw = mxfp4.mxfp4_quant(torch.zeros(8, 64, device="cuda"))
    ok = (q, w.t(), s, sw)

    def mm(i, v, **kw):
        args = list(ok)
        if i is not None:
            args[i] = v
        return lambda: mxfp4.mxfp4_mm(*args, **kw)
    for err, call in [
            (ValueError, lambda: mxfp4.mxfp4_quant(x[:, :48])),
            (ValueError, lambda: mxfp4.mxfp4_quant(x[0])),
            (ValueError, lambda: mxfp4.mxfp4_quant(x[:, :0])),
            (NotSupported, lambda: mxfp4.mxfp4_quant(x.double())),
            (NotSupported, lambda: mxfp4.mxfp4_quant(torch.zeros(64, 64, device="cuda").t())),
            (ValueError, lambda: mxfp4.mxfp4_dequant(q, s[:2])),
            (ValueError, lambda: mxfp4.mxfp4_dequant(q[:, :24], s)),
            (NotSupported, lambda: mxfp4.mxfp4_dequant(q, s.int())),
            (NotSupported, lambda: mxfp4.mxfp4_dequant(q, s, torch.int8)),
            (ValueError, lambda: mxfp4.mxfp4_dequant(q, s.cpu())),
            (ValueError, lambda: mxfp4.add_rmsnorm_mxfp4_quant(x, None, x[0, :32], 1e-6)),
            (ValueError, lambda: mxfp4.add_rmsnorm_mxfp4_quant(x, x[:2], x[0], 1e-6)),
            (NotSupported, lambda: mxfp4.add_rmsnorm_mxfp4_quant(x, x.half(), x[0], 1e-6)),
            (NotSupported, lambda: mxfp4.add_rmsnorm_mxfp4_quant(x.float(), None, x[0], 1e-6)),
            (NotSupported, lambda: mxfp4.silu_mul_mxfp4_quant(x[:, ::2])),
            (ValueError, lambda: mxfp4.silu_mul_mxfp4_quant(x[:, :48].contiguous())),
            (ValueError, mm(1, w)), (ValueError, mm(2, s[:3])), (ValueError, mm(3, s)),
            (NotSupported, mm(0, q.to(torch.int8))), (NotSupported, mm(2, s.float())),
            (ValueError, mm(3, sw.cpu())), (NotSupported, mm(1, w.t().cpu())),
            (NotSupported, mm(None, None, out_dtype=torch.int32)),
            (ValueError, mm(None, None, bias=torch.zeros(7, device="cuda"))),
            (NotSupported, mm(None, None, bias=torch.zeros(8, dtype=torch.int32, device="cuda")))]:
        with pytest.raises(err):
            call()
    assert torch.equal(mm(None, None)(), torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"))
