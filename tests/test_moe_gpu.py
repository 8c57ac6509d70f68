"""The operators over experts on the GPU, against the restatement (tests/moe_restated.py).

Picks, orders and products are compared bit for bit: the products are exact integers and the epilogue
is the same float32 steps.  Where a tolerance stands, it is derived beside it.
"""

from __future__ import annotations

import math

import pytest
import torch

import moe_restated as ref
from helpers import ints, randn, say
from int8_linear import NotSupported, moe
from int8_linear import fused_quant as fq

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return torch.equal(a.cpu(), b.cpu())


# ------------------------------------------------------------------ the router
def check_route(x: torch.Tensor, k: int, scoring="softmax", renormalize=True):
    say(f"route {tuple(x.shape)} k={k} {x.dtype} {scoring} {renormalize}")
    r = moe.moe_route(x, k, scoring=scoring, renormalize=renormalize)
    host = x.cpu()
    experts = ref.picks(host, k)
    assert same(r.experts, experts)
    offsets, tokens, places = ref.order(experts, x.shape[1])
    assert same(r.offsets, offsets) and same(r.tokens, tokens) and same(r.places, places)
    want = ref.weights(host, experts, scoring, renormalize)
    got = r.weights.cpu().double()
    # The difference x - max of logits within 32 of each other is off by 32 * 2^-24 at most, so is
    # its exponential's logarithm; the exponential itself, its sum of up to 512 positive terms (8
    # levels of lanes, 8 in a lane) and the quotient add 2^-22, 16 * 2^-24 and 2^-24.  The total enters
    # with the same error: 2^-18 + 2^-19 together, below 2^-17.  A weight below the range of exp (-87)
    # may be 0: 1e-37.
    assert ((got - want).abs() <= 2.0 ** -17 * want + 1e-37).all()
    return r


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 8), (2, 60, 4), (3, 64, 1), (17, 65, 8), (75, 128, 8),
                                   (128, 128, 8), (129, 128, 8), (33, 160, 6), (40, 256, 8), (9, 257, 3),
                                   (20, 512, 64), (1023, 1, 1), (1025, 1, 1), (700, 100, 5)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_route_sizes(t, e, k, dt):
    check_route(randn((t, e), t + e + k, 2.0, DT[dt]), k)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("scoring", moe.SCORING)
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_forms(dt, scoring, renormalize):
    check_route(randn((50, 96), 7, 2.0, DT[dt]), 6, scoring, renormalize)


def test_route_many_tokens():
    check_route(randn((5001, 128), 3, 1.5), 8)


def test_route_ties_go_to_the_lower_expert():
    x = torch.zeros(4, 130)
    x[1, 64:] = 1.0                      # the first of a later register
    x[2, ::2] = -0.0                     # equals +0
    x[3] = torch.arange(130) % 3 - 1.0
    check_route(x.cuda(), 7)


@pytest.mark.parametrize("scoring", moe.SCORING)
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_masks(scoring, renormalize):
    low = torch.finfo(torch.float32).min
    x = randn((12, 70), 5, 1.0, torch.float32, "cpu")
    x[0] = -math.inf                     # a token that may take none
    x[1, 3:] = -math.inf                 # fewer than it takes
    x[2] = math.nan
    x[3, ::3] = math.nan
    x[4, 5] = math.inf
    x[5, 5] = x[5, 66] = math.inf
    x[6] = low                           # masked by the lowest value: pickable, all alike
    x[7, 1:] = low
    x[8, ::2] = -math.inf
    x[9, 10] = x[9, 69] = math.nan
    x[10] = -200.0                       # sigmoids that are 0 in fp32: equal shares all the same
    x[11, 0] = 1e30
    r = check_route(x.cuda(), 5, scoring, renormalize)
    assert r.experts[0].tolist() == [-1] * 5 and r.weights[0].tolist() == [0.0] * 5
    assert not r.weights.isnan().any()


def test_route_reads_rows_at_any_distance():
    wide = randn((40, 200), 9, 2.0)
    check_route(wide[:, 60:188], 8)
    check_route(wide[:1].expand(40, 200), 3)
    check_route(randn((9, 64), 1, 2.0, torch.float32)[::2], 3)


def test_route_of_no_tokens():
    r = moe.moe_route(torch.empty(0, 16, device="cuda"), 4)
    assert r.offsets.tolist() == [0] * 17 and r.places.shape == (0, 4) and r.tokens.shape == (0,)


@pytest.mark.parametrize("t,e,k", [(1, 4, 1), (75, 60, 4), (64, 512, 16), (65, 512, 16), (3001, 33, 3), (20000, 8, 8),
                                   (2048, 512, 1)])
def test_order(t, e, k):
    say(f"order {t} {e} {k}")
    g = torch.Generator().manual_seed(t)
    x = torch.randint(-3, e + 3, (t, k), generator=g, dtype=torch.int32)   # the same expert twice, too
    x[0, 0], x[-1, -1] = -2 ** 31, 2 ** 31 - 1
    for got, want in zip(moe.moe_order(x.cuda(), e), ref.order(x, e)):
        assert same(got, want)


def test_order_of_one_expert_and_of_none():
    for fill in (3, -1):
        x = torch.full((500, 4), fill, dtype=torch.int32)
        for got, want in zip(moe.moe_order(x.cuda(), 8), ref.order(x, 8)):
            assert same(got, want)
    x = torch.arange(24, dtype=torch.int32).view(4, 6).t()                  # not contiguous
    for got, want in zip(moe.moe_order(x.cuda(), 24), ref.order(x, 24)):
        assert same(got, want)


# ------------------------------------------------------------------ the grouped product
def problem(sizes, k, n, seed=0, tokens=None, gone=0):
    """Operands of experts with these rows, `gone` rows behind them; tokens: rows read through rows=."""
    e, r = len(sizes), sum(sizes) + gone
    g = torch.Generator().manual_seed(seed)
    m = r if tokens is None else tokens
    offsets = torch.tensor([0] + list(sizes)).cumsum(0).int()
    rows = None if tokens is None else torch.randint(0, m, (r,), generator=g, dtype=torch.int32).cuda()
    return dict(a=ints((m, k), seed + 1), w=ints((e, n, k), seed + 2),
                sa=(torch.rand(m, 1, generator=g) * 0.01 + 1e-3).cuda(),
                sb=(torch.rand(e, n, generator=g) * 0.01 + 1e-3).cuda(), offsets=offsets.cuda(), rows=rows)


def check_mm(p, dt=torch.bfloat16, bias=None, silu=False, out=None):
    call = moe.w8a8_grouped_mm_silu_mul if silu else moe.w8a8_grouped_mm
    say(f"{call.__name__} a {tuple(p['a'].shape)} w {tuple(p['w'].shape)} {dt} rows {p['rows'] is not None} "
        f"bias {bias is not None} offsets {p['offsets'].tolist()[:20]}")
    end = p["offsets"][-1].item()
    r = p["a"].shape[0] if p["rows"] is None else p["rows"].numel()
    width = p["w"].shape[1] // (2 if silu else 1)
    if out is None:
        out = torch.full((r, width), 7.0, dtype=dt, device="cuda")
    before = out.clone()
    got = call(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"], dt, bias, rows=p["rows"], out=out)
    assert got is out
    assert torch.equal(out[end:], before[end:])
    v = ref.grouped(p["a"], p["w"], p["sa"], p["sb"], p["offsets"], bias, p["rows"])[:end]
    if not silu:
        assert same(out[:end], v.to(dt))
        return out
    want = ref.silu_mul(v)
    # exp(-g) is off by |g| 2^-24 (16-bit outputs: its argument is rounded) and 2^-22, the sum, the
    # quotient and the product by 2^-22 together; then half a step of the output, and of its
    # smallest numbers.  A sigmoid below 2^-126 (a gate below -87, whose exp(-g) or its reciprocal leaves
    # the range) may be 0: what is lost is |g u| 2^-126.
    g, u = v.double().abs().chunk(2, 1)
    rel = 2.0 ** -20 + (g * 2.0 ** -23 if dt != torch.float32 else 0)
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    err = (out[:end].cpu().double() - want).abs()
    assert (err <= want.abs() * (rel + torch.finfo(dt).eps / 2 * (1 + 2 ** -9)) + tiny + g * u * 2.0 ** -126).all()
    return out


SIZES = {"one": [1], "empty ends": [0, 3, 0], "eight of many": [0] * 5 + [1] * 8 + [0] * 50,
         "ragged": [5, 0, 17, 64, 1, 33, 0, 130], "skewed": [1, 0, 300, 2], "sixteens": [16, 32, 64, 128],
         "more than a wave of experts": [i % 4 for i in range(150)]}


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("k,n", [(256, 128), (768, 200), (144, 72)])
def test_mm_spreads(name, k, n):
    check_mm(problem(SIZES[name], k, n, tokens=40))
    check_mm(problem(SIZES[name], k, n, gone=9))
    check_mm(problem(SIZES[name], k, n, tokens=7, gone=3), silu=True)


@pytest.mark.parametrize("k,n", [(1, 2), (7, 10), (16, 8), (48, 24), (100, 6), (128, 64), (136, 66), (200, 130),
                                 (1000, 40), (1040, 264), (2880, 96), (20, 514)])
@pytest.mark.parametrize("silu", [False, True])
def test_mm_sizes(k, n, silu):
    check_mm(problem([3, 0, 20, 70], k, n, tokens=30), silu=silu)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bias", [None, *DT])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("sizes", [[4, 9], [200, 150]])
def test_mm_types(dt, bias, silu, sizes):
    p = problem(sizes, 256, 128, tokens=50)
    b = None if bias is None else randn((2, 128), 4, 1.0, DT[bias])
    check_mm(p, DT[dt], b, silu)


@pytest.mark.parametrize("sizes", [[300, 0, 40, 700], [128] * 8, [2000], [37] * 60])
@pytest.mark.parametrize("k,n", [(512, 512), (768, 264), (640, 1408), (1408, 256), (2048, 384)])
def test_mm_many_rows(sizes, k, n):
    check_mm(problem(sizes, k, n, tokens=500, gone=5))
    check_mm(problem(sizes, k, n), silu=True)


def test_mm_of_one_scale_and_other_shapes():
    p = problem([5, 6], 64, 32)
    p["sa"] = torch.tensor([0.02], device="cuda")
    check_mm(p)
    p["sa"] = torch.tensor(0.02, device="cuda")
    check_mm(p)
    p = problem([5, 6], 64, 32)
    p["sa"], p["sb"] = p["sa"].view(-1), p["sb"].view(2, 32, 1)
    check_mm(p)


@pytest.mark.parametrize("sizes", [[3, 9], [260, 90]])
def test_mm_extreme_codes(sizes):
    p = problem(sizes, 1024, 128)
    p["a"].fill_(-128)
    p["w"].fill_(-128)
    check_mm(p, torch.float32)
    p["w"].fill_(127)
    check_mm(p, torch.float32)


@pytest.mark.parametrize("sizes", [[4, 9], [150, 150]])
@pytest.mark.parametrize("pad", [1, 4, 8, 16])
def test_mm_strides_and_alignment(sizes, pad):
    k, n = 256, 128
    p = problem(sizes, k, n, tokens=33)
    a = torch.zeros(33, k + 2 * pad, dtype=torch.int8, device="cuda")
    a[:, pad:pad + k] = p["a"]
    w = torch.zeros(2, n + 1, k + pad, dtype=torch.int8, device="cuda")
    w[:, :n, :k] = p["w"]
    p["a"], p["w"] = a[:, pad:pad + k], w[:, :n, :k]
    check_mm(p)
    r = p["rows"].numel()
    wide = torch.full((r, n + pad), 3.0, dtype=torch.bfloat16, device="cuda")
    check_mm(p, out=wide[:, pad:])
    assert (wide[:, :pad] == 3).all()
    half = torch.full((r, n // 2 + pad), 3.0, dtype=torch.bfloat16, device="cuda")
    check_mm(p, silu=True, out=half[:, :n // 2])
    assert (half[:, n // 2:] == 3).all()


@pytest.mark.parametrize("shift", [1, 2])
@pytest.mark.parametrize("sizes", [[4, 9], [150, 150]])
def test_mm_scales_and_bias_off_their_alignment(shift, sizes):
    p = problem(sizes, 256, 128)
    flat = torch.zeros(2 * 128 + shift, device="cuda")
    flat[shift:] = p["sb"].flatten()
    p["sb"] = flat[shift:].view(2, 128)
    b = randn((2 * 128 + shift,), 4)[shift:].view(2, 128)
    check_mm(p, bias=b)
    check_mm(p, bias=b, silu=True)


def test_mm_one_weight_for_every_expert():
    p = problem([9, 100, 3], 256, 64)
    p["w"] = p["w"][:1].expand(3, -1, -1)
    check_mm(p)


def test_mm_of_nothing():
    p = problem([0, 0, 0], 64, 32, tokens=5, gone=0)
    assert check_mm(p).shape == (0, 32)
    p = problem([0, 0, 0], 256, 128, tokens=5, gone=20)     # every pair belongs elsewhere
    check_mm(p)
    check_mm(p, silu=True)


def test_mm_without_out():
    p = problem([30, 40], 256, 128, tokens=9)
    o = moe.w8a8_grouped_mm(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"], rows=p["rows"])
    assert same(o, ref.grouped(p["a"], p["w"], p["sa"], p["sb"], p["offsets"], None, p["rows"]).bfloat16())


@pytest.mark.parametrize("k,n,r", [(256, 128, 60), (512, 256, 700), (100, 24, 60)])
def test_mm_offsets_and_rows_out_of_range_are_held_in(k, n, r):
    """Offsets past the rows or descending are clamped, and a row outside a_q gives NaN."""
    e = 5
    p = problem([r // e] * e, k, n, tokens=50)
    rows = p["rows"].clone()
    rows[3], rows[r // 2], rows[-1] = -1, 50, 2 ** 31 - 1
    o = moe.w8a8_grouped_mm(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"], rows=rows)
    bad = torch.tensor([3, r // 2, r - 1])
    want = ref.grouped(p["a"], p["w"], p["sa"], p["sb"], p["offsets"], None, rows.clamp(0, 49)).bfloat16()
    want[bad] = math.nan
    assert torch.equal(o.cpu().nan_to_num(123.0), want.nan_to_num(123.0)) and o[bad.cuda()].isnan().all()
    h = moe.w8a8_grouped_mm_silu_mul(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"], rows=rows)
    assert h[bad.cuda()].isnan().all() and h.isnan().sum() == 3 * n // 2

    broken = torch.tensor([-7, r // 3, 5, r + 1000, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    held = torch.tensor([0, r // 3, r // 3, r, r, r], dtype=torch.int32)
    out = torch.full((r, n), 7.0, dtype=torch.bfloat16, device="cuda")
    moe.w8a8_grouped_mm(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], broken, rows=p["rows"], out=out)
    # expert 0: [0, r/3); 1: nothing, as 5 < r/3; 2: from 5 (its own offset) to r
    want = ref.grouped(p["a"], p["w"], p["sa"], p["sb"], held, None, p["rows"]).bfloat16()
    e2 = ref.grouped(p["a"], p["w"], p["sa"], p["sb"], torch.tensor([0, 0, 5, r, r, r]), None, p["rows"]).bfloat16()
    both = slice(5, r // 3)              # rows that two experts claim: either's
    o = out.cpu()
    assert torch.equal(o[:5], want[:5]) and torch.equal(o[r // 3:], e2[r // 3:])
    assert ((o[both] == want[both]) | (o[both] == e2[both])).all()


def test_mm_refuses():
    p = problem([5, 6], 64, 32, tokens=9)

    def call(**kw):
        args = dict(a_q=p["a"], b_q=p["w"].transpose(1, 2), scale_a=p["sa"], scale_b=p["sb"],
                    offsets=p["offsets"], rows=p["rows"]) | kw
        return moe.w8a8_grouped_mm(**args)
    call()
    for kw in (dict(a_q=p["a"][:, :48]), dict(scale_a=p["sa"][:5]), dict(scale_b=p["sb"][:, :16]),
               dict(offsets=p["offsets"][:2]), dict(rows=p["rows"].view(1, -1)), dict(bias=p["sb"][0]),
               dict(out=torch.empty(11, 16, dtype=torch.bfloat16, device="cuda")),
               dict(out=torch.empty(11, 32, device="cuda")), dict(b_q=p["w"][0].t()),
               dict(offsets=p["offsets"].cpu()), dict(scale_b=p["sb"].cpu()), dict(rows=p["rows"].cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(b_q=p["w"].transpose(1, 2).contiguous()), dict(a_q=p["a"].t().contiguous().t()),
               dict(out=torch.empty(1, 32, dtype=torch.bfloat16, device="cuda").expand(11, 32)),
               dict(out=torch.empty(32, 11, dtype=torch.bfloat16, device="cuda").t())):
        with pytest.raises(NotSupported):
            call(**kw)


def test_an_output_written_over_is_seen_by_autograd():
    p = problem([5, 6], 64, 32)
    out = torch.ones(11, 32, device="cuda")
    x = torch.ones(11, 32, device="cuda", requires_grad=True)
    y = (x * out).sum()
    moe.w8a8_grouped_mm(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"], torch.float32, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ------------------------------------------------------------------ the sum
def check_combine(y, w, places, base=None):
    say(f"combine y {tuple(y.shape)} {y.dtype} places {tuple(places.shape)} base {base is not None}")
    got = moe.moe_combine(y, w, places, base=base)
    want, size = ref.combine(y, w, places, base)
    # k products and k sums in fp32, 2 k 2^-24 of the magnitudes' sum; then half a step of the output
    k, dt = places.shape[1], y.dtype
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    err = (got.cpu().double() - want).abs()
    assert (err <= 2 * k * 2.0 ** -24 * size + want.abs() * torch.finfo(dt).eps / 2 + tiny).all()
    return got


def places_of(t, k, r, seed, gone=0.3):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, r, (t, k), generator=g, dtype=torch.int32)
    return torch.where(torch.rand(t, k, generator=g) < gone, -1, p).int().cuda()


@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 8, 2048), (5, 3, 7), (40, 8, 2048), (3, 9, 1000), (300, 4, 516),
                                   (2, 64, 72), (7, 2, 5000), (1000, 8, 64)])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("base", [False, True])
def test_combine(t, k, n, dt, base):
    r = t * k
    w = torch.rand(t, k, generator=torch.Generator().manual_seed(1)).cuda()
    check_combine(randn((r, n), 2, 1.0, DT[dt]), w, places_of(t, k, r, 3), randn((t, n), 4, 1.0, DT[dt]) if base else None)


def test_combine_leaves_out_what_has_no_place():
    y = randn((6, 64), 1)
    y[0] = math.nan                                     # a row that no place names
    w = torch.full((3, 2), math.inf, device="cuda")     # of places without a row
    places = torch.tensor([[-1, 6], [2 ** 31 - 1, -2 ** 31], [1, -5]], dtype=torch.int32).cuda()
    w[2, 0] = 0.5
    got = check_combine(y, w, places)
    assert (got[:2] == 0).all() and same(got[2], (y[1].float() * 0.5).bfloat16())
    assert (moe.moe_combine(y[:0], w, places) == 0).all()


def test_combine_strides():
    y = randn((30, 200), 1)
    w = torch.rand(10, 3, device="cuda")
    places = places_of(10, 3, 30, 5)
    base = randn((10, 300), 6)
    check_combine(y[:, 8:136], w, places, base[:, :128])
    check_combine(y[:, 3:131], w, places, base[:, 1:129])
    check_combine(y[:1].expand(30, 200), w, places)
    check_combine(y.t()[:100].t(), w.t().contiguous().t(), places.t().contiguous().t())
    assert moe.moe_combine(y, w[:0], places[:0]).shape == (0, 200)


def test_combine_refuses():
    y, w, places = randn((6, 64), 1), torch.rand(3, 2, device="cuda"), places_of(3, 2, 6, 1)
    for bad in (dict(weights=w[:2]), dict(places=places.cpu()), dict(base=y[:2])):
        with pytest.raises(ValueError):
            moe.moe_combine(**(dict(y=y, weights=w, places=places) | bad))
    for bad in (dict(weights=w.half()), dict(places=places.long()), dict(base=y[:3].float())):
        with pytest.raises(NotSupported):
            moe.moe_combine(**(dict(y=y, weights=w, places=places) | bad))


# ------------------------------------------------------------------ the layer
class Layer:
    """The MLP of a layer over experts, as a server runs it."""

    def __init__(self, e=12, k=3, hidden=256, inter=192, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.k = k
        self.w13, self.w2 = ints((e, 2 * inter, hidden), seed), ints((e, hidden, inter), seed + 1)
        self.s13 = (torch.rand(e, 2 * inter, generator=g) * 1e-3 + 1e-4).cuda()
        self.s2 = (torch.rand(e, hidden, generator=g) * 1e-3 + 1e-4).cuda()

    def __call__(self, x, logits):
        q, s = fq.quant_per_token(x)
        r = moe.moe_route(logits, self.k)
        y = moe.w8a8_grouped_mm_silu_mul(q, self.w13.transpose(1, 2), s, self.s13, r.offsets, rows=r.tokens)
        q, s = fq.quant_per_token(y)
        y = moe.w8a8_grouped_mm(q, self.w2.transpose(1, 2), s, self.s2, r.offsets)
        return moe.moe_combine(y, r.weights, r.places)

    def plain(self, x, logits):
        """The same tokens through the dense operators, an expert at a time, in float64 between."""
        experts = ref.picks(logits.cpu(), self.k)
        w = ref.weights(logits.cpu(), experts, "softmax", True)
        out = torch.zeros(x.shape, dtype=torch.float64)
        q, s = fq.quant_per_token(x)
        for j in range(self.k):
            for t in range(len(x)):
                e = experts[t, j].item()
                v = ref.grouped(q[t:t + 1], self.w13[e:e + 1], s[t:t + 1], self.s13[e:e + 1], torch.tensor([0, 1]))
                y = ref.silu_mul(v).bfloat16()
                q2, s2 = fq.quant_per_token(y.cuda())
                o = ref.grouped(q2, self.w2[e:e + 1], s2, self.s2[e:e + 1], torch.tensor([0, 1])).bfloat16()
                out[t] += w[t, j] * o[0].double()
        return out


@pytest.mark.parametrize("t", [1, 23])
def test_layer(t):
    layer = Layer()
    x, logits = randn((t, 256), 1), randn((t, 12), 2, 2.0)
    got, want = layer(x, logits).cpu().double(), layer.plain(x, logits)
    # A bf16 value of silu(g) u whose fp32 value lies next to a rounding's border may fall to the
    # other side: at most a code of the 192 of a row per such value, each worth a 127th of the row's
    # peak times the weight; a few of them in a row at most, 1% of the output's size.
    assert (got - want).abs().max() <= 0.01 * want.abs().max()


def test_layer_in_a_graph_with_other_choices():
    """Captured once and replayed with other tokens and another spread over the experts."""
    layer = Layer()
    for t in (5, 400):
        xs = [randn((t, 256), 10 + i) for i in range(4)]
        ls = [randn((t, 12), 20 + i, 2.0) for i in range(3)] + [torch.zeros(t, 12).bfloat16().cuda()]
        eager = [layer(x, l) for x, l in zip(xs, ls)]
        x, l = xs[0].clone(), ls[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, l)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, l)
        for i in (1, 3, 0, 2, 1):
            x.copy_(xs[i])
            l.copy_(ls[i])
            out.fill_(math.nan)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[i])
            layer(xs[2], ls[2])
            torch.cuda.synchronize()


def test_layer_on_another_stream():
    layer = Layer()
    x, logits = randn((50, 256), 1), randn((50, 12), 2, 2.0)
    want = layer(x, logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x, logits)
    side.synchronize()
    assert torch.equal(got, want)


def test_ranks_of_a_split_layer_sum_to_the_whole():
    """Two ranks with half of the experts each, the second adding to what the first gave."""
    layer = Layer()
    x, logits = randn((37, 256), 1), randn((37, 12), 2, 2.0)
    q, s = fq.quant_per_token(x)
    r = moe.moe_route(logits, 3)
    parts = []
    for a, b in ((0, 5), (5, 12)):
        offsets, tokens, places = moe.moe_order(r.experts - a, b - a)
        y = moe.w8a8_grouped_mm_silu_mul(q, layer.w13[a:b].transpose(1, 2), s, layer.s13[a:b], offsets, rows=tokens)
        q2, s2 = fq.quant_per_token(torch.nan_to_num(y))
        y = moe.w8a8_grouped_mm(q2, layer.w2[a:b].transpose(1, 2), s2, layer.s2[a:b], offsets, torch.float32)
        parts.append(moe.moe_combine(y, r.weights, places, base=parts[-1] if parts else None))
    want = layer(x, logits).double()
    # each expert's output is rounded to bf16 in the whole layer and not in the parts, and the sum
    # once more: half a step each, of values that may be larger than the sum
    assert (parts[1].double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_custom_ops_run():
    ops = torch.ops.int8_linear
    logits = randn((9, 12), 2, 2.0)
    r = moe.moe_route(logits, 3)
    for a, b in zip(ops.moe_route(logits, 3, "softmax", True), r):
        assert torch.equal(a, b)
    for a, b in zip(ops.moe_order(r.experts, 12), r[2:]):
        assert torch.equal(a, b)
    p = problem([4] * 12, 64, 32, tokens=9)
    args = (p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], r.offsets)
    y = ops.w8a8_grouped_mm(*args, torch.bfloat16, None, r.tokens)
    assert torch.equal(y, moe.w8a8_grouped_mm(*args, rows=r.tokens))
    h = ops.w8a8_grouped_mm_silu_mul(*args, torch.bfloat16, None, r.tokens)
    assert torch.equal(h, moe.w8a8_grouped_mm_silu_mul(*args, rows=r.tokens))
    assert torch.equal(ops.moe_combine(y, r.weights, r.places, None), moe.moe_combine(y, r.weights, r.places))


# ------------------------------------------------------------------ the C++ binding
def test_the_binding_takes_plain_calls_and_gives_the_same(monkeypatch):
    from int8_linear import _lib
    f = _lib.fast()
    assert f is not None
    logits = randn((9, 12), 2, 2.0)
    p = problem([4] * 12, 64, 32, tokens=9)
    bias = randn((12, 32), 3)
    base = randn((9, 32), 4)

    def calls():
        r = moe.moe_route(logits, 3, scoring="sigmoid", renormalize=False)
        args = (p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], r.offsets)
        y = moe.w8a8_grouped_mm(*args, torch.float16, bias, rows=r.tokens)
        h = moe.w8a8_grouped_mm_silu_mul(*args, rows=r.tokens, out=torch.zeros(27, 16, dtype=torch.bfloat16, device="cuda"))
        z = moe.moe_combine(y, r.weights, r.places, base=base.half())
        return [*r, *moe.moe_order(r.experts, 10), y, h, z]
    before = f.launches()
    fast = calls()
    assert f.launches() == before + 5
    monkeypatch.setattr("int8_linear.moe._fast", lambda *a: None)
    slow = calls()
    assert f.launches() == before + 5
    for a, b in zip(fast, slow):
        assert torch.equal(a, b)


def test_the_binding_declines_a_lost_gradient():
    p = problem([4, 4], 64, 32)
    for name in ("sa", "sb"):
        args = dict(p, **{name: p[name].clone().requires_grad_()})
        with pytest.raises(NotSupported, match="no gradient"):
            moe.w8a8_grouped_mm(args["a"], args["w"].transpose(1, 2), args["sa"], args["sb"], args["offsets"])
    with pytest.raises(NotSupported, match="no gradient"):
        moe.moe_route(torch.zeros(2, 4, device="cuda", requires_grad=True), 2)
    y = torch.zeros(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(NotSupported, match="no gradient"):
        moe.moe_combine(y, torch.zeros(2, 2, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ every schedule
@pytest.mark.parametrize("each", [1, 5, 6, 13, 14, 19, 20, 40, 63, 64, 200, 256])
@pytest.mark.parametrize("k,n", [(128, 64), (144, 80), (896, 96), (1024, 272), (1040, 48), (1920, 320), (4112, 160)])
def test_mm_at_the_borders_of_the_schedules(each, k, n):
    """Each schedule at a K of whole and broken steps, shorter and longer than what it holds ahead."""
    spread = [max(0, each + d) for d in (-3, 0, 4, -each, 0, each - 1)]
    p = problem(spread + [6 * each - sum(spread)] if sum(spread) < 6 * each else spread, k, n, tokens=33)
    check_mm(p)
    check_mm(p, torch.float16, randn((p["w"].shape[0], n), 1, 1.0, torch.float16))
    check_mm(p, silu=True)
    check_mm(p, torch.float32, silu=True)


def test_mm_operands_far_apart():
    """Offsets past 32 bits: rows of A, experts, rows of the output."""
    k, n = 256, 64
    p = problem([3, 20, 70], k, n, tokens=3)
    far = torch.zeros(2 * 1_100_000_000 + k, dtype=torch.int8, device="cuda")
    a = far.as_strided((3, k), (1_100_000_000, 1))
    a.copy_(p["a"])
    q = dict(p, a=a)
    check_mm(q)
    check_mm(q, silu=True)
    w = torch.zeros(2 * 1_100_000_000 + n * k, dtype=torch.int8, device="cuda").as_strided(
        (3, n, k), (1_100_000_000, k, 1))
    w.copy_(p["w"])
    check_mm(dict(p, w=w))
    del far, w, a, q
    out = torch.zeros(92 * 50_000_000 + n, dtype=torch.bfloat16, device="cuda").as_strided((93, n), (50_000_000, 1))
    check_mm(p, out=out)


def test_combine_rows_far_apart():
    y = torch.zeros(3 * 1_200_000_000 + 64, dtype=torch.bfloat16, device="cuda").as_strided((4, 64), (1_200_000_000, 1))
    y.copy_(randn((4, 64), 1))
    w = torch.rand(5, 2, device="cuda")
    check_combine(y, w, places_of(5, 2, 4, 1))
