"""Every schedule of the grouped product on the GPU: each output and bias type, several tiles a workgroup and more
than its table holds, both sides of each border, offsets and rows out of range.

The products are compared bit for bit with the definition's: sums in float64 on the device (exact: below
2^53), then the epilogue's float32 steps, an operation each.
"""

from __future__ import annotations

import math

import pytest
import torch

from helpers import say
from int8_linear import moe
from int8_linear.kernel import w8a8_mm
from test_grouped_tiles import BORDERS, LONG, MANY, schedule_of

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TOKENS = 400


def problem(sizes, n, k, seed=0, gone=9):
    """Operands of experts with these rows, read through rows=; `gone` more rows belong elsewhere."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    e, r = len(sizes), sum(sizes) + gone

    def codes(*shape):
        return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device="cuda")

    def scales(*shape):
        return torch.rand(shape, generator=g, device="cuda") * 0.01 + 1e-3
    return dict(a=codes(TOKENS, k), w=codes(e, n, k), sa=scales(TOKENS, 1), sb=scales(e, n),
                offsets=torch.tensor([0, *sizes]).cumsum(0).int().cuda(),
                rows=torch.randint(0, TOKENS, (r,), generator=g, dtype=torch.int32, device="cuda"))


def bias_of(p, dt):
    g = torch.Generator(device="cuda").manual_seed(9)
    return torch.randn(p["sb"].shape, generator=g, device="cuda").to(dt)


def call(p, dt, bias, silu, out=None, offsets=None, rows=None):
    f = moe.w8a8_grouped_mm_silu_mul if silu else moe.w8a8_grouped_mm
    return f(p["a"], p["w"].transpose(1, 2), p["sa"], p["sb"], p["offsets"] if offsets is None else offsets, dt,
             bias, rows=p["rows"] if rows is None else rows, out=out)


def values(p, e, rows, bias):
    """The fp32 epilogue values of these rows with expert e's weight; NaN where the row is outside."""
    ok = (rows >= 0) & (rows < TOKENS)
    r = torch.where(ok, rows, 0).long()
    v = (p["a"][r].double() @ p["w"][e].double().t()).float()
    v = v * torch.where(ok, p["sa"].view(-1)[r], math.nan)[:, None]
    v = v * p["sb"][e]
    return v if bias is None else v + bias[e].float()


def check(p, dt, bias=None, silu=False, ends=None, **kw):
    """One call into an output of sevens; ends: the offsets as they are held, where others are passed."""
    n = p["w"].shape[1]
    r, width = p["rows"].numel(), n // 2 if silu else n
    out = torch.full((r, width), 7.0, dtype=dt, device="cuda")
    call(p, dt, bias, silu, out, **kw)
    rows = kw.get("rows", p["rows"])
    ends = p["offsets"].tolist() if ends is None else ends
    assert (out[ends[-1]:] == 7).all() and (out[:ends[0]] == 7).all()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if lo == hi:
            continue
        got, v = out[lo:hi], values(p, e, rows[lo:hi], bias)
        if not silu:
            want = v.to(dt)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1), want.nan_to_num(1))
            continue
        g, u = v.double().chunk(2, 1)
        want = g * torch.sigmoid(g) * u
        # exp(-g) is off by |g| 2^-24 (16-bit outputs: its argument is rounded) and 2^-22, the sum, the
        # quotient and the product by 2^-22 together; then half a step of the output, and of its smallest
        # numbers.  A sigmoid below 2^-126 may be 0: what is lost is |g u| 2^-126.
        rel = 2.0 ** -20 + (g.abs() * 2.0 ** -23 if dt != torch.float32 else 0)
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 + (g * u).abs() * 2.0 ** -126
        bound = want.abs() * (rel + torch.finfo(dt).eps / 2 * (1 + 2 ** -9)) + tiny
        fits = want.abs() < torch.finfo(dt).max
        bad = got.isnan() != want.isnan()
        bad |= fits & ~((got.double() - want).abs() <= bound)
        assert not bad.any()


@pytest.mark.parametrize("bias", [None, "bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bm,stream", list(MANY))
def test_several_tiles_a_workgroup(bm, stream, dt, bias):
    sizes, n, k = MANY[bm, stream]
    say(f"grouped {bm} rows, streamed {stream}, {len(sizes)} experts {k} -> {n}, {dt}, bias {bias}")
    p = problem(sizes, n, k)
    assert schedule_of(p["rows"].numel(), len(sizes), n, k) == (bm, 256, int(stream))
    b = None if bias is None else bias_of(p, DT[bias])
    check(p, DT[dt], b)
    check(p, DT[dt], b, silu=True)


@pytest.mark.parametrize("dt,bias,silu", [("bf16", None, False), ("fp16", "fp16", True), ("fp32", "bf16", False)])
@pytest.mark.parametrize("bm,stream", list(LONG))
def test_more_tiles_a_workgroup_than_its_table_holds(bm, stream, dt, bias, silu):
    sizes, n, k = LONG[bm, stream]
    say(f"grouped {bm} rows, streamed {stream}, {len(sizes)} experts {k} -> {n}, {dt}, silu {silu}")
    p = problem(sizes, n, k)
    assert schedule_of(p["rows"].numel(), len(sizes), n, k) == (bm, 256, int(stream))
    check(p, DT[dt], None if bias is None else bias_of(p, DT[bias]), silu)


@pytest.mark.parametrize("border,e,n,k", [b[:4] for b in BORDERS])
@pytest.mark.parametrize("rest", [-1, 0])
def test_both_sides_of_each_border(border, e, n, k, rest):
    say(f"grouped {border} rows an expert {rest:+d}, {e} experts {k} -> {n}")
    sizes = [max(0, border + d) for _ in range(e) for d in (-3, 0, 4, -border, border, -1)][:e]
    total = border * e + rest
    for i in range(e):                       # (the spread is cut or filled up to the average)
        sizes[i] = min(sizes[i], total - sum(sizes[:i]))
    sizes[-1] += total - sum(sizes)
    p = problem(sizes, n, k, gone=0)
    check(p, torch.bfloat16)
    if n % 16 == 0:
        check(p, torch.float16, bias_of(p, torch.float16), silu=True)


SCHEDULES = [*MANY.values(), ([1, 0, 7, 3, 0, 9], 64, 256), ([13, 0, 25, 3, 17, 9], 64, 256),
             ([40, 0, 65, 3, 64, 29], 64, 256), ([40, 0, 65, 3, 64, 29], 60, 100)]


@pytest.mark.parametrize("sizes,n,k", SCHEDULES)
@pytest.mark.parametrize("silu", [False, True])
def test_rows_out_of_range_give_nan(sizes, n, k, silu):
    say(f"grouped, bad rows, {len(sizes)} experts {k} -> {n}, silu {silu}")
    p = problem(sizes, n, k)
    rows = p["rows"].clone()
    end = sum(sizes)
    for i, v in zip((0, 3, end // 3, end // 2 + 1, end - 1), (-1, TOKENS, 2 ** 31 - 1, -2 ** 31, -2)):
        rows[i] = v
    check(p, torch.float32, silu=silu, rows=rows)


@pytest.mark.parametrize("sizes,n,k", SCHEDULES)
@pytest.mark.parametrize("broken", ["descending", "past the rows", "both"])
def test_offsets_out_of_range_are_held(sizes, n, k, broken):
    """Each within the rows, and to those before it: a row is one expert's, the first to claim it."""
    say(f"grouped, {broken} offsets, {len(sizes)} experts {k} -> {n}")
    p = problem(sizes, n, k, gone=0)
    r, e = p["rows"].numel(), len(sizes)
    offsets = p["offsets"].tolist()
    if broken != "past the rows":
        offsets[0], offsets[2], offsets[e // 2] = -7, r // 3, 1
    if broken != "descending":
        offsets[-3], offsets[-2], offsets[-1] = r + 1000, 2 ** 31 - 1, -2 ** 31
    held, most = [], 0
    for x in offsets:
        most = max(most, min(max(x, 0), r))
        held.append(most)
    assert held != offsets
    check(p, torch.bfloat16, ends=held, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("sizes,n,k", SCHEDULES)
def test_rows_before_the_first_offset_are_left(sizes, n, k):
    say(f"grouped, offsets from 5 on, {len(sizes)} experts {k} -> {n}")
    p = problem(sizes, n, k)
    p["offsets"] += 5
    check(p, torch.bfloat16)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("r", [3, 30, 70, 500])
def test_one_expert_is_the_dense_product(r, bias, dt):
    """The arithmetic of w8a8_mm, bit for bit."""
    say(f"grouped and dense, {r} rows, {dt}, bias {bias}")
    p = problem([r], 512, 1024, gone=0)
    b = bias_of(p, DT[dt]) if bias else None
    rows = p["rows"].clamp(max=TOKENS - 1).long()
    a, sa = p["a"][rows], p["sa"][rows]
    want = w8a8_mm(a, p["w"][0].t(), sa, p["sb"].t(), DT[dt], b[0] if bias else None)
    assert torch.equal(call(p, DT[dt], b, False), want)


def test_two_streams_at_once():
    """Two products in flight together, each of several tiles a workgroup."""
    sizes, n, k = MANY[256, False]
    say("grouped on two streams")
    ps = [problem(sizes, n, k, seed) for seed in (1, 2)]
    want = [call(p, torch.bfloat16, None, False) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(3):
        got = []
        for p, s in zip(ps, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(call(p, torch.bfloat16, None, False))
        torch.cuda.synchronize()
        assert all(torch.equal(a[:sum(sizes)], b[:sum(sizes)]) for a, b in zip(got, want))
