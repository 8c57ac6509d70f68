"""The router on the values that its keys treat apart, in every type: ties, signed zeros, subnormals,
infinities, NaN of either sign, masks of the type's lowest value and tokens that may take no expert; in each
of its kernels (by the number of tokens) and with wide and single loads (by the number of experts)."""

from __future__ import annotations

import math

import pytest
import torch

import moe_restated as ref
from helpers import say
from int8_linear import moe

gpu = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PICKS = 5
# (tokens, the first one's kind): pairs up to 64 (one wave orders them), one workgroup, two launches
TOKENS = [(12, 0), (12, 5), (60, 0), (65, 3), (700, 7)]


def rows_of(e: int, dt: torch.dtype) -> torch.Tensor:
    """[17, E] of the type, a kind of row each."""
    info, g = torch.finfo(dt), torch.Generator().manual_seed(e)
    x = torch.randn(17, e, generator=g).to(dt)
    x[0] = 0.0
    x[0, 1::2] = -0.0                             # all equal
    x[1] = -1.0
    x[1, e // 2:] = 1.0                           # the best in later lanes
    x[2] = (torch.arange(e) % 3 - 1).to(dt)
    x[3] = -math.inf                              # a token that may take none
    x[4, 3:] = -math.inf                          # fewer than it takes
    x[5] = math.nan
    x[6, ::3] = math.nan
    x[7, e // 2] = math.inf
    x[8, 5] = x[8, e - 1] = math.inf
    x[9] = info.min                               # pickable, all alike
    x[10, 1:] = info.min
    x[11, ::2] = -math.inf
    x[12] = -200.0                                # sigmoids that are 0 in fp32: equal shares all the same
    x[13, 0] = info.max
    x[13, 1] = info.min
    tiny = info.smallest_normal * info.eps        # the smallest subnormal
    x[14] = ((torch.arange(e) * 7 % 11 - 5).double() * tiny).to(dt)
    whole = torch.int32 if dt == torch.float32 else torch.int16
    for row, sign in ((15, 0), (16, 1)):          # NaN of either sign with the smallest and the largest payload
        b = x[row].view(whole)
        inf = torch.full((1,), math.inf, dtype=dt).view(whole).item()
        low = inf + 1 - (sign << (torch.iinfo(whole).bits - 1))
        high = torch.iinfo(whole).max - (sign << (torch.iinfo(whole).bits - 1))
        b[::4], b[1::4] = low, high
        x[row, 2::8] = -math.inf
    return x


def test_the_rows_hold_what_they_say():
    for dt in DT.values():
        x = rows_of(70, dt)
        assert x[15].isnan().sum() == x[16].isnan().sum() == 36 and (x[16, 0].signbit() and not x[15, 0].signbit())
        assert x[14].double().unique().numel() == 11 and x[14].abs().max() < torch.finfo(dt).smallest_normal
        assert x[12].isfinite().all() and x[13, 0].isfinite()


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("e", [70, 128, 200, 512])
@pytest.mark.parametrize("t,first", TOKENS)
def test_picks_order_and_weights(dt, e, t, first):
    kinds = rows_of(e, DT[dt])
    x = kinds[(torch.arange(t) + first) % len(kinds)]
    for scoring in moe.SCORING:
        for renormalize in (False, True):
            say(f"route {t} of {e}, {dt}, {scoring}, renormalize {renormalize}")
            r = moe.moe_route(x.cuda(), PICKS, scoring=scoring, renormalize=renormalize)
            experts = ref.picks(x, PICKS)
            assert torch.equal(r.experts.cpu(), experts)
            for got, want in zip((r.offsets, r.tokens, r.places), ref.order(experts, e)):
                assert torch.equal(got.cpu(), want)
            want, got = ref.weights(x, experts, scoring, renormalize), r.weights.cpu().double()
            assert not got.isnan().any() and (got[experts < 0] == 0).all()
            # The argument x - max (or x of a sigmoid) is off by 104 * 2^-24 at most where its exponential
            # is not 0, the exponential by 2^-22, its sum of up to 32 terms in a lane and 4 levels of
            # lanes by 36 * 2^-24, a quotient by 2^-24: below 146 * 2^-24, and the total by the same again,
            # 2^-15 together.  Below the smallest normal number, 1e-37.
            assert ((got - want).abs() <= 2.0 ** -15 * want + 1e-37).all()
