"""Values past the rotated ones are normalized only: what one of them holds (a NaN or an infinity, its own
or its weight's) does not reach another."""

from __future__ import annotations

import pytest
import torch

import mx_restated as mx
from helpers import say
from int8_linear import qk_rope
from test_qk_rope_gpu import EPS, _case, _check, _views

pytestmark = pytest.mark.gpu

# (head size, rotated values): 16-byte runs, 8-byte runs, any
SIZES = [(128, 64), (256, 32), (80, 40), (72, 24), (96, 24), (80, 20), (17, 16)]


def _run(c, interleaved):
    q, k = _views(c, c["qkv"].cuda())
    return qk_rope.qk_norm_rope(q, k, c["qw"].cuda(), c["kw"].cuda(), c["cs"].cuda(), c["pos"].cuda(),
                                EPS, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d,rot", SIZES)
def test_a_non_finite_weight_past_the_rotated_values(d, rot, value, interleaved):
    say(f"qk_norm_rope heads of {d}, {rot} rotated, a weight of {value}, interleaved={interleaved}")
    for at in {rot, d - 1, (rot + d) // 2}:
        c = _case(9, 5, 2, d, rot)
        c["qw"][at] = value
        qo, ko = _run(c, interleaved)
        others = [i for i in range(d) if i != at]
        assert not torch.isfinite(qo[..., at]).any() and torch.isfinite(qo[..., others]).all()
        # the rest as without it
        c["qw"][at] = 1.0
        want = _run(c, interleaved)
        assert torch.equal(qo[..., others], want[0][..., others]) and torch.equal(ko, want[1])
        _check(ko, c["k"], c["kw"], c, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", SIZES)
def test_an_infinite_value_past_the_rotated_ones(d, rot, interleaved):
    """The head's norm is infinite: its finite values become zeros, the infinite one a NaN."""
    say(f"qk_norm_rope heads of {d}, {rot} rotated, an infinite value, interleaved={interleaved}")
    for at in {rot, d - 1, (rot + d) // 2}:
        c = _case(4, 3, 1, d, rot)
        c["qkv"][2, d + at] = float("inf")
        qo, ko = _run(c, interleaved)
        want = mx.qk(c["q"], c["qw"], c["cs"], c["pos"], EPS, interleaved)
        assert torch.isnan(want[2, 1]).sum() == 1
        assert torch.equal(torch.isnan(qo.cpu()), torch.isnan(want))
        assert (qo[2, 1][[i for i in range(d) if i != at]] == 0).all()
        _check(ko, c["k"], c["kw"], c, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 64), (80, 40), (80, 20)])
def test_zeros_past_the_rotated_values_keep_their_signs(d, rot, interleaved):
    c = _case(5, 4, 2, d, rot)
    c["q"][..., rot::2] = -0.0
    c["q"][..., rot + 1::4] = 0.0
    qo, _ = _run(c, interleaved)
    past = c["q"][..., rot:]
    assert torch.equal(torch.signbit(qo[..., rot:].cpu())[past == 0], torch.signbit(past)[past == 0])
