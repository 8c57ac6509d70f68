"""The grouped product at the ends of what its indexes count."""

from __future__ import annotations

import pytest
import torch

from helpers import ints, say
from int8_linear import moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("r,k", [(4, 64), (20, 64), (300, 64), (2100, 64), (300, 60)])
def test_row_scales_past_32_bits_of_bytes(r, k, silu):
    """Rows from 2^30 on have their own scales in every schedule: one row of codes, expanded to more
    rows than 32 bits of bytes can tell the scales of apart."""
    m, n = 2 ** 30 + 4096, 64
    say(f"grouped {m} scales, {r} rows, K {k}, silu {silu}")
    row, w = ints((1, k), 1), ints((1, n, k), 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    sa = torch.zeros(m, device="cuda")
    for part in (slice(0, 4096), slice(m - 4096, m)):
        sa[part] = torch.rand(4096, generator=g, device="cuda") * 1e-3 + 1e-4
    sb = torch.rand((1, n), generator=g, device="cuda") * 0.01 + 1e-3
    rows = torch.arange(m - r, m, device="cuda").int()
    offsets = torch.tensor([0, r], dtype=torch.int32, device="cuda")
    call = moe.w8a8_grouped_mm_silu_mul if silu else moe.w8a8_grouped_mm
    got = call(row.expand(m, k), w.transpose(1, 2), sa, sb, offsets, torch.float32, rows=rows)
    acc = row.cpu().double() @ w[0].cpu().double().t()
    v = acc.float() * sa[m - r:].cpu()[:, None] * sb.cpu()
    if not silu:
        assert torch.equal(got.cpu(), v)
        return
    gate, up = v.double().chunk(2, 1)
    want = gate * torch.sigmoid(gate) * up
    # exp(-g) is off by |g| 2^-24 and 2^-22, the sum, the quotient and the product by 2^-22 together (g is small
    # here), then half a step
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -20 * want.abs() + 1e-38).all()
