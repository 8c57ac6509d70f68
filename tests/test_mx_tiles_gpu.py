"""Every macro tile of the MXFP4 product on the GPU, with several tiles a workgroup and with K in parts,
each output and bias type, against the product of the decoded operands in float64.

The sums are exact in fp32 (multiples of a power of two u whose magnitudes sum below 2^23 u, checked),
so the outputs are compared bit for bit.
"""

from __future__ import annotations

import pytest
import torch

from helpers import say
from int8_linear import mxfp4
from test_mx_tiles import MANY, PARTS, tile_of

pytestmark = pytest.mark.gpu

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _operand(rows, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, generator=g, device="cuda")
    s = torch.randint(126, 129, (rows, k // 32), dtype=torch.uint8, generator=g, device="cuda")
    table = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device="cuda")
    v = torch.empty(rows, k, dtype=torch.float64, device="cuda")
    v[:, 0::2], v[:, 1::2] = table[(q & 15).int()], table[(q >> 4).int()]
    v.unflatten(1, (-1, 32)).mul_(torch.exp2(s.double() - 127)[..., None])
    return q, s, v


@pytest.mark.parametrize("tile,parts,m,n,k", MANY + PARTS)
def test_every_tile(tile, parts, m, n, k):
    assert tile_of(m, n, k) == (tile, parts)
    a, sa, av = _operand(m, k, 1)
    w, sw, wv = _operand(n, k, 2)
    assert (av.abs() @ wv.abs().t()).max().item() + 64 < 2.0 ** (23 - 4)   # u = (1/2 * 2^-1)^2
    want = av @ wv.t()
    b = torch.randint(-64, 64, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    for dtype in TYPES:
        for bias in (None, b.to(dtype)):
            say(f"mxfp4_mm {m}x{n}x{k} tile {tile} parts {parts} {dtype} bias={bias is not None}")
            out = mxfp4.mxfp4_mm(a, w.t(), sa, sw, dtype, bias)
            ref = (want if bias is None else want + b).float().to(dtype)
            assert torch.equal(out, ref)


@pytest.mark.parametrize("tile,parts,m,n,k", [MANY[2], MANY[7], PARTS[2]])
def test_nan_scales_reach_their_rows_and_columns_only(tile, parts, m, n, k):
    """A NaN scale in a tile that is not a workgroup's first, in the last blocks of K and the first."""
    say(f"mxfp4_mm with NaN scales {m}x{n}x{k}")
    a, sa, _ = _operand(m, k, 1)
    w, sw, _ = _operand(n, k, 2)
    clean = mxfp4.mxfp4_mm(a, w.t(), sa, sw, torch.float32)
    sa[m - 1, k // 32 - 1] = 255
    sw[n - 1, 0] = 255
    out = mxfp4.mxfp4_mm(a, w.t(), sa, sw, torch.float32)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m - 1], bad[:, n - 1] = True, True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])
