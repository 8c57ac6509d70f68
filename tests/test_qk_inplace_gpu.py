"""qk_norm_rope in place is an in-place operation to autograd: a backward that saved what it wrote over
is refused, as after torch's own."""

from __future__ import annotations

import pytest
import torch

from int8_linear import qk_rope

pytestmark = pytest.mark.gpu


def test_a_backward_that_saved_the_heads_is_refused():
    qkv = torch.randn(6, 4 * 64, device="cuda").bfloat16()
    q, k = qkv[:, :128].unflatten(1, (2, 64)), qkv[:, 128:192].unflatten(1, (1, 64))
    cs, pos = qk_rope.rope_cos_sin(16, 64), torch.arange(6, device="cuda")
    leaf = torch.ones(4 * 64, device="cuda").bfloat16().requires_grad_()
    kept = (leaf * qkv).sum()                                # saves qkv
    qk_rope.qk_norm_rope(q, k, None, None, cs, pos, 1e-6)    # leaves it as it is
    kept.backward(retain_graph=True)
    assert torch.isfinite(leaf.grad).all()
    before = q._version, k._version
    qo, ko = qk_rope.qk_norm_rope(q, k, None, None, cs, pos, 1e-6, inplace=True)
    assert q._version > before[0] and k._version > before[1] and qo is q and ko is k
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


def test_in_place_in_inference_mode():
    with torch.inference_mode():
        q, k = (torch.randn(3, n, 64, device="cuda").bfloat16() for n in (2, 1))
        cs, pos = qk_rope.rope_cos_sin(16, 64), torch.arange(3, device="cuda")
        want = qk_rope.qk_norm_rope(q, k, None, None, cs, pos, 1e-6)
        qk_rope.qk_norm_rope(q, k, None, None, cs, pos, 1e-6, inplace=True)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
