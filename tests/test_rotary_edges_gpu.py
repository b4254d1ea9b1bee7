"""Rotary embedding in the calls that its kernel does not take: odd widths, function transforms, traced tensors."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rot", [(65, 64), (65, 32), (3, 2), (129, 6)])
def test_odd_head_widths_keep_their_last_channel(d: int, rot: int, dtype: torch.dtype, interleave: bool) -> None:
    from priml_b200 import ops
    from priml_b200.models.rope import RoPE
    from priml_b200.ops import native, reference

    g = torch.Generator().manual_seed(d + rot)
    q = torch.randn(2, 5, 3, d, generator=g).to(dtype).cuda().requires_grad_()
    k = torch.randn(2, 5, 1, d, generator=g).to(dtype).cuda().requires_grad_()
    ang = torch.randn(2, 5, 1, rot // 2, generator=g).cuda()
    gq, gk = torch.randn(2, 5, 3, d, generator=g).to(dtype).cuda(), torch.randn(2, 5, 1, d, generator=g).to(dtype).cuda()
    want = [reference.rotate(x, ang.cos(), ang.sin(), interleave) for x in (q, k)]
    ref = torch.autograd.grad(want, (q, k), (gq, gk))
    for turn in (lambda *a: ops.rotary(*a, interleave=interleave), lambda *a: RoPE.rotate(*a, interleave)):
        # memory that the outputs are likely to get: what is not written shows
        junk = [torch.full_like(x, 1e4) for x in (q, k, q, k)]
        del junk
        out = turn(q, k, ang.cos(), ang.sin())
        got = torch.autograd.grad(out, (q, k), (gq, gk))
        for a, c in zip((*out, *got), (*want, *ref), strict=True):
            assert torch.equal(a, c)
    with pytest.raises(ValueError, match="even"):
        native().rotary(q.detach(), k.detach(), ang.cos(), ang.sin(), interleave)
