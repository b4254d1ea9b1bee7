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


def _inputs() -> tuple[torch.Tensor, ...]:
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn(2, 6, 4, 24, generator=g).cuda(), torch.randn(2, 6, 2, 24, generator=g).cuda()
    ang = torch.randn(2, 6, 1, 4, generator=g).cuda()
    return q, k, ang.cos(), ang.sin()


@pytest.mark.parametrize("interleave", [False, True])
def test_forward_mode_and_function_transforms(interleave: bool) -> None:
    import torch.autograd.forward_ad as fw

    from priml_b200.models.rope import RoPE
    from priml_b200.ops import reference

    q, k, cos, sin = _inputs()
    want = reference.rotate(q, cos, sin, interleave), reference.rotate(k, cos, sin, interleave)

    def turn(a: torch.Tensor, c: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return RoPE.rotate(a, c, cos, sin, interleave)

    with fw.dual_level():
        out = turn(fw.make_dual(q, q), k)
        primal, tangent = fw.unpack_dual(out[0])
        assert torch.equal(primal, want[0]) and torch.equal(tangent, want[0]) and torch.equal(out[1], want[1])
        learned = fw.make_dual(cos, torch.ones_like(cos))
        assert fw.unpack_dual(RoPE.rotate(q, k, learned, sin, interleave)[1]).tangent is not None
    for a, c in zip(torch.func.jvp(turn, (q, k), (q, k))[1], want, strict=True):
        assert torch.equal(a, c)
    many = torch.func.vmap(turn)(torch.stack([q, q]), torch.stack([k, k]))
    assert torch.equal(many[0][1], want[0]) and torch.equal(many[1][0], want[1])
    grad = torch.func.grad(lambda a: turn(a, k)[0].sum())(q)
    again = q.clone().requires_grad_()
    turn(again, k)[0].sum().backward()
    assert torch.equal(grad, again.grad)


def test_compiled_without_a_graph_break() -> None:
    from priml_b200.models.rope import RoPE

    q, k, cos, sin = _inputs()
    run = torch.compile(lambda *a: RoPE.rotate(*a, True), fullgraph=True, backend="eager")
    for a, c in zip(run(q, k, cos, sin), RoPE.rotate(q, k, cos, sin, True), strict=True):
        assert torch.equal(a, c)


@pytest.mark.parametrize("interleave", [False, True])
def test_traced_graphs_rotate_the_inputs_that_they_are_given(interleave: bool) -> None:
    from torch.fx.experimental.proxy_tensor import make_fx

    from priml_b200.models.rope import RoPE

    q, k, cos, sin = _inputs()

    def turn(a: torch.Tensor, c: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return RoPE.rotate(a, c, cos, sin, interleave)

    for run in (make_fx(turn)(q, k), torch.jit.trace(turn, (q, k))):
        for a, c in zip(run(q + 1, k * 2), turn(q + 1, k * 2), strict=True):
            # A traced graph may be compiled, with a product and a sum rounded once together: the unrounded product, under
            # 2**3, is then off by at most 2**-22. A result held from the tracing is off by one and more.
            torch.testing.assert_close(a, c, rtol=0, atol=2.0**-21)
