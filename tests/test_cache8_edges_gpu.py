"""8-bit cache kernels where they can go wrong: rows that see nothing, block scales far apart, values that are not
finite, outlying channels, long runs whose every block shows in the output, models that no kernel covers."""

from __future__ import annotations

import pytest
import torch
from torch import Tensor

from tests.cache8_cases import filled_cache

pytestmark = pytest.mark.gpu


def _status_clean() -> None:
    from priml_b200.ops import native

    torch.cuda.synchronize()
    assert int(native().read_status(True)) == 0


def _queries(b: int, s: int, h: int, d: int, seed: int) -> Tensor:
    return (torch.randn(b, s, h, d, generator=torch.Generator().manual_seed(seed)) * 0.125).bfloat16().cuda()


def _ints(values: list[int]) -> Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("shift", [0, 14, 20, 100])
@pytest.mark.parametrize("b,s,h,hkv,d,ends", [(1, 129, 4, 2, 64, [128]), (2, 300, 4, 1, 128, [256, 100]), (3, 900, 2, 2, 64, [897, 640, 0])])
def test_queries_before_their_sequence_give_zeros_whatever_the_scales(b, s, h, hkv, d, ends, shift) -> None:  # noqa: ANN001
    """More queries than keys in row tiles that other rows see: every block of the tile holds large values."""
    from priml_b200 import ops

    t = max(ends)
    k, ks = filled_cache(b, hkv, t, d, seed=1, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=2, device="cuda")
    q = _queries(b, s, h, d, seed=3)
    out = ops.cache_attention(q, k, v, ks, vs * 2.0**shift, _ints(ends))
    base = ops.cache_attention(q, k, v, ks, vs, _ints(ends))
    _status_clean()
    for i, n in enumerate(ends):
        assert (out[i, : max(0, s - n)] == 0).all()
    # the shift moves exponents by roundings only: neighbours in bf16, 2**-7 apart, but where terms cancel
    size = (v.float().abs().amax((-1, -2)) * vs.amax(-1)).max()
    assert ((out.float() * 2.0**-shift - base.float()).abs() <= base.float().abs() * 2.0**-7 + size * 2.0**-16).all()
