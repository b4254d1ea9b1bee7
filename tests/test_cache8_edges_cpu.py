"""8-bit cache operators on the CPU where they can go wrong: host reads, caches that share memory, the decoder's tables."""

from __future__ import annotations

import torch
from torch._subclasses import FakeTensorMode

from priml_b200.ops import reference


def test_the_torch_form_reads_nothing_on_the_host() -> None:
    """A CUDA graph cannot hold a host read, and a tensor without data cannot give one."""
    b, s, h, hkv, t, d = 2, 5, 4, 2, 70, 16
    with FakeTensorMode():
        k, v = (torch.empty(b, hkv, t, d).to(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.empty(b, hkv, 3) for _ in range(2))
        q, x = torch.empty(b, s, h, d), torch.empty(b, s, hkv, d)
        n = torch.empty(b, dtype=torch.int32)
        table = torch.empty(t, d // 2)
        out = reference.rotary_append(q, x, x, k, v, ks, vs, n, table, table, False)
        seen = reference.cache_attention(out, k, v, ks, vs, n, scale=0.25, window=7, offset=s)
    assert seen.shape == (b, s, h, d)
