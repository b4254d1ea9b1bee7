"""Rotary embedding of tensors that have no data: shapes and types are traced without a kernel."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses import FakeTensorMode

from priml_b200.models.rope import RoPE


@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fake_tensors(device: str, interleave: bool) -> None:
    with FakeTensorMode():
        q = torch.empty(2, 6, 4, 24, device=device, dtype=torch.float16)
        k = torch.empty(2, 6, 2, 24, device=device, dtype=torch.float16)
        cos = torch.empty(2, 6, 1, 4, device=device)
        out = RoPE.rotate(q, k, cos, cos, interleave)
    assert [x.shape for x in out] == [q.shape, k.shape] and out[0].dtype == torch.float16 and out[1].device == k.device
