"""8-bit cache operators on the CPU where they can go wrong: host reads, caches that share memory, the decoder's tables."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses import FakeTensorMode

from priml_b200 import ops
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


def _halves() -> tuple[list, list]:
    """(k, v, k scales, v scales) cut from one buffer each: ones that share a part, ones that do not."""
    rows = torch.zeros(2, 4, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales, own = torch.ones(2, 4, 2), torch.ones(2, 2, 2)
    pairs = rows.view(4, 2, 64, 64)
    shared = [
        (rows[:, :2], rows[:, 1:3], scales[:, :2], scales[:, 2:]),  # a head of both
        (rows[:, 0:4:2], rows[:, 2:4], scales[:, :2], scales[:, 2:]),  # strides of their own
        (rows[:, :2], rows[:, 2:], scales[:, 1:3], scales[:, 2:]),
        (rows[:, :2], rows.flatten()[64 * 64 + 1024 :][: 4 * 64 * 64].view(2, 2, 64, 64), own, own.clone()),  # half a head
        (rows[:, :2], rows[:, :2], own, own.clone()),
        (rows[:1, :2].expand(2, -1, -1, -1), rows[:, 2:], own, own.clone()),  # one cache for both sequences
    ]
    apart = [
        (rows[:, :2], rows[:, 2:], scales[:, :2], scales[:, 2:]),
        (rows[:, 0::2], rows[:, 1::2], scales[:, 0::2], scales[:, 1::2]),
        (rows[:, :2], rows[:, 2:].clone(), scales[:, 2:], scales[:, :2].clone()),
        (pairs[:2], pairs[2:], own, own.clone()),
        (pairs[0::2], pairs[1::2], scales.view(4, 2, 2)[0::2], scales.view(4, 2, 2)[1::2]),
        (pairs.transpose(0, 1)[:, :2], pairs.transpose(0, 1)[:, 2:], own, own.clone()),  # heads outside sequences
    ]
    return shared, apart


@pytest.mark.parametrize("which", range(6))
def test_append_refuses_caches_that_share_a_part(which: int) -> None:
    shared, apart = _halves()
    q, x, n = torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 2, 64), torch.tensor([3, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="of their own|overlap"):
        ops.rotary_append(q, x, x, *shared[which], n)
    assert ops.rotary_append(q, x, x, *apart[which], n) is q


def test_a_decoder_leaves_the_model_its_rotary_table() -> None:
    """A captured training step reads the table's memory, and the next one would have to make it again."""
    from priml_b200.inference import Decoder
    from priml_b200.models.presets import tiny_lm

    model = tiny_lm().make().eval()
    rope = model.blocks[0].attn.rope
    table = rope.table(24, torch.device("cpu"))
    dec = Decoder(model, batch=1, max_seq=64, kv_dtype=torch.float8_e4m3fn)
    assert rope.table(24, torch.device("cpu"))[0] is table[0]
    for own, whole in zip((dec.caches[0].cos, dec.caches[0].sin), rope(torch.arange(64)), strict=True):
        assert torch.equal(own, whole[:, 0])


def test_layers_with_equal_factors_share_one_rotary_table() -> None:
    from priml_b200.inference import Decoder
    from priml_b200.models.presets import tiny_lm
    from priml_b200.models.rope import RoPE

    model = tiny_lm().make().eval()
    dec = Decoder(model, batch=1, max_seq=64, kv_dtype=torch.float8_e4m3fn)
    a, c = dec.caches
    assert a.cos is c.cos and a.sin is c.sin
    model.blocks[1].attn.rope = RoPE.Config(32, base=5e5).make()
    other = Decoder(model, batch=1, max_seq=64, kv_dtype=torch.float8_e4m3fn)
    a, c = other.caches
    assert torch.equal(a.cos, dec.caches[0].cos) and not torch.equal(a.cos, c.cos)
