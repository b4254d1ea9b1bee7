"""8-bit cache operators on the CPU: the oracle against 64 bits, refusals, and the decoder over an 8-bit cache."""

from __future__ import annotations

import pytest
import torch

from priml_b200 import ops
from priml_b200.ops import reference
from tests.cache8_cases import BLOCK, append64, attend64, filled_cache


def _inputs(b: int, s: int, h: int, hkv: int, d: int, t: int, seed: int, dtype=torch.float32):  # noqa: ANN001, ANN202
    g = torch.Generator().manual_seed(seed)
    k, ks = filled_cache(b, hkv, t, d, seed)
    v, vs = filled_cache(b, hkv, t, d, seed + 1)
    return torch.randn(b, s, h, d, generator=g).to(dtype), k, v, ks, vs


@pytest.mark.parametrize("window", [None, 0, 5, 40])
def test_attention_oracle_matches_64_bits(window: int | None) -> None:
    q, k, v, ks, vs = _inputs(4, 3, 6, 2, 16, 77, seed=1)
    ends = [77, 40, 2, 0]  # a full cache, a short one, fewer keys than queries, none
    out = ops.cache_attention(q, k, v, ks, vs, torch.tensor(ends), window=window)
    want = attend64(q, k, v, ks, vs, ends, window=window)
    # fp32 sums of 77 terms: 77 * 2**-24 relative to max|V| with room for the products' own roundings
    assert (out - want).abs().max() <= 200 * 2.0**-24 * want.abs().max().clamp_min(1) * 8
    assert out[3].abs().max() == 0 and out[2, 0].abs().max() == 0
    shifted = ops.cache_attention(q, k, v, ks, vs, torch.tensor(ends) - 3, offset=3, window=window)
    assert torch.equal(shifted, out)


def test_hidden_rows_may_hold_anything() -> None:
    q, k, v, ks, vs = _inputs(1, 4, 2, 1, 16, 64, seed=2)
    clean = ops.cache_attention(q, k, v, ks, vs, torch.tensor([40]))
    k.view(torch.uint8)[:, :, 40:] = 0x7F
    v.view(torch.uint8)[:, :, 40:] = 0xFF
    assert torch.equal(ops.cache_attention(q, k, v, ks, vs, torch.tensor([40])), clean)
    v.view(torch.uint8)[:, :, 39, 3] = 0x7F  # the last token's value: only the last query sees it
    out = ops.cache_attention(q, k, v, ks, vs, torch.tensor([40]))
    assert torch.equal(out[:, :3], clean[:, :3]) and out[:, 3, :, 3].isnan().all()


@pytest.mark.parametrize("start,s", [(0, 1), (0, 70), (31, 1), (31, 2), (5, 20), (32, 32), (60, 30)])
def test_append_oracle_matches_the_definition(start: int, s: int) -> None:
    b, hkv, t, d = 2, 3, 80, 16  # the last case passes the cache's end
    k, ks = filled_cache(b, hkv, t, d, seed=3)
    v, vs = filled_cache(b, hkv, t, d, seed=4)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, b, s, hkv, d, generator=g) * torch.exp2(torch.randint(-6, 7, (2, b, s, hkv, 1), generator=g).float())
    want = [append64(x[i], c, f, [start, max(0, start - 3)]) for i, (c, f) in enumerate(((k, ks), (v, vs)))]
    q = torch.randn(b, s, 6, d)
    out = ops.rotary_append(q, x[0], x[1], k, v, ks, vs, torch.tensor([start, max(0, start - 3)]))
    assert out is q
    for c, f, (held, scale) in ((k, ks, want[0]), (v, vs, want[1])):
        assert torch.equal(c.double(), held) and torch.equal(f.double(), scale)


def test_append_scale_borders_and_values_that_are_not_finite() -> None:
    k, ks = filled_cache(1, 1, 64, 16, seed=6)
    v, vs = k.clone(), ks.clone()
    x = torch.zeros(1, 1, 1, 16)
    for size, want in ((448.0, 1.0), (448.5, 2.0), (0.0, 2.0**-100), (1e-38, 2.0**-100), (3.0e38, 2.0**120), (1.75, 2.0**-8)):
        x[..., 0] = size
        ops.rotary_append(x, x, x, k, v, ks, vs, torch.tensor([32]))
        assert ks[0, 0, 1].item() == want
    x[..., 0], x[..., 1], x[..., 2] = float("inf"), float("nan"), 7.0
    ops.rotary_append(x, x, x, k, v, ks, vs, torch.tensor([32]))
    row = k[0, 0, 32].float() * ks[0, 0, 1]
    assert row[0].isnan() and row[1].isnan() and row[2].item() == 7.0 and ks[0, 0, 1].item() == 2.0**-6
    before = k.clone()
    ops.rotary_append(x, x, x, k, v, ks, vs, torch.tensor([64]))  # behind the last row
    ops.rotary_append(x, x, x, k, v, ks, vs, torch.tensor([-1]))
    assert torch.equal(before.view(torch.uint8), k.view(torch.uint8))


@pytest.mark.parametrize("interleave", [False, True])
def test_append_rotates_at_the_sequence_positions(interleave: bool) -> None:
    b, s, hkv, t, d, rot = 2, 3, 1, 64, 16, 8
    k, ks = filled_cache(b, hkv, t, d, seed=7)
    v, vs = filled_cache(b, hkv, t, d, seed=8)
    ang = torch.arange(t)[:, None] * 0.3 ** torch.arange(rot // 2)
    q, x, y = torch.randn(b, s, 2, d), torch.randn(b, s, hkv, d), torch.randn(b, s, hkv, d)
    start = torch.tensor([10, 45])
    at = start[:, None] + torch.arange(s)
    c, n = ang.cos()[at][:, :, None], ang.sin()[at][:, :, None]
    qr, kr = ops.rotary(q, x, c, n, interleave=interleave)
    want = append64(kr, k, ks, start.tolist())
    out = ops.rotary_append(q, x, y, k, v, ks, vs, start, cos=ang.cos(), sin=ang.sin(), interleave=interleave)
    assert torch.equal(out, qr) and torch.equal(k.double(), want[0]) and torch.equal(ks.double(), want[1])


@pytest.mark.parametrize("interleave", [False, True])
def test_rotary_gradients_against_differences(interleave: bool) -> None:
    g = torch.Generator().manual_seed(9)
    q, k = torch.randn(2, 3, 2, 10, generator=g).double(), torch.randn(2, 3, 1, 10, generator=g).double()
    ang = torch.randn(2, 3, 1, 3, generator=g).double()

    def turn(a: torch.Tensor, c: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        # the oracle computes in fp32: differences of 2**-10 leave its roundings at 2**-13 of the slope
        return ops.rotary(a, c, ang.cos(), ang.sin(), interleave=interleave)

    assert torch.autograd.gradcheck(turn, (q.requires_grad_(), k.requires_grad_()), eps=2.0**-10, atol=2.0**-10, nondet_tol=0)


def _good() -> dict:
    q, k, v, ks, vs = _inputs(2, 1, 4, 2, 64, 40, seed=10)
    return dict(q=q, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, lengths=torch.tensor([3, 4], dtype=torch.int32))


@pytest.mark.parametrize(
    "change,error",
    [
        (dict(q=torch.zeros(2, 64)), ValueError),
        (dict(q=torch.zeros(3, 1, 4, 64)), ValueError),
        (dict(q=torch.zeros(2, 1, 5, 64)), ValueError),
        (dict(q=torch.zeros(2, 1, 4, 32)), ValueError),
        (dict(k_cache=torch.zeros(2, 2, 40, 64)), TypeError),
        (dict(v_cache=torch.zeros(2, 2, 39, 64).to(torch.float8_e4m3fn)), ValueError),
        (dict(k_scale=torch.ones(2, 2, 1)), ValueError),
        (dict(v_scale=torch.ones(2, 2, 2).double()), ValueError),
        (dict(lengths=torch.tensor([1, 2, 3])), ValueError),
        (dict(lengths=torch.tensor([1.0, 2.0])), ValueError),
        (dict(offset=-1), ValueError),
        (dict(q=torch.zeros(2, 1, 4, 64, requires_grad=True)), RuntimeError),
    ],
)
def test_attention_refusals(change: dict, error: type) -> None:
    with pytest.raises(error):
        ops.cache_attention(**(_good() | change))


@pytest.mark.parametrize(
    "change,error",
    [
        (dict(k=torch.zeros(2, 1, 3, 64), v=torch.zeros(2, 1, 3, 64)), ValueError),
        (dict(v=torch.zeros(2, 2, 2, 64)), ValueError),
        (dict(cos=torch.ones(40, 32)), ValueError),
        (dict(cos=torch.ones(40, 33), sin=torch.ones(40, 33)), ValueError),
        (dict(cos=torch.ones(1, 40, 32), sin=torch.ones(1, 40, 32)), ValueError),
        (dict(k=torch.zeros(2, 1, 2, 64, requires_grad=True)), RuntimeError),
    ],
)
def test_append_refusals(change: dict, error: type) -> None:
    good = _good() | dict(k=torch.zeros(2, 1, 2, 64), v=torch.zeros(2, 1, 2, 64))
    with pytest.raises(error):
        ops.rotary_append(**(good | change))


def test_empty_batches_and_chunks() -> None:
    _, k, v, ks, vs = _inputs(2, 1, 4, 2, 16, 40, seed=11)
    n = torch.tensor([3, 4])
    assert ops.cache_attention(torch.zeros(2, 0, 4, 16), k, v, ks, vs, n).shape == (2, 0, 4, 16)
    e = torch.zeros(2, 0, 2, 16)
    assert ops.rotary_append(torch.zeros(2, 0, 4, 16), e, e, k, v, ks, vs, n).shape == (2, 0, 4, 16)
    assert reference.CACHE_BLOCK == BLOCK == ops.CACHE_BLOCK


# --------------------------------------------------------------------------- the cache in a decoder
def _decoders(batch: int, max_seq: int):  # noqa: ANN202
    from priml_b200.inference import Decoder
    from priml_b200.models.presets import tiny_lm

    torch.manual_seed(0)
    model = tiny_lm().make().eval()
    return Decoder(model, batch=batch, max_seq=max_seq), Decoder(
        model, batch=batch, max_seq=max_seq, kv_dtype=torch.float8_e4m3fn
    )


def test_decoder_with_an_8_bit_cache_holds_the_rounded_keys() -> None:
    full, small = _decoders(2, 96)
    prompt = torch.randint(0, 512, (2, 45), generator=torch.Generator().manual_seed(1))
    full.prefill(prompt)
    small.prefill(prompt)
    for t in range(3):
        full.step(prompt[:, t])
        small.step(prompt[:, t])
    a, c = full.caches[0], small.caches[0]  # the first layer's keys and values depend on the tokens alone
    for exact, rows, scale in ((a.k, c.k, c.k_scale), (a.v, c.v, c.v_scale)):
        per_row = scale.repeat_interleave(BLOCK, dim=2)[:, :, :96, None]
        held = rows.float() * per_row
        # one rounding: half a step of a 4-bit mantissa (2**-4 of the value) or of e4m3's least step, 2**-10 of the
        # scale; the block that fills row by row may be rounded again whenever its scale doubles, each time by half
        # as much as the scale then allows: together twice that. fp32 rotation order adds under 2**-20.
        limit = 2 * torch.maximum(exact.abs() * 2.0**-4, per_row * 2.0**-10) + 2.0**-20
        assert ((held - exact).abs()[:, :, :48] <= limit[:, :, :48]).all()
        assert (rows.float()[:, :, 48:] == 0).all()


def test_decoder_with_an_8_bit_cache_does_not_care_how_a_prompt_is_cut() -> None:
    _, whole = _decoders(1, 96)
    _, parts = _decoders(1, 96)
    prompt = torch.randint(0, 512, (1, 80), generator=torch.Generator().manual_seed(2))
    want = whole.prefill(prompt)
    for lo in (0, 32, 64):  # whole blocks: the scales are found from the same rows
        got = parts.prefill(prompt[:, lo : lo + 32])
    # the same cache bytes; the fp32 sums run over other shapes
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
    for a, c in zip(whole.caches, parts.caches, strict=True):
        assert (a.k.view(torch.uint8) == c.k.view(torch.uint8)).float().mean() > 0.99
    before = [c.k.clone() for c in parts.caches]
    parts.reset()
    again = parts.prefill(prompt)
    torch.testing.assert_close(again, want, rtol=1e-4, atol=1e-4)
    assert len(before) == len(parts.caches)


def test_decoder_refuses_other_cache_types_and_overflow() -> None:
    from priml_b200.inference import CacheState, Decoder, Fp8KVCache
    from priml_b200.models.presets import tiny_lm

    model = tiny_lm().make().eval()
    with pytest.raises(ValueError, match="kv_dtype"):
        Decoder(model, batch=1, max_seq=8, kv_dtype=torch.float16)
    dec = Decoder(model, batch=1, max_seq=8, kv_dtype=torch.float8_e4m3fn)
    dec.prefill(torch.zeros(1, 8, dtype=torch.long))
    with pytest.raises(ValueError, match="overflow"):
        dec.step(torch.zeros(1, dtype=torch.long))
    with pytest.raises(ValueError, match="positions"):
        Fp8KVCache.alloc(CacheState.create(1, 64), heads=1, channels_head=8, cos=torch.ones(63, 4), sin=torch.ones(63, 4))
    cache = dec.caches[0]
    factors = torch.ones(1, 1, 16)
    with pytest.raises(ValueError, match="cos_sin"):
        model.blocks[0].attn(torch.zeros(1, 1, 128), cache=cache, cos_sin=(factors, factors))
