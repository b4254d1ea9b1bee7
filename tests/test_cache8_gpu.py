"""8-bit cache kernels on the GPU against 64 bits.

Head dims, groups, lengths from none to full caches, chunks that end inside a block, windows, strided queries and
caches, rows that hold NaN where nobody looks, graph replay, other streams, and the calls that are refused.
"""

from __future__ import annotations

import pytest
import torch

from tests.cache8_cases import append64, attend64, attention_tolerance, filled_cache

pytestmark = pytest.mark.gpu


def _status_clean() -> None:
    from priml_b200.ops import native

    torch.cuda.synchronize()
    assert int(native().read_status(True)) == 0


CASES = [  # B, s, H, Hkv, T, D, ends (None: full), window
    (1, 1, 1, 1, 1, 64, None, None),
    (1, 1, 8, 1, 33, 128, [32], None),
    (3, 1, 4, 4, 70, 64, [0, 1, 70], None),
    (2, 1, 15, 3, 300, 128, [300, 129], None),  # a group of 5
    (2, 1, 12, 1, 200, 64, [31, 200], None),  # two row tiles
    (1, 1, 40, 2, 500, 128, None, None),  # a group of 20: two row groups
    (4, 1, 8, 2, 1000, 128, [1000, 64, 65, 999], 37),
    (2, 1, 4, 2, 260, 64, [260, 7], 0),
    (1, 1, 8, 8, 9000, 64, None, None),  # many splits
    (2, 3, 8, 2, 100, 64, [100, 2], None),  # a chunk longer than one cache
    (2, 4, 8, 2, 120, 128, [97, 33], 3),
    (1, 16, 4, 1, 90, 128, [90], None),
    (2, 33, 6, 2, 150, 64, [150, 40], None),
    (1, 40, 4, 2, 333, 128, [301], 50),
    (3, 130, 4, 2, 400, 64, [400, 131, 130], None),
    (1, 257, 2, 1, 700, 128, [690], None),
    (2, 65, 7, 1, 300, 128, [300, 66], 64),
    (16, 1, 8, 8, 2100, 64, None, None),  # long runs: the copies' ring wraps
    (4, 2, 32, 4, 12000, 128, [12000, 11999, 11990, 1], None),  # the same at 16 rows
    (1, 520, 2, 1, 3001, 128, [2999], None),  # several row tiles over many key tiles
]


@pytest.mark.parametrize("b,s,h,hkv,t,d,ends,window", CASES)
def test_attention_matches_64_bits(b, s, h, hkv, t, d, ends, window) -> None:  # noqa: ANN001
    from priml_b200 import ops

    ends = [t] * b if ends is None else ends
    k, ks = filled_cache(b, hkv, t, d, seed=b * 131 + t, device="cuda", pad_heads=1)
    v, vs = filled_cache(b, hkv, t, d, seed=b * 131 + t + 1, device="cuda", pad_heads=1)
    for i, n in enumerate(ends):  # rows behind the last token may hold anything
        k.view(torch.uint8)[i, :, n:] = 0x7F
        v.view(torch.uint8)[i, :, n:] = 0xFF
        ks[i, :, -(-n // 32) :] = float("nan")
        vs[i, :, -(-n // 32) :] = float("inf")
    g = torch.Generator().manual_seed(s)
    # scores of a few units: keys reach 2**3 * 4, so queries of about 2**-3
    q = (torch.randn(b, s, h + 2, d, generator=g) * 0.125).bfloat16().cuda()[:, :, 1 : h + 1]
    lengths = torch.tensor(ends, dtype=torch.int32, device="cuda")
    out = ops.cache_attention(q, k, v, ks, vs, lengths, window=window)
    want = attend64(q, k, v, ks, vs, ends, window=window)
    _status_clean()
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    err = (out.cpu().double() - want).abs().max().item()
    live = vs.cpu().nan_to_num(0, posinf=0)
    assert err <= attention_tolerance(v, live), err
    for i, n in enumerate(ends):
        if n < s:
            assert out[i, : s - n].abs().max().item() == 0
    if s == 1:
        one = ops.cache_attention(q[:, 0], k, v, ks, vs, lengths - 1, window=window, offset=1)
        assert torch.equal(one, out[:, 0])


@pytest.mark.parametrize("s", [1, 6, 150])
def test_attention_scale_sizes_and_large_scores(s: int) -> None:
    """Queries and caches far from one: the row and block factors carry the size."""
    from priml_b200 import ops

    b, h, hkv, t, d = 1, 4, 2, 400, 64
    k, ks = filled_cache(b, hkv, t, d, seed=5, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=6, device="cuda")
    q = (torch.randn(b, s, h, d, generator=torch.Generator().manual_seed(7)) * 0.125).bfloat16().cuda()
    n = torch.tensor([t], dtype=torch.int32, device="cuda")
    base = ops.cache_attention(q, k, v, ks, vs, n).float()
    big = ops.cache_attention(q * 2.0**40, k, v, ks * 2.0**-30, vs * 2.0**20, n, scale=d**-0.5 * 2.0**-10).float()
    # The many-row form adds log2 of V's scale to the exponents: the shift by 20 moves arguments of size up to 2**6
    # by roundings of 2**-19 at most, the weights by 2**-18 of themselves and, numerator and sum, the output by
    # 2**-17 max|V|; where that crosses a rounding border of bf16 the results are neighbours, 2**-7 apart at most.
    limit = base.abs() * 2.0**-7 + 2.0**-17 * attention_tolerance(v, vs) * 2.0**8
    assert ((big * 2.0**-20 - base).abs() <= limit).all()
    # one key outweighs all others: the output is its value row
    sharp = ops.cache_attention(q * 64, k, v, ks, vs, n)
    want = attend64(q * 64, k, v, ks, vs, [t])
    # scores up to 2**12 in log2 units are exact to 2**-24 of their size: exp2 is off by up to 2**-11
    assert (sharp.cpu().double() - want).abs().max().item() <= 2 * attention_tolerance(v, vs)


@pytest.mark.parametrize("s", [1, 5, 150])
def test_nan_reaches_only_the_queries_that_see_it(s: int) -> None:
    from priml_b200 import ops

    b, h, hkv, t, d = 2, 8, 2, 300, 128
    k, ks = filled_cache(b, hkv, t, d, seed=8, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=9, device="cuda")
    q = (torch.randn(b, s, h, d, generator=torch.Generator().manual_seed(s)) * 0.125).bfloat16().cuda()
    n = torch.tensor([250, 280], dtype=torch.int32, device="cuda")
    clean = ops.cache_attention(q, k, v, ks, vs, n, window=60)
    v.view(torch.uint8)[0, 1, 249, 5] = 0x7F  # the newest value row of one head: its last query only
    v.view(torch.uint8)[1, 0, 280 - s - 61, 7] = 0xFF  # one row before any query's window
    k.view(torch.uint8)[1, 0, 280 - s - 61, 7] = 0xFF
    out = ops.cache_attention(q, k, v, ks, vs, n, window=60)
    _status_clean()
    hit = torch.zeros(b, s, h, dtype=torch.bool, device="cuda")
    hit[0, s - 1, 4:] = True
    assert torch.equal(out.isnan().any(-1), hit)
    assert torch.equal(out[~hit], clean[~hit])


def test_infinite_and_nan_queries_stay_in_their_rows() -> None:
    from priml_b200 import ops

    k, ks = filled_cache(1, 1, 100, 64, seed=1, device="cuda")
    v, vs = filled_cache(1, 1, 100, 64, seed=2, device="cuda")
    n = torch.tensor([100], dtype=torch.int32, device="cuda")
    for s in (2, 140):
        q = (torch.randn(1, s, 4, 64, generator=torch.Generator().manual_seed(3)) * 0.1).bfloat16().cuda()
        clean = ops.cache_attention(q, k, v, ks, vs, n)
        q[0, s - 1, 0, 0], q[0, s - 1, 2, 5] = float("nan"), float("inf")
        out = ops.cache_attention(q, k, v, ks, vs, n)
        keep = torch.ones(s, 4, dtype=torch.bool, device="cuda")
        keep[s - 1, 0] = keep[s - 1, 2] = False
        assert torch.equal(out[0][keep], clean[0][keep]) and out[0, s - 1, 0].isnan().all() and out[0, s - 1, 2].isnan().all()


def test_attention_of_more_sequences_than_one_launch_takes() -> None:
    from priml_b200 import ops

    b = 1030
    k, ks = filled_cache(b, 1, 40, 64, seed=3, device="cuda")
    v, vs = filled_cache(b, 1, 40, 64, seed=4, device="cuda")
    ends = [(7 * i) % 41 for i in range(b)]
    q = (torch.randn(b, 1, 2, 64, generator=torch.Generator().manual_seed(1)) * 0.125).bfloat16().cuda()
    out = ops.cache_attention(q, k, v, ks, vs, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    want = attend64(q, k, v, ks, vs, ends)
    assert (out.cpu().double() - want).abs().max().item() <= attention_tolerance(v, vs)


@pytest.mark.parametrize("s", [1, 4, 30])
def test_scales_of_blocks_that_no_query_sees_may_hold_anything(s: int) -> None:
    from priml_b200 import ops

    b, h, hkv, t, d, window = 2, 4, 1, 500, 64, 50
    k, ks = filled_cache(b, hkv, t, d, seed=1, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=2, device="cuda")
    q = (torch.randn(b, s, h, d, generator=torch.Generator().manual_seed(s)) * 0.125).bfloat16().cuda()
    ends = [430, 300]
    n = torch.tensor(ends, dtype=torch.int32, device="cuda")
    clean = ops.cache_attention(q, k, v, ks, vs, n, window=window)
    for i, end in enumerate(ends):
        lo, hi = (end - s - window) // 32, -(-end // 32)
        for scale in (ks, vs):
            scale[i, :, :lo], scale[i, :, hi:] = float("nan"), float("inf")
        for rows in (k, v):
            rows.view(torch.uint8)[i, :, : end - s - window] = 0x7F
    assert torch.equal(ops.cache_attention(q, k, v, ks, vs, n, window=window), clean)


def test_many_row_launches_are_split_by_sequences_and_by_tokens() -> None:
    from priml_b200 import ops

    b, s = 1100, 20  # more row tiles than one launch lists
    k, ks = filled_cache(b, 1, 40, 64, seed=3, device="cuda")
    v, vs = filled_cache(b, 1, 40, 64, seed=4, device="cuda")
    ends = [20 + (7 * i) % 21 for i in range(b)]
    q = (torch.randn(b, s, 1, 64, generator=torch.Generator().manual_seed(1)) * 0.125).bfloat16().cuda()
    out = ops.cache_attention(q, k, v, ks, vs, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    pick = [0, 1, 1022, 1023, 1024, 1025, 1099]
    want = attend64(q[pick], k[pick], v[pick], ks[pick], vs[pick], [ends[i] for i in pick])
    assert (out[pick].cpu().double() - want).abs().max().item() <= attention_tolerance(v, vs)

    s, h, t = 600, 512, 640  # 512 query heads on one KV head: 1200 row tiles of one sequence
    k, ks = filled_cache(1, 1, t, 64, seed=5, device="cuda")
    v, vs = filled_cache(1, 1, t, 64, seed=6, device="cuda")
    q = (torch.randn(1, s, h, 64, generator=torch.Generator().manual_seed(2)) * 0.125).bfloat16().cuda()
    out = ops.cache_attention(q, k, v, ks, vs, torch.tensor([630], dtype=torch.int32, device="cuda"))
    for i in (0, 1, 511, 512, 513, 599):  # query i alone stands at 30 + i
        want = attend64(q[:, i : i + 1], k, v, ks, vs, [31 + i])
        assert (out[:, i : i + 1].cpu().double() - want).abs().max().item() <= attention_tolerance(v, vs)
    _status_clean()


def test_long_cache_past_32_bit_offsets() -> None:
    """Byte offsets past 2**31 inside one cache: 2 sequences x 2 heads x 2**23 + 40 rows of 128."""
    from priml_b200 import ops

    b, hkv, t, d = 2, 2, (1 << 23) + 40, 128
    k = torch.full((b, hkv, t, d), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # all ones
    v = torch.zeros((b, hkv, t, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ks = torch.ones(b, hkv, -(-t // 32), device="cuda")
    vs = torch.ones_like(ks)
    q = torch.zeros(b, 1, 4, d, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(b, 3, hkv, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    start = torch.tensor([t - 3, t - 36], dtype=torch.int32, device="cuda")
    ops.rotary_append(torch.zeros(b, 3, 4, d, dtype=torch.bfloat16, device="cuda"), x, x, k, v, ks, vs, start)
    out = ops.cache_attention(q, k, v, ks, vs, start, offset=3, window=2)  # equal weights on the last three rows
    at = start.long()[:, None] + torch.arange(3, device="cuda")
    i = torch.arange(b, device="cuda")[:, None]
    rows = v[i, :, at].float() * vs[i, :, at // 32][..., None]
    torch.testing.assert_close(out[:, 0].view(b, hkv, 2, d).float(), rows.mean(1)[:, :, None].expand(-1, -1, 2, -1), rtol=2**-7, atol=2**-7)
    full = ops.cache_attention(q, k, v, ks, vs, start, offset=3)
    assert full.isfinite().all()
    _status_clean()


APPENDS = [  # B, s, H, Hkv, T, D, rot, interleave, starts
    (1, 1, 2, 1, 1, 64, 64, False, [0]),
    (3, 1, 8, 2, 100, 128, 128, False, [0, 31, 99]),
    (2, 1, 4, 4, 64, 64, 32, True, [32, 33]),
    (2, 31, 6, 3, 100, 128, 42, False, [1, 33]),
    (2, 77, 5, 1, 130, 64, 0, False, [53, 20]),
    (1, 300, 4, 2, 290, 128, 64, True, [9]),  # runs past the cache's end
    (3, 5, 4, 2, 64, 128, 6, True, [64, 70, 60]),  # behind the end: nothing, nothing, four rows
    (2, 64, 4, 2, 200, 64, 62, False, [32, 17]),
]


@pytest.mark.parametrize("b,s,h,hkv,t,d,rot,interleave,starts", APPENDS)
def test_append_matches_the_definition(b, s, h, hkv, t, d, rot, interleave, starts) -> None:  # noqa: ANN001
    from priml_b200 import ops
    from priml_b200.ops import reference

    g = torch.Generator().manual_seed(t + s)
    qkv = torch.randn(b, s, h + 2 * hkv, d, generator=g) * torch.exp2(torch.randint(-4, 5, (b, s, 1, 1), generator=g).float())
    q, x, y = qkv.bfloat16().cuda().split([h, hkv, hkv], dim=2)
    cos = sin = None
    if rot:
        ang = torch.arange(t, dtype=torch.float64)[:, None] * 0.5 ** torch.arange(rot // 2)
        cos, sin = ang.cos().float().cuda(), ang.sin().float().cuda()
    k, ks = filled_cache(b, hkv, t, d, seed=1, device="cuda", pad_heads=1)
    v, vs = filled_cache(b, hkv, t, d, seed=2, device="cuda", pad_heads=1)
    lengths = torch.tensor(starts, dtype=torch.int32, device="cuda")
    copies = [z.clone() for z in (k, v, ks, vs)]
    want_q = reference.rotary_append(q, x, y, *copies, lengths, cos, sin, interleave)
    out = ops.rotary_append(q, x, y, k, v, ks, vs, lengths, cos=cos, sin=sin, interleave=interleave)
    # the same fp32 operations, rounded at the same places: equal to the last bit
    assert torch.equal(out, want_q)
    for got, want in zip((k, v, ks, vs), copies, strict=True):
        assert torch.equal(got.float(), want.float())
    if not rot:
        v0, vs0 = filled_cache(b, hkv, t, d, seed=2)
        held, scale = append64(y, v0, vs0, starts)
        assert torch.equal(v.cpu().double(), held) and torch.equal(vs.cpu().double(), scale)


def test_append_token_by_token_and_at_once_agree_on_scales() -> None:
    from priml_b200 import ops

    g = torch.Generator().manual_seed(3)
    x = (torch.randn(2, 40, 2, 64, generator=g) * torch.exp2(torch.arange(40)[:, None, None] / 4)).bfloat16().cuda()
    caches = [[z for pair in (filled_cache(2, 2, 64, 64, seed=1, device="cuda") for _ in range(2)) for z in pair] for _ in range(2)]
    q = torch.zeros(2, 40, 4, 64, dtype=torch.bfloat16, device="cuda")
    k, ks, v, vs = caches[0]
    ops.rotary_append(q, x, x, k, v, ks, vs, torch.zeros(2, dtype=torch.int32, device="cuda"))
    k1, ks1, v1, vs1 = caches[1]
    for i in range(40):
        ops.rotary_append(q[:, :1], x[:, i : i + 1], x[:, i : i + 1], k1, v1, ks1, vs1, torch.full((2,), i, dtype=torch.int32, device="cuda"))
    assert torch.equal(ks[:, :, :2], ks1[:, :, :2]) and torch.equal(vs[:, :, :2], vs1[:, :, :2])
    a = k[:, :, :40].float() * ks.repeat_interleave(32, 2)[:, :, :40, None]
    c = k1[:, :, :40].float() * ks1.repeat_interleave(32, 2)[:, :, :40, None]
    # each requantisation rounds once more, by half a step of 2**-4 or of the least step 2**-10 of the scale; at most
    # ten of them, each at a scale twice the last
    step = ks.repeat_interleave(32, 2)[:, :, :40, None] * 2.0**-9
    assert ((a - c).abs() <= torch.maximum(a.abs() * 2.0**-3, 2 * step)).all()


def test_append_stores_values_that_are_not_finite_as_nan() -> None:
    from priml_b200 import ops

    k, ks = filled_cache(1, 1, 32, 64, seed=1, device="cuda")
    v, vs = k.clone(), ks.clone()
    x = torch.full((1, 1, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    x[..., 0], x[..., 1], x[..., 2] = float("inf"), -float("inf"), float("nan")
    ops.rotary_append(x, x, x, k, v, ks, vs, torch.zeros(1, dtype=torch.int32, device="cuda"))
    row = k[0, 0, 0].float() * ks[0, 0, 0]
    assert row[:3].isnan().all() and (row[3:] == 3.0).all() and ks[0, 0, 0].item() == 2.0**-7


@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,s,h,hk,d,rot,per_seq", [(2, 7, 3, 1, 64, 64, True), (1, 1, 1, 1, 2, 2, False), (3, 5, 4, 2, 96, 24, True), (2, 9, 2, 2, 80, 42, False), (1, 130, 17, 1, 128, 32, True), (2, 3, 2, 1, 10, 6, True)])
def test_rotary_and_its_gradient_match_torch(b, s, h, hk, d, rot, per_seq, dtype, interleave) -> None:  # noqa: ANN001
    from priml_b200 import ops
    from priml_b200.ops import reference

    g = torch.Generator().manual_seed(d + s)
    wide = torch.randn(b, s, h, d + 6, generator=g).to(dtype).cuda()
    q = wide[..., 6:].requires_grad_()  # a slice: rows that are not 16-byte aligned
    k = torch.randn(b, s, hk, d, generator=g).to(dtype).cuda().requires_grad_()
    ang = torch.randn((b, s, 1, rot // 2) if per_seq else (s, 1, rot // 2), generator=g).cuda()
    out = ops.rotary(q, k, ang.cos(), ang.sin(), interleave=interleave)
    want = reference.rotate(q, ang.cos(), ang.sin(), interleave), reference.rotate(k, ang.cos(), ang.sin(), interleave)
    gq, gk = torch.randn(b, s, h, d, generator=g).to(dtype).cuda(), torch.randn(b, s, hk, d, generator=g).to(dtype).cuda()
    got = torch.autograd.grad(out, (q, k), (gq, gk))
    ref = torch.autograd.grad(want, (q, k), (gq, gk))
    for a, c in zip((*out, *got), (*want, *ref), strict=True):
        assert a.dtype == dtype and torch.equal(a, c)


@pytest.mark.parametrize("shape", [(1, 6, 1, 8), (6, 4, 8), (2, 6, 4, 8)])  # one table as a batch, factors per head
def test_rotary_broadcasts_its_factors(shape: tuple) -> None:
    from priml_b200 import ops
    from priml_b200.models.rope import RoPE
    from priml_b200.ops import reference

    q, k = torch.randn(2, 6, 4, 24, device="cuda"), torch.randn(2, 6, 4, 24, device="cuda")
    ang = torch.randn(shape, device="cuda")
    got = ops.rotary(q, k, ang.cos(), ang.sin(), interleave=True)
    assert torch.equal(got[0], reference.rotate(q, ang.cos(), ang.sin(), True))
    assert torch.equal(RoPE.rotate(q, k, ang.cos(), ang.sin(), True)[1], reference.rotate(k, ang.cos(), ang.sin(), True))
    learned = ang.cos().requires_grad_()  # factors with a gradient take the torch operations
    assert torch.autograd.grad(ops.rotary(q, k, learned, ang.sin(), interleave=True)[0].sum(), learned)[0].shape == shape


def test_rotary_second_derivative_and_one_sided_gradients() -> None:
    from priml_b200 import ops

    q = torch.randn(2, 3, 2, 8, device="cuda", requires_grad=True)
    k = torch.randn(2, 3, 1, 8, device="cuda")
    ang = torch.randn(2, 3, 1, 2, device="cuda")
    qo, ko = ops.rotary(q, k, ang.cos(), ang.sin(), interleave=True)
    (dq,) = torch.autograd.grad((qo * qo).sum() / 2, q, create_graph=True)
    torch.testing.assert_close(dq, q, rtol=1e-5, atol=1e-6)  # a rotation keeps the square: the gradient is q itself
    (ddq,) = torch.autograd.grad(dq.sum(), q)
    torch.testing.assert_close(ddq, torch.ones_like(q), rtol=1e-5, atol=1e-6)


def test_run_of_the_operators_captured_on_another_stream() -> None:
    """Append and attention in one graph, twice captured, replayed as lengths and inputs change."""
    from priml_b200 import ops

    b, h, hkv, t, d = 3, 8, 2, 200, 64
    ang = torch.arange(t, device="cuda")[:, None] * 0.5 ** torch.arange(d // 2, device="cuda")
    cos, sin = ang.cos(), ang.sin()

    def fresh() -> list[torch.Tensor]:
        return [*filled_cache(b, hkv, t, d, seed=1, device="cuda"), *filled_cache(b, hkv, t, d, seed=2, device="cuda")]

    def step(qkv: torch.Tensor, lengths: torch.Tensor, c: list[torch.Tensor]) -> torch.Tensor:
        q, k, v = qkv.split([h, hkv, hkv], dim=2)
        q = ops.rotary_append(q, k, v, c[0], c[2], c[1], c[3], lengths, cos=cos, sin=sin)
        return ops.cache_attention(q, c[0], c[2], c[1], c[3], lengths, offset=1)

    eager, graphed = fresh(), fresh()
    qkv = torch.randn(b, 1, h + 2 * hkv, d, device="cuda").bfloat16()
    lengths = torch.tensor([0, 31, 150], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(qkv, lengths, fresh())
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                o = step(qkv, lengths, graphed)
            graphs.append((gr, o))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)).bfloat16())
        want = step(qkv, lengths, eager)
        gr, o = graphs[i % 2]
        gr.replay()
        assert torch.equal(o, want)
        lengths.add_(1)
    for a, c in zip(eager, graphed, strict=True):
        assert torch.equal(a.float(), c.float())
    _status_clean()


def test_refusals_on_the_device() -> None:
    from priml_b200 import ops

    k, ks = filled_cache(2, 2, 64, 64, seed=1, device="cuda")
    v, vs = filled_cache(2, 2, 64, 64, seed=2, device="cuda")
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="device"):
        ops.cache_attention(q, k, v, ks, vs, n.cpu())
    with pytest.raises(ValueError, match="device"):
        ops.cache_attention(q, k.cpu(), v, ks, vs, n)
    with pytest.raises(ValueError, match="contiguous"):  # rows with a stride of their own
        wide = torch.zeros(2, 2, 64, 128, device="cuda").to(torch.float8_e4m3fn)
        ops.cache_attention(q, wide[..., :64], v, ks, vs, n)
    with pytest.raises(ValueError, match="aligned"):
        flat = torch.zeros(2 * 2 * 64 * 64 + 8, dtype=torch.uint8, device="cuda")[8:].view(torch.float8_e4m3fn)
        ops.cache_attention(q, flat.view(2, 2, 64, 64), v, ks, vs, n)
    with pytest.raises(ValueError, match="overlap"):  # one cache for both sequences
        ops.rotary_append(q, x, x, k[:1].expand(2, -1, -1, -1), v, ks, vs, n)
    with pytest.raises(ValueError, match="overlap"):
        ops.rotary_append(q, x, x, k, v, ks, vs[:, :1].expand(-1, 2, -1), n)
    with pytest.raises(ValueError, match="of their own"):
        ops.rotary_append(q, x, x, k, k, ks, vs, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cache_attention(q.detach().requires_grad_(), k, v, ks, vs, n)
    with pytest.raises(ValueError):
        ops.rotary_append(q, x, x, k, v, ks, vs, n, cos=torch.ones(4, 33, device="cuda"), sin=torch.ones(4, 33, device="cuda"))
    assert ops.cache_attention(q, k[:1].expand(2, -1, -1, -1), v, ks, vs, n).shape == q.shape  # reading one is fine


@pytest.mark.parametrize("head_dim", [64, 128])
def test_decoder_with_an_8_bit_cache_graph_equals_eager(head_dim: int) -> None:
    from priml_b200.inference import Decoder
    from priml_b200.models.presets import dense_lm

    torch.manual_seed(0)
    cfg = dense_lm(vocab=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=head_dim, ffn_hidden=512,
                   rope_theta=1e4, norm_eps=1e-6, init_std=None)  # fmt: skip
    model = cfg.make().cuda().to(torch.bfloat16).eval()
    prompt = torch.randint(0, 512, (4, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    kw = dict(batch=4, max_seq=128, kv_dtype=torch.float8_e4m3fn)
    graphed, eager = Decoder(model, **kw), Decoder(model, **kw, cuda_graph=False)
    assert torch.equal(
        graphed.generate(prompt, max_new_tokens=40, temperature=0), eager.generate(prompt, max_new_tokens=40, temperature=0)
    )
    for a, c in zip(graphed.caches, eager.caches, strict=True):
        assert torch.equal(a.k.float()[:, :, :72], c.k.float()[:, :, :72]) and torch.equal(a.v_scale, c.v_scale)
    exact = Decoder(model, batch=4, max_seq=128, cuda_graph=False)
    exact.prefill(prompt)
    eager.reset()
    eager.prefill(prompt)
    k, c = exact.caches[0].k[:, :, :33].float(), eager.caches[0]
    scale = c.k_scale.repeat_interleave(32, dim=2)[:, :, :33, None]
    # the bf16 cache's keys are rounded by 2**-9 of themselves, the 8-bit ones by 2**-4 or by 2**-10 of the scale
    limit = torch.maximum(k.abs() * (2.0**-4 + 2.0**-8), scale * 2.0**-10 + k.abs() * 2.0**-8) + 2.0**-20
    assert ((c.k.float()[:, :, :33] * scale - k).abs() <= limit).all()
    _status_clean()
