"""8-bit cache kernels where they can go wrong: rows that see nothing, block scales far apart, values that are not
finite, outlying channels, long runs whose every block shows in the output, models that no kernel covers."""

from __future__ import annotations

import pytest
import torch
from torch import Tensor

from tests.cache8_cases import BLOCK, attend64, filled_cache

pytestmark = pytest.mark.gpu


def _status_clean() -> None:
    from priml_b200.ops import native

    torch.cuda.synchronize()
    assert int(native().read_status(True)) == 0


def _queries(b: int, s: int, h: int, d: int, seed: int) -> Tensor:
    return (torch.randn(b, s, h, d, generator=torch.Generator().manual_seed(seed)) * 0.125).bfloat16().cuda()


def _ints(values: list[int]) -> Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _limit(want: Tensor, spread: Tensor) -> Tensor:
    """How far a kernel's output may be from 64 bits: ``spread`` is the same attention over |V|.

    Each weight p is rounded to f16, half a step being 2**-11 of it, and the sum of p is not rounded with it: 2**-11 of
    sum p |V|. Scores of up to 2**7 are off by a few 2**-24 of their size, weights by less than 2**-15, numerator and
    sum alike: 2**-14 more. The rounding to bf16 is half a step of an 8-bit significand: 2**-8 of the result.
    """
    return want.abs() * 2.0**-8 + spread * (2.0**-11 + 2.0**-13) * (1 + 2.0**-8)


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


@pytest.mark.parametrize("s", [1, 5, 150])
@pytest.mark.parametrize("large", [7, 20, 40, 90])
@pytest.mark.parametrize("zero_first", [True, False])
def test_blocks_of_zeros_beside_large_values(s: int, large: int, zero_first: bool) -> None:
    """A block of zeros has the least scale, 2**-100; its keys count in the sum of the weights all the same."""
    from priml_b200 import ops

    b, h, hkv, t, d = 2, 8, 2, 700, 64
    k, ks = filled_cache(b, hkv, t, d, seed=11, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=12, device="cuda")
    q = _queries(b, s, h, d, seed=13)
    zero = (torch.arange(-(-t // BLOCK), device="cuda") % 3 == 1) ^ (torch.arange(-(-t // BLOCK), device="cuda") < 6)
    if not zero_first:
        zero = ~zero
    rows = zero.repeat_interleave(BLOCK)[:t]
    v.view(torch.uint8)[:, :, rows] = 0
    vs[:, :, zero], vs[:, :, ~zero] = 2.0**-100, vs[:, :, ~zero] * 2.0**large
    ends = [t, 400]
    out = ops.cache_attention(q, k, v, ks, vs, _ints(ends)).cpu().double()
    _status_clean()
    want = attend64(q, k, v, ks, vs, ends)
    spread = attend64(q, k, v.float().abs().to(v.dtype), ks, vs, ends)
    assert ((out - want).abs() <= _limit(want, spread)).all()


@pytest.mark.parametrize("b,s,h,hkv,t,d,ends,window", [
    (2, 1, 8, 2, 300, 128, [300, 270], None),
    (2, 1, 16, 1, 300, 64, [300, 17], 60),
    (2, 5, 4, 2, 300, 64, [300, 270], None),
    (2, 5, 8, 1, 300, 128, [290, 31], 40),  # a group of 8: the many-row form, both groups on the same rows
    (2, 150, 4, 2, 300, 64, [300, 270], None),
    (2, 150, 4, 2, 300, 128, [300, 100], 60),
    (1, 700, 2, 1, 4500, 128, [4444], None),  # runs that are cut and joined
])  # fmt: skip
def test_a_value_that_is_nan_stays_in_its_channel(b, s, h, hkv, t, d, ends, window) -> None:  # noqa: ANN001
    from priml_b200 import ops
    from priml_b200.ops import reference

    k, ks = filled_cache(b, hkv, t, d, seed=31, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=32, device="cuda")
    q = _queries(b, s, h, d, seed=33)
    g = torch.Generator().manual_seed(34)
    bits = v.view(torch.uint8)
    at = [(i, int(torch.randint(hkv, (), generator=g)), max(0, ends[i] - 1 - back), int(torch.randint(d, (), generator=g)))
          for i in range(b) for back in (0, 1, 7, s - 1, s + 20, 90)]  # fmt: skip
    for where in at:
        bits[where] = 0
    clean = ops.cache_attention(q, k, v, ks, vs, _ints(ends), window=window)
    for n, where in enumerate(at):
        bits[where] = 0x7F if n % 2 else 0xFF
    out = ops.cache_attention(q, k, v, ks, vs, _ints(ends), window=window)
    _status_clean()
    want = reference.cache_attention(
        *(x.cpu() for x in (q.float(), k, v, ks, vs, _ints(ends))), scale=d**-0.5, window=window
    ).isnan()
    assert torch.equal(out.cpu().isnan(), want) and want.any() and not want.all()
    assert torch.equal(out[~want.cuda()], clean[~want.cuda()])


@pytest.mark.parametrize("s", [1, 6, 150])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_scale_that_is_nan_reaches_the_queries_that_see_its_block(s: int, which: str) -> None:
    from priml_b200 import ops
    from priml_b200.ops import reference

    b, h, hkv, t, d = 2, 8, 2, 330, 64
    k, ks = filled_cache(b, hkv, t, d, seed=21, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=22, device="cuda")
    q, ends = _queries(b, s, h, d, seed=23), [330, 200]
    clean = ops.cache_attention(q, k, v, ks, vs, _ints(ends), window=40)
    scale = ks if which == "k" else vs
    scale[0, 1, (330 - s // 2) // BLOCK] = float("nan")
    scale[1, 0, 170 // BLOCK] = float("nan")
    out = ops.cache_attention(q, k, v, ks, vs, _ints(ends), window=40)
    _status_clean()
    want = reference.cache_attention(
        *(x.cpu() for x in (q.float(), k, v, ks, vs, _ints(ends))), scale=d**-0.5, window=40
    ).isnan()
    assert torch.equal(out.cpu().isnan(), want) and want.any() and not want.all()
    assert torch.equal(out[~want.cuda()], clean[~want.cuda()])


@pytest.mark.parametrize("s", [1, 6, 150])
@pytest.mark.parametrize("power", [0, 16, 22])
def test_an_outlying_query_channel_leaves_the_others_their_bits(s: int, power: int) -> None:
    """One channel of the queries is 2**power times the others and meets keys that are zero there."""
    from priml_b200 import ops

    b, h, hkv, t, d = 1, 4, 2, 300, 64
    k, ks = filled_cache(b, hkv, t, d, seed=41, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=42, device="cuda")
    k.view(torch.uint8)[..., 5] = 0
    q = _queries(b, s, h, d, seed=43) * 8  # scores of some tens: a relative 2**-8 of one would show
    plain = q.clone()
    q[..., 5] = 2.0**power
    plain[..., 5] = 0
    out = ops.cache_attention(q, k, v, ks, vs, _ints([t])).cpu().double()
    _status_clean()
    want = attend64(plain, k, v, ks, vs, [t])
    spread = attend64(plain, k, v.float().abs().to(v.dtype), ks, vs, [t])
    assert ((out - want).abs() <= _limit(want, spread)).all()


@pytest.mark.parametrize("s", [1, 6, 150])
@pytest.mark.parametrize("size", [-100, 60, 127])
def test_queries_of_any_finite_size(s: int, size: int) -> None:
    from priml_b200 import ops

    b, h, hkv, t, d = 1, 4, 2, 300, 64
    k, ks = filled_cache(b, hkv, t, d, seed=44, device="cuda")
    v, vs = filled_cache(b, hkv, t, d, seed=45, device="cuda")
    q = _queries(b, s, h, d, seed=46)
    base = ops.cache_attention(q, k, v, ks, vs, _ints([t]))
    far = (q.float() * 2.0**size).bfloat16()
    assert far.isfinite().all()
    out = ops.cache_attention(far, k, v, ks, vs, _ints([t]), scale=d**-0.5 * 2.0**-size)
    _status_clean()
    if size < 120:  # powers of two all along: the same bits
        assert torch.equal(out, base)
        return
    # scale * log2(e) is 2**-129.5, a subnormal fp32 number: half a step, 2**-150, is 2**-20 of it. Scores stay under 2**6,
    # so exponents are off by 2**-14, numerator and sum by 2**-14 of themselves; the roundings to bf16 may then be neighbours.
    size_v = (v.float().abs().amax((-1, -2)) * vs.amax(-1)).max()
    assert ((out.float() - base.float()).abs() <= base.float().abs() * 2.0**-7 + 2.0**-13 * size_v).all()


@pytest.mark.parametrize("head_dim,dtype", [(32, torch.bfloat16), (32, torch.float32), (64, torch.float32), (128, torch.float16)])
def test_decoder_with_an_8_bit_cache_captures_models_that_no_kernel_covers(head_dim: int, dtype: torch.dtype) -> None:
    from priml_b200.inference import Decoder
    from priml_b200.models.presets import dense_lm

    torch.manual_seed(0)
    cfg = dense_lm(vocab=512, d_model=128, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=head_dim, ffn_hidden=256,
                   rope_theta=1e4, norm_eps=1e-6, init_std=None)  # fmt: skip
    model = cfg.make().cuda().to(dtype).eval()
    prompt = torch.randint(0, 512, (3, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    kw = dict(batch=3, max_seq=96, kv_dtype=torch.float8_e4m3fn)
    graphed, eager = Decoder(model, **kw), Decoder(model, **kw, cuda_graph=False)
    kw = dict(max_new_tokens=40, temperature=0)
    assert torch.equal(graphed.generate(prompt, **kw), eager.generate(prompt, **kw))
    for a, c in zip(graphed.caches, eager.caches, strict=True):
        assert torch.equal(a.k.view(torch.uint8)[:, :, :72], c.k.view(torch.uint8)[:, :, :72])
        assert torch.equal(a.v_scale[:, :, :2], c.v_scale[:, :, :2])
    assert len(graphed._graphs) == 1


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 32), (torch.float32, 64)])
def test_the_torch_form_gives_the_same_bytes_on_both_devices(dtype: torch.dtype, d: int) -> None:
    from priml_b200 import ops

    b, s, hkv, t = 3, 40, 2, 100
    g = torch.Generator().manual_seed(61)
    x = (torch.randn(2, b, s, hkv, d, generator=g) * torch.exp2(torch.randint(-60, 61, (b, s, 1, 1), generator=g).float())).to(dtype)
    x[0, 0, 3, 1, 2], x[1, 2, 39, 0, 0] = float("nan"), float("inf")
    n = torch.tensor([0, 31, 70], dtype=torch.int32)
    held = []
    for device in ("cpu", "cuda"):
        k, ks = filled_cache(b, hkv, t, d, seed=62, device=device)
        v, vs = filled_cache(b, hkv, t, d, seed=63, device=device)
        ops.rotary_append(x[0].to(device), *x.to(device), k, v, ks, vs, n.to(device))
        held.append([z.cpu() for z in (k.float(), v.float(), ks, vs)])
    for a, c in zip(*held, strict=True):
        assert torch.equal(a.nan_to_num(1e9), c.nan_to_num(1e9))


def test_append_refuses_caches_that_share_a_part() -> None:
    """(Refused before anything is launched.)"""
    from priml_b200 import ops

    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    n = _ints([3, 4])
    from tests.test_cache8_edges_cpu import _halves

    with torch.device("cuda"):
        shared, apart = _halves()
    for case in shared:
        with pytest.raises(ValueError, match="of their own|overlap"):
            ops.rotary_append(q, x, x, *case, n)
    for case in apart:
        assert ops.rotary_append(q, x, x, *case, n) is q
    _status_clean()


def _telling_cache(b: int, hkv: int, t: int, d: int, seed: int) -> tuple[Tensor, Tensor]:
    """Values that are positive in one channel per block of 32 rows, ``block % d``, and zero elsewhere: an output channel
    is the sum of few blocks' parts, none of which can be lost unseen."""
    g = torch.Generator().manual_seed(seed)
    nb = -(-t // BLOCK)
    x = torch.zeros(b, hkv, nb, BLOCK, d)
    x[:, :, torch.arange(nb), :, torch.arange(nb) % d] = 1 + torch.rand(nb, b, hkv, BLOCK, generator=g)
    x *= torch.exp2(torch.randint(-1, 2, (b, hkv, nb, 1, 1), generator=g).float())
    scale = torch.exp2(torch.ceil(torch.log2(x.amax((-1, -2)) / 448)))
    rows = (x / scale[..., None, None]).to(torch.float8_e4m3fn).view(b, hkv, nb * BLOCK, d)
    return rows[:, :, :t].contiguous().cuda(), scale.cuda()


LONG = [  # B, s, H, Hkv, T, D, ends, window
    (1, 1, 8, 8, 9000, 64, [9000], None),
    (16, 1, 8, 8, 2100, 64, [2100] * 16, None),
    (4, 2, 32, 4, 12000, 128, [12000, 11999, 11990, 2], None),
    (1, 1, 16, 1, 60001, 128, [60001], None),  # one item over the whole grid
    (3, 5, 8, 1, 9001, 64, [9001, 5000, 33], None),  # many-row form, both groups on the same rows
    (1, 520, 2, 1, 3001, 128, [2999], None),
    (1, 150, 4, 2, 20000, 128, [19999], None),
    (2, 260, 2, 2, 6000, 64, [6000, 5500], 3000),
    (1, 2100, 2, 1, 2100, 128, [2100], None),  # a whole fresh prompt
    (2, 1300, 4, 2, 1300, 64, [1300, 1300], 100),
]


@pytest.mark.parametrize("b,s,h,hkv,t,d,ends,window", LONG)
def test_every_block_of_a_long_run_is_in_the_output(b, s, h, hkv, t, d, ends, window) -> None:  # noqa: ANN001
    from priml_b200 import ops

    k, ks = filled_cache(b, hkv, t, d, seed=51, device="cuda")
    v, vs = _telling_cache(b, hkv, t, d, seed=52)
    q = _queries(b, s, h, d, seed=53) * 0.25
    n = _ints(ends)
    out = ops.cache_attention(q, k, v, ks, vs, n, window=window)
    again = ops.cache_attention(q, k, v, ks, vs, n, window=window)
    _status_clean()
    assert torch.equal(out, again)  # sums in a fixed order
    want = attend64(q, k, v, ks, vs, ends, window=window)
    limit = _limit(want, want)  # V >= 0
    assert ((out.cpu().double() - want).abs() <= limit).all()
    # The same result without one block of keys is out of that limit, for every block of which a query sees half. (One
    # key of the 15 x 32 that share a channel in the longest case is 2**-9 of it, the limit 2**-8 + 2**-11 + 2**-13.)
    block = torch.arange(t) // BLOCK
    for i in range(b):
        for head in (0, h - 1):
            kv = head // (h // hkv)
            pos = ends[i] - 1
            lo = 0 if window is None else max(0, pos - window)
            kk = k[i, kv].cpu().double() * ks[i, kv].cpu().double()[block, None]
            vv = v[i, kv].cpu().double() * vs[i, kv].cpu().double()[block, None]
            p = (kk[lo : pos + 1] @ q[i, s - 1, head].cpu().double() * d**-0.5).softmax(-1)
            full = p @ vv[lo : pos + 1]
            torch.testing.assert_close(full, want[i, s - 1, head])
            seen = block[lo : pos + 1]
            blocks, rows = seen.unique(return_counts=True)
            for j in blocks[rows >= BLOCK // 2].tolist() if len(blocks) > 1 else []:
                keep = seen != j
                lost = p[keep] @ vv[lo : pos + 1][keep] / p[keep].sum()
                assert ((lost - full).abs() > 2 * limit[i, s - 1, head]).any(), (i, head, j)


def test_threads_that_call_first_together() -> None:
    """Several host threads, each on its own stream, in a process that has not called the operator before."""
    import subprocess
    import sys

    code = """
import threading
import torch
from priml_b200 import ops
from tests.cache8_cases import filled_cache

k, ks = filled_cache(2, 2, 500, 64, seed=1, device="cuda")
v, vs = filled_cache(2, 2, 500, 64, seed=2, device="cuda")
n = torch.tensor([500, 130], dtype=torch.int32, device="cuda")
q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
torch.cuda.synchronize()
outs = [None] * 6
gate = threading.Barrier(6)

def run(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        gate.wait()
        outs[i] = ops.cache_attention(q, k, v, ks, vs, n)
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=run, args=(i,)) for i in range(6)]
[t.start() for t in threads]
[t.join() for t in threads]
assert all(torch.equal(o, outs[0]) for o in outs) and outs[0].isfinite().all()
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]
