"""Measured operators: rotary embedding, 8-bit cache append, and attention over the 8-bit cache.

Four kinds of case, each one call (or one forward and backward) that a user's program makes:

``rotary``  rotation of queries and keys, half-split or interleaved pairs, all or the first
            ``rot`` channels of a head, one table for the batch or positions per sequence;
            forward and backward (a training step's use).
``append``  a step's or a prompt chunk's queries rotated, its keys rotated, its keys and values
            quantised to e4m3 with one power-of-two scale per 32 tokens and head, and written to
            the cache behind each sequence's tokens.
``decode``  one query token per sequence over that cache.
``chunk``   a chunk of query tokens per sequence (the last ones in the cache) over it, causal.

``own`` is set by whoever measures: false runs the plain form, true the framework's kernels.
"""

import math
import random

import torch

own = False

BLOCK = 32  # tokens that share a scale
CHANNELS_REST = 128  # channels beside the rotated ones where a rotated slice of wider heads is taken


def listed():
    return [
        # rotary: the rotated slice of latent attention's heads in training (16 heads, one shared key head)
        dict(name="rotary latent train", op="rotary", b=4, s=4096, h=16, hk=1, d=64, rot=64, inter=True, per_seq=False,
             sliced=True, dtype="bf16"),  # fmt: skip
        # a quarter of each head rotated, sequences at positions of their own
        dict(name="rotary partial train", op="rotary", b=8, s=2048, h=32, hk=8, d=128, rot=32, inter=False, per_seq=True,
             sliced=False, dtype="bf16"),  # fmt: skip
        # a short odd batch in 32 bits, where latency counts
        dict(name="rotary odd fp32", op="rotary", b=3, s=77, h=5, hk=1, d=80, rot=42, inter=False, per_seq=True,
             sliced=False, dtype="fp32"),  # fmt: skip
        # append: one token of each of 64 sequences (8 key heads of 128)
        dict(name="append token", op="append", b=64, s=1, h=32, hk=8, d=128, t=1024, rot=128, inter=False, ragged=1),
        # a prompt chunk behind a partly filled cache
        dict(name="append chunk", op="append", b=4, s=2048, h=32, hk=8, d=128, t=4096, rot=128, inter=False, ragged=2),
        # an odd chunk of narrow heads, half of each rotated in interleaved pairs
        dict(name="append odd", op="append", b=5, s=77, h=12, hk=4, d=64, t=333, rot=32, inter=True, ragged=3),
        # decode: one short sequence of narrow heads: latency
        dict(name="decode one", op="decode", b=1, s=1, h=32, hk=8, d=64, t=1000, window=-1, ragged=0),
        # a full batch of long sequences: bandwidth
        dict(name="decode full", op="decode", b=64, s=1, h=32, hk=8, d=128, t=8192, window=-1, ragged=0),
        # few sequences of very different lengths up to a long one, one key head for 16 query heads
        dict(name="decode ragged", op="decode", b=9, s=1, h=16, hk=1, d=128, t=100001, window=-1, ragged=4),
        # chunk: a handful of tokens checked at once behind long caches
        dict(name="chunk few", op="chunk", b=8, s=5, h=32, hk=8, d=128, t=16384, window=-1, ragged=5),
        # a prompt's chunk over a long cache: the largest
        dict(name="chunk long", op="chunk", b=1, s=2048, h=32, hk=8, d=128, t=32768, window=-1, ragged=0),
        # whole odd prompts of narrow heads, with a sliding window
        dict(name="chunk window", op="chunk", b=4, s=1111, h=32, hk=8, d=64, t=2500, window=512, ragged=6),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode", "chunk", "chunk"])
    if op == "rotary":
        d = rng.choice([32, 64, 80, 96, 128, 192, 256])
        hk = rng.choice([1, 2, 4, 5, 8])
        case = dict(op=op, b=_log(rng, 1, 16), s=_log(rng, 1, 8192), h=hk * rng.choice([1, 2, 3, 4, 8]), hk=hk, d=d,
                    rot=rng.choice([d, d // 2, d // 4, 2 * rng.randint(1, d // 2)]), inter=rng.random() < 0.5,
                    per_seq=rng.random() < 0.5, sliced=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))  # fmt: skip
        while case["b"] > 1 and case["b"] * case["s"] * (case["h"] + hk) * d > 1 << 27:
            case["b"] = max(1, case["b"] // 2)
        while case["s"] > 1 and case["b"] * case["s"] * (case["h"] + hk) * d > 1 << 27:
            case["s"] = max(1, case["s"] // 2)
        case["rot"] += case["rot"] % 2
        return case
    d = rng.choice([64, 128])
    hk = rng.choice([1, 2, 3, 4, 8])
    h = hk * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    seed = rng.randint(1, 10**6)
    if op == "append":
        b = _log(rng, 1, 128)
        s = _log(rng, 1, max(1, min(4096, 16384 // b)))
        t = s + _log(rng, 1, 4096)
        while t > s and b * hk * t * d > 1 << 26:
            t = max(s, t // 2)
        return dict(op=op, b=b, s=s, h=h, hk=hk, d=d, t=t, rot=rng.choice([0, d, d // 2, 2 * rng.randint(1, d // 2)]),
                    inter=rng.random() < 0.4, ragged=seed)  # fmt: skip
    s = 1 if op == "decode" else _log(rng, 2, 2048)
    t = max(s, _log(rng, 2, 131072))
    b = _log(rng, 1, 128)
    while b > 1 and (b * hk * t * d > 1 << 28 or b * h * s * t * (d + 32) > 1 << 37):
        b //= 2
    while t > s and (b * hk * t * d > 1 << 28 or b * h * s * t * (d + 32) > 1 << 37):
        t = max(s, t // 2)
    return dict(op=op, b=b, s=s, h=h, hk=hk, d=d, t=t, window=rng.choice([-1, -1, _log(rng, 1, 4096)]),
                ragged=rng.choice([0, seed]))  # fmt: skip


def _ends(case):
    """Tokens in the cache after the call, for each sequence: full caches, or lengths of their own."""
    b, s, t = case["b"], case["s"], case["t"]
    if not case["ragged"]:
        return [t] * b
    rng = random.Random(case["ragged"])
    ends = [min(t, s + round((t - s) * rng.random() ** 2)) for _ in range(b)]
    ends[rng.randrange(b)] = t
    return ends


def _pairs(case):
    """(query, key) pairs that the masks leave, and key rows that some query sees, of one head over all sequences."""
    pairs = rows = 0
    for n in _ends(case):
        first, w = n - case["s"], case["window"]
        if w < 0:
            pairs += sum(range(first + 1, n + 1))
            rows += n
        else:
            pairs += sum(min(p, w) + 1 for p in range(first, n))
            rows += n - max(0, first - w)
    return pairs, rows


def work(case):
    b, s, h, hk, d = (case[n] for n in ("b", "s", "h", "hk", "d"))
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        values = b * s * (h + hk) * d
        table = (b if case["per_seq"] else 1) * s * case["rot"] * 4
        return {"bytes": 4 * values * size + 2 * table, "flops": 6 * b * s * (h + hk) * case["rot"]}
    if case["op"] == "append":
        blocks = b * hk * 2 * ((s + BLOCK - 1) // BLOCK)
        table = s * case["rot"] * 4
        return {"bytes": b * s * (2 * h * d * 2 + 2 * hk * d * 3) + 4 * blocks + table + 4 * b,
                "flops": b * s * (3 * (h + hk) * case["rot"] + 4 * hk * d)}  # fmt: skip
    pairs, rows = _pairs(case)
    return {"bytes": hk * rows * 2 * (d + 4 / BLOCK) + 2 * b * s * h * d * 2 + 4 * b, "flops": 4 * d * h * pairs}


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _angles(positions, rot, base=5e5):
    """cos and sin of ``positions * base ** (-2 i / rot)``; far positions need the angle in 64 bits."""
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=positions.device) / max(rot, 1))
    ang = positions.double()[..., None] * freq
    return ang.cos().float(), ang.sin().float()


def _power_of_two(amax):
    """The smallest power of two ``p`` with ``amax / p <= 448`` (448 = 1.75 * 2**8), at least 2**-100."""
    mant, exp = torch.frexp(amax)  # amax = mant * 2**exp with mant in [0.5, 1)
    exp = exp - 9 + (mant > 0.875).to(exp.dtype)
    exp = torch.where(amax > 0, exp, torch.full_like(exp, -100)).clamp(-100, 120)
    return torch.ldexp(torch.ones_like(amax), exp)


def _filled(shape, gen, spread):
    """A quantised cache ``[B, Hkv, T, D]`` of normal values, channels of unequal size: (e4m3 values, scales)."""
    b, hk, t, d = shape
    nb = (t + BLOCK - 1) // BLOCK
    data = torch.empty(b, hk, nb * BLOCK, d, dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(b, hk, nb, dtype=torch.float32, device="cuda")
    size = 1 + spread * torch.rand(hk, 1, 1, d, generator=gen, device="cuda")
    for i in range(b):
        x = torch.randn(hk, nb, BLOCK, d, generator=gen, device="cuda") * size
        p = _power_of_two(x.abs().amax((-1, -2)))
        scale[i] = p
        data[i] = (x / p[..., None, None]).to(torch.float8_e4m3fn).view(hk, nb * BLOCK, d)
    return data[:, :, :t].contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    b, s, h, hk, d = (case[n] for n in ("b", "s", "h", "hk", "d"))

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    if case["op"] == "rotary":
        dtype = _DTYPES[case["dtype"]]
        rest = CHANNELS_REST if case["sliced"] else 0
        q = normal(b, s, h, rest + d, dtype=dtype)[..., rest:]
        k = normal(b, s, hk, d, dtype=dtype)
        pos = torch.arange(s, device="cuda")
        if case["per_seq"]:
            pos = pos + torch.randint(0, 100000, (b, 1), generator=gen, device="cuda")
        cos, sin = _angles(pos, case["rot"])
        return dict(case=case, q=q.requires_grad_(), k=k.requires_grad_(), gq=normal(b, s, h, d, dtype=dtype),
                    gk=normal(b, s, hk, d, dtype=dtype), cos=cos[..., None, :], sin=sin[..., None, :])  # fmt: skip
    t = case["t"]
    ends = torch.tensor(_ends(case), dtype=torch.int32, device="cuda")
    state = dict(case=case, q=normal(b, s, h, d))
    state["k_cache"], state["k_scale"] = _filled((b, hk, t, d), gen, 2.0)
    state["v_cache"], state["v_scale"] = _filled((b, hk, t, d), gen, 0.5)
    if case["op"] == "append":
        state["lengths"] = ends - s
        # one fused projection's output: queries, keys and values are slices of it
        qkv = normal(b, s, h + 2 * hk, d)
        state["q"], state["k"], state["v"] = qkv.split([h, hk, hk], dim=2)
        state["cos"] = state["sin"] = None
        if case["rot"]:
            state["cos"], state["sin"] = _angles(torch.arange(t, device="cuda"), case["rot"])
        return state
    state["lengths"] = ends
    if case["op"] == "decode":
        state["q"] = state["q"][:, 0].contiguous()
    state["window"] = None if case["window"] < 0 else case["window"]
    return state


# --------------------------------------------------------------------------- plain forms
def _rotated(x, cos, sin, inter):
    """``x`` (fp32) with its first ``2 * cos.shape[-1]`` channels rotated pair by pair."""
    rot = 2 * cos.shape[-1]
    r = x[..., :rot]
    if inter:
        a, c = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - c * sin, c * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, c = r[..., : rot // 2], r[..., rot // 2 :]
        y = torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _append(x, cache, scale, lengths):
    """Quantise ``[B, s, Hkv, D]`` fp32 rows into rows ``lengths[b] + i`` of the cache, in place."""
    b, s, hk, d = x.shape
    t = cache.shape[2]
    nb = (s + 2 * BLOCK - 2) // BLOCK  # blocks that a chunk can touch
    first = lengths.long() // BLOCK
    row = first[:, None] * BLOCK + torch.arange(nb * BLOCK, device=x.device)  # [B, nb * BLOCK] cache rows
    token = row - lengths[:, None]
    new = (token >= 0) & (token < s) & (row < t)
    old = (token < 0) & (row < t)
    at = torch.arange(b, device=x.device)[:, None]
    rows = x[at, token.clamp(0, s - 1)].transpose(1, 2)  # [B, Hkv, rows, D]
    block = first[:, None] + torch.arange(nb, device=x.device)
    has_new = new.view(b, nb, BLOCK).any(-1)[:, None]
    has_old = old.view(b, nb, BLOCK).any(-1)[:, None]
    amax = rows.abs().masked_fill(~new[:, None, :, None], 0).view(b, hk, nb, BLOCK, d).amax((-1, -2))
    bc = block.clamp(max=scale.shape[2] - 1)
    before = scale[at, :, bc].transpose(1, 2)  # [B, Hkv, nb]
    after = torch.where(has_old, torch.maximum(before, _power_of_two(amax)), _power_of_two(amax))
    after = torch.where(has_new, after, before)
    rc = row.clamp(max=t - 1)
    held = cache[at, :, rc].transpose(1, 2).float().view(b, hk, nb, BLOCK, d) * (before / after)[..., None, None]
    put = rows.reshape(b, hk, nb, BLOCK, d) / after[..., None, None]
    value = torch.where(new.view(b, 1, nb, BLOCK, 1), put, held).to(cache.dtype).view(b, hk, nb * BLOCK, d)
    touched = (new | old) & has_new[:, 0].repeat_interleave(BLOCK, dim=1)
    bi, ri = touched.nonzero(as_tuple=True)
    cache.view(torch.uint8)[bi, :, row[bi, ri]] = value.view(torch.uint8)[bi, :, ri]
    bi, ni = has_new[:, 0].nonzero(as_tuple=True)
    scale[bi, :, block[bi, ni]] = after[bi, :, ni]


def _seen(lengths, s, t, window, device):
    """[B, s, T]: which cache rows each query sees."""
    pos = lengths.long()[:, None] - s + torch.arange(s, device=device)
    key = torch.arange(t, device=device)
    ok = key <= pos[..., None]
    if window is not None:
        ok &= key >= pos[..., None] - window
    return ok


def _attend(q, k_cache, v_cache, k_scale, v_scale, lengths, window):
    b, s, h, d = q.shape
    hk, t = k_cache.shape[1], k_cache.shape[2]
    g = h // hk
    k = k_cache.float() * k_scale.repeat_interleave(BLOCK, dim=2)[:, :, :t, None]
    v = v_cache.float() * v_scale.repeat_interleave(BLOCK, dim=2)[:, :, :t, None]
    x = q.float().view(b, s, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * s, d)
    z = (x @ k.transpose(-1, -2)).view(b, hk, g, s, t) * d**-0.5
    z.masked_fill_(~_seen(lengths, s, t, window, q.device)[:, None, None], float("-inf"))
    z = (z - z.amax(-1, keepdim=True)).exp_()
    o = (z.view(b, hk, g * s, t) @ v).view(b, hk, g, s, d) / z.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(b, s, h, d).to(q.dtype)


def _plain(state):
    case = state["case"]
    q = state["q"]
    if case["op"] == "rotary":
        k, cos, sin, inter = state["k"], state["cos"], state["sin"], case["inter"]
        with torch.no_grad():
            out = [_rotated(x.float(), cos, sin, inter).to(x.dtype) for x in (q, k)]
            # the rotation is orthogonal up to its factors: the gradient turns the other way
            grad = [_rotated(x.float(), cos, -sin, inter).to(x.dtype) for x in (state["gq"], state["gk"])]
        return dict(q=out[0], k=out[1], dq=grad[0], dk=grad[1])
    if case["op"] == "append":
        qf, kf, vf = q.float(), state["k"].float(), state["v"].float()
        if state["cos"] is not None:
            pos = (state["lengths"].long()[:, None] + torch.arange(case["s"], device=q.device))
            pos = pos.clamp(max=state["cos"].shape[0] - 1)
            cos, sin = state["cos"][pos][:, :, None], state["sin"][pos][:, :, None]
            qf, kf = _rotated(qf, cos, sin, case["inter"]), _rotated(kf, cos, sin, case["inter"])
        _append(kf, state["k_cache"], state["k_scale"], state["lengths"])
        _append(vf, state["v_cache"], state["v_scale"], state["lengths"])
        return dict(q=qf.to(q.dtype), **{n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")})
    q4 = q[:, None] if case["op"] == "decode" else q
    out = _attend(q4, state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"], state["lengths"], state["window"])
    return out[:, 0] if case["op"] == "decode" else out


def run(state):
    if not own:
        return _plain(state)
    from priml_b200 import ops

    case = state["case"]
    if case["op"] == "rotary":
        q, k = ops.rotary(state["q"], state["k"], state["cos"], state["sin"], interleave=case["inter"])
        dq, dk = torch.autograd.grad([q, k], [state["q"], state["k"]], [state["gq"], state["gk"]])
        return dict(q=q, k=k, dq=dq, dk=dk)
    cache = [state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")]
    if case["op"] == "append":
        q = ops.rotary_append(state["q"], state["k"], state["v"], *cache, state["lengths"], cos=state["cos"],
                              sin=state["sin"], interleave=case["inter"])  # fmt: skip
        return dict(q=q, **{n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")})
    return ops.cache_attention(state["q"], *cache, state["lengths"], window=state["window"])


# --------------------------------------------------------------------------- 64 bits, from the definitions
def _turn64(x, angle_cos, angle_sin, inter, sign=1.0):
    """Pair (a, b) as the complex number a + ib times cos + i sin."""
    r = 2 * angle_cos.shape[-1]
    part = x[..., :r].double()
    pair = part.unflatten(-1, (-1, 2)) if inter else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.complex(pair[..., 0], pair[..., 1]) * torch.complex(angle_cos.double(), sign * angle_sin.double())
    pair = torch.view_as_real(z)
    part = pair.flatten(-2) if inter else pair.transpose(-1, -2).flatten(-2)
    return torch.cat([part, x[..., r:].double()], dim=-1)


def _append64(x, data, scale, start):
    """The definition, sequence by sequence and block by block: (values, scales) after the append."""
    data, scale = data.double(), scale.double()
    s, t = x.shape[1], data.shape[2]
    for b, n in enumerate(start.tolist()):
        for blk in range(n // BLOCK, (min(n + s, t) + BLOCK - 1) // BLOCK):
            lo, hi = max(n, blk * BLOCK), min(n + s, (blk + 1) * BLOCK, t)
            rows = x[b, lo - n : hi - n].transpose(0, 1)  # [Hkv, rows, D]
            amax = rows.abs().amax((1, 2))
            need = torch.exp2(torch.ceil(torch.log2(amax.clamp_min(1e-300) / 448)).clamp(-100, 120))
            if lo > blk * BLOCK:
                held = scale[b, :, blk].clone()
                need = torch.maximum(need, held)
                before = data[b, :, blk * BLOCK : lo]
                data[b, :, blk * BLOCK : lo] = (before * (held / need)[:, None, None]).float().to(torch.float8_e4m3fn).double()
            data[b, :, lo:hi] = (rows / need[:, None, None]).float().to(torch.float8_e4m3fn).double()
            scale[b, :, blk] = need
    return data, scale


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        q = state["q"]
        if case["op"] == "rotary":
            out = {}
            for n, g in (("q", "gq"), ("k", "gk")):
                out[n] = _turn64(state[n], state["cos"], state["sin"], case["inter"])
                out["d" + n] = _turn64(state[g], state["cos"], state["sin"], case["inter"], -1.0)
            return out
        lengths = state["lengths"].tolist()
        if case["op"] == "append":
            k, v, q = state["k"].double(), state["v"].double(), q.double()
            if state["cos"] is not None:
                at = torch.stack([torch.arange(n, n + case["s"], device=q.device) for n in lengths]).clamp_max(case["t"] - 1)
                c, w = state["cos"][at].unsqueeze(2), state["sin"][at].unsqueeze(2)
                q, k = _turn64(q, c, w, case["inter"]), _turn64(k, c, w, case["inter"])
            out = {"q": q}
            for n, x in (("k", k), ("v", v)):
                out[n + "_cache"], out[n + "_scale"] = _append64(x, state[n + "_cache"], state[n + "_scale"], state["lengths"])
            return out
        q = q.double()
        q = q.unsqueeze(1) if case["op"] == "decode" else q
        s, h, hk, d = case["s"], case["h"], case["hk"], case["d"]
        out = torch.zeros_like(q)
        for b, n in enumerate(lengths):
            lo = 0 if case["window"] < 0 else max(0, n - s - case["window"])
            key = torch.arange(lo, n, device=q.device)
            pos = torch.arange(n - s, n, device=q.device)[:, None]
            hide = (key > pos) if case["window"] < 0 else (key > pos) | (key < pos - case["window"])
            for i in range(hk):
                k = state["k_cache"][b, i, lo:n].double() * state["k_scale"][b, i, key // BLOCK].double()[:, None]
                v = state["v_cache"][b, i, lo:n].double() * state["v_scale"][b, i, key // BLOCK].double()[:, None]
                heads = slice(i * (h // hk), (i + 1) * (h // hk))
                z = torch.einsum("shd,td->hst", q[b, :, heads], k) / math.sqrt(d)
                p = torch.softmax(z.masked_fill(hide, -math.inf), dim=-1)
                out[b, :, heads] = torch.einsum("hst,td->shd", p, v)
        return out[:, 0] if case["op"] == "decode" else out
