"""Builders shared by the 8-bit cache tests: filled caches and the operators in 64 bits, row by row."""

from __future__ import annotations

import math

import torch
from torch import Tensor

BLOCK = 32


def filled_cache(
    b: int, hkv: int, t: int, d: int, seed: int, device: str = "cpu", pad_heads: int = 0, spread: float = 1.0
) -> tuple[Tensor, Tensor]:
    """``[B, Hkv, T, D]`` e4m3 rows and their scales, sizes changing from block to block; ``pad_heads`` widens the
    head axis of the buffers, so that the batch stride is not the packed one."""
    g = torch.Generator().manual_seed(seed)
    nb = -(-t // BLOCK)
    x = torch.randn(b, hkv, nb, BLOCK, d, generator=g) * torch.exp2(
        torch.randint(-3, 4, (b, hkv, nb, 1, 1), generator=g).float() * spread
    )
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448)))
    rows = (x / scale[..., None, None]).to(torch.float8_e4m3fn).view(b, hkv, nb * BLOCK, d)[:, :, :t]
    buf = torch.zeros(b, hkv + pad_heads, t, d, dtype=torch.float8_e4m3fn)
    buf.view(torch.uint8)[:, :hkv] = rows.contiguous().view(torch.uint8)
    sbuf = torch.ones(b, hkv + pad_heads, nb)
    sbuf[:, :hkv] = scale
    return buf.to(device)[:, :hkv], sbuf.to(device)[:, :hkv]


def attend64(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    ks: Tensor,
    vs: Tensor,
    ends: list[int],
    scale: float | None = None,
    window: int | None = None,
) -> Tensor:
    """Attention of ``[B, s, H, D]`` queries, one sequence, query and head at a time, in 64 bits on the CPU."""
    q, k, v, ks, vs = (x.detach().cpu() for x in (q, k, v, ks, vs))
    b, s, h, d = q.shape
    hkv, t = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(b, s, h, d, dtype=torch.float64)
    block = torch.arange(t) // BLOCK
    for i in range(b):
        n = min(max(ends[i], 0), t)
        for hk in range(hkv):
            kk = k[i, hk, :n].double() * ks[i, hk].double()[block[:n], None]
            vv = v[i, hk, :n].double() * vs[i, hk].double()[block[:n], None]
            for j in range(s):
                pos = n - s + j
                lo = 0 if window is None else max(0, pos - window)
                if pos < 0:
                    continue
                heads = slice(hk * (h // hkv), (hk + 1) * (h // hkv))
                z = q[i, j, heads].double() @ kk[lo : pos + 1].T * scale
                out[i, j, heads] = z.softmax(-1) @ vv[lo : pos + 1]
    return out


def attention_tolerance(v: Tensor, vs: Tensor) -> float:
    """How far a kernel's output may be from 64 bits, in absolute terms.

    The weights p of a row sum to one; each is rounded to f16 (half a step: 2**-11 of it) and stands for a score
    that the fp32 products leave off by a few 2**-23 of its size (scores here stay under 2**6, so exp2 is off by
    under 2**-15); the sum of p is not rounded with them, so the output is off by at most
    (2**-11 + 2**-14) max|V|. Its rounding to bf16 adds 2**-9 of a value that is at most max|V| (half a step of an
    8-bit mantissa). Together less than 2**-8 max|V|.
    """
    biggest = (v.detach().cpu().float().abs().nan_to_num(0.0).amax((-1, -2)) * vs.detach().cpu().amax(-1)).max().item()
    return 2.0**-8 * biggest


def append64(x: Tensor, cache: Tensor, scale: Tensor, start: list[int]) -> tuple[Tensor, Tensor]:
    """The append's definition on ``[B, s, Hkv, D]`` rows in 64 bits: (values held, scales), of CPU copies."""
    x = x.detach().cpu().double()
    held, scale = cache.detach().cpu().double(), scale.detach().cpu().double().clone()
    t = held.shape[2]
    for b, n in enumerate(start):
        for hk in range(x.shape[2]):
            for blk in range(n // BLOCK, -(-min(n + x.shape[1], t) // BLOCK)):
                lo, hi = max(n, blk * BLOCK), min(n + x.shape[1], blk * BLOCK + BLOCK, t)
                rows = x[b, lo - n : hi - n, hk]
                size = rows[rows.isfinite()].abs().max().item() if rows.isfinite().any() else 0.0
                e = -100 if size == 0 else max(-100, math.ceil(math.log2(size / 448)))
                if size > 0 and size / 2.0 ** (e - 1) <= 448 and e > -100:  # log2's rounding next to a border
                    e -= 1
                if size > 0 and size / 2.0**e > 448:
                    e += 1
                now = 2.0**e
                if lo > blk * BLOCK:
                    now = max(now, scale[b, hk, blk].item())
                    old = held[b, hk, blk * BLOCK : lo] * (scale[b, hk, blk].item() / now)
                    held[b, hk, blk * BLOCK : lo] = old.float().to(torch.float8_e4m3fn).double()
                held[b, hk, lo:hi] = (
                    torch.where(rows.isfinite(), rows / now, torch.nan).float().to(torch.float8_e4m3fn).double()
                )
                scale[b, hk, blk] = now
    return held, scale
