"""Pure-torch oracles for every hand-written kernel.

These are the semantics the CUDA kernels reproduce; tests compare the kernels
against them computed in fp32. They are also the CPU execution path (the
reference framework itself runs these ops through ATen:
``priml/model/norm.py:36-74``, ``priml/model/rope.py:348-387``,
``priml/model/attention.py:107-193``, ``priml/model/swiglu.py:190-213``,
``priml/baselines/nanochat/train_step.py:43-79``,
``priml/optimizers/fused_adamw.py:42-83``).
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch import Tensor


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    w = weight.to(x.dtype)
    return F.linear(x, w, None if bias is None else bias.to(x.dtype))


def rms_norm(x: Tensor, weight: Tensor | None, eps: float | None) -> Tensor:
    return F.rms_norm(x, (x.shape[-1],), weight, eps)


def rotate_half(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Half-split rotation in fp32, rounded once (HuggingFace convention)."""
    dtype = x.dtype
    x = x.float()
    half = x.shape[-1] // 2
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], dim=-1).to(dtype)


def rotate(x: Tensor, cos: Tensor, sin: Tensor, interleave: bool = False) -> Tensor:
    """Rotation of the first ``2 * cos.shape[-1]`` channels of ``[..., S, H, D]`` in fp32, rounded once.

    The pairs are channels ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with ``interleave``; the others are copied.
    """
    rot = 2 * cos.shape[-1]
    if rot > x.shape[-1]:
        raise ValueError(f"{rot} rotated channels do not fit {x.shape[-1]} channels.")
    turned, rest = x[..., :rot].float(), x[..., rot:]
    a, c = (turned[..., 0::2], turned[..., 1::2]) if interleave else turned.chunk(2, dim=-1)
    pair = (a * cos - c * sin, c * cos + a * sin)
    y = torch.stack(pair, dim=-1).flatten(-2) if interleave else torch.cat(pair, dim=-1)
    return torch.cat([y.to(x.dtype), rest], dim=-1) if rest.shape[-1] else y.to(x.dtype)


def attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    causal: bool = True,
    scale: float | None = None,
    window: int | None = None,
) -> Tensor:
    """``[B, S, H, D]`` x ``[B, T, Hkv, D]`` -> ``[B, S, H, Dv]``; grouped KV heads
    are shared by ``H // Hkv`` consecutive query heads. Causal masks are aligned
    bottom-right (query ``i`` sees keys ``<= T - S + i``); ``window`` limits the
    look-back to ``window`` keys (``key >= pos - window``)."""
    B, S, H, D = q.shape
    T, Hkv = k.shape[1], k.shape[2]
    g = H // Hkv
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    qf = q.float().transpose(1, 2)  # B H S D
    kf = k.float().transpose(1, 2).repeat_interleave(g, dim=1)
    vf = v.float().transpose(1, 2).repeat_interleave(g, dim=1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    if causal or window is not None:
        qi = torch.arange(S, device=q.device)[:, None] + (T - S)
        kj = torch.arange(T, device=q.device)[None, :]
        allowed = torch.ones(S, T, dtype=torch.bool, device=q.device)
        if causal:
            allowed &= kj <= qi
        if window is not None:
            allowed &= kj >= qi - window
        s = s.masked_fill(~allowed, float("-inf"))
    p = torch.softmax(s, dim=-1)
    p = torch.nan_to_num(p, nan=0.0)
    o = torch.matmul(p, vf)
    return o.transpose(1, 2).to(q.dtype)


def swiglu(gate_up: Tensor) -> Tensor:
    gate, up = gate_up.chunk(2, dim=-1)
    return F.silu(gate) * up


def decode_attention(
    q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, *, scale: float, window: int | None = None
) -> Tensor:
    """fp32 oracle of the decode kernel: ``[B, H, D]`` queries over ``[B, Hkv, T, D]`` caches."""
    b, h, _ = q.shape
    hkv, t = k_cache.shape[1], k_cache.shape[2]
    kf = k_cache.float().repeat_interleave(h // hkv, dim=1)
    vf = v_cache.float().repeat_interleave(h // hkv, dim=1)
    s = torch.einsum("bhd,bhtd->bht", q.float(), kf) * scale
    pos = torch.arange(t, device=q.device)
    n = lengths.to(device=q.device, dtype=torch.long).clamp(0, t)[:, None]
    ok = pos[None, :] < n
    if window is not None:
        ok &= pos[None, :] >= n - 1 - window
    s = s.masked_fill(~ok[:, None, :], float("-inf"))
    p = torch.nan_to_num(s.softmax(dim=-1), nan=0.0)  # an empty row gives zeros
    return torch.einsum("bht,bhtd->bhd", p, vf).to(q.dtype)


CACHE_BLOCK = 32
"""Cache rows of one head that share a scale."""


def cache_scale(amax: Tensor) -> Tensor:
    """The least power of two ``p`` in [2**-100, 2**120] with ``amax / p <= 448``, e4m3's largest value."""
    mant, exp = torch.frexp(amax.float())  # amax = mant * 2**exp, mant in [0.5, 1); 448 = 0.875 * 2**9
    exp = exp - 9 + (mant > 0.875).to(exp.dtype)
    exp = torch.where(amax > 0, exp, torch.full_like(exp, -100)).clamp(-100, 120)
    return torch.ldexp(torch.ones_like(mant), exp)


def _to_e4m3(x: Tensor) -> Tensor:
    return torch.where(x.isfinite(), x, torch.full_like(x, float("nan"))).to(torch.float8_e4m3fn)


def cache_append(x: Tensor, cache: Tensor, scale: Tensor, lengths: Tensor) -> None:
    """Quantise ``[B, s, Hkv, D]`` rows into rows ``lengths[b] + i`` of an 8-bit cache ``[B, Hkv, T, D]``.

    A block of 32 rows that held rows before keeps its scale unless the new rows need a larger one, in
    which case its old rows are requantised. Values that are not finite are stored as NaN and do not
    enter the scale. Rows at or past ``T`` are dropped; a negative length appends nothing. Nothing is
    read on the host, so that a CUDA graph can hold the call.
    """
    b, s, hkv, d = x.shape
    t = cache.shape[2]
    if x.numel() == 0 or t == 0:
        return
    n = (s + 2 * CACHE_BLOCK - 2) // CACHE_BLOCK  # blocks that s rows can touch
    start = lengths.to(device=x.device, dtype=torch.long)[:, None]
    inside = (start >= 0) & (start < t)
    first = torch.where(inside, start, 0) // CACHE_BLOCK
    at = torch.arange(b, device=x.device)[:, None]
    row = first * CACHE_BLOCK + torch.arange(n * CACHE_BLOCK, device=x.device)  # [B, n * 32]: the window's cache rows
    token = row - start
    new = inside & (token >= 0) & (token < s) & (row < t)
    touched = new.view(b, n, CACHE_BLOCK).any(-1)[:, None]  # [B, 1, n] blocks
    old = inside & (token < 0)

    rows = x[at, token.clamp(0, s - 1)].transpose(1, 2).float()  # [B, Hkv, n * 32, D]
    size = torch.where(rows.isfinite() & new[:, None, :, None], rows.abs(), 0.0).view(b, hkv, n, CACHE_BLOCK, d).amax((3, 4))
    block = first + torch.arange(n, device=x.device)
    block = block.clamp(max=scale.shape[2] - 1)
    held = scale[at, :, block].transpose(1, 2)  # [B, Hkv, n]
    keeps = old.view(b, n, CACHE_BLOCK).any(-1)[:, None]
    now = cache_scale(size)
    now = torch.where(touched, torch.where(keeps, torch.maximum(now, held), now), held)

    # Rows past the end stand for the last row, blocks for the last block: they write what those write.
    row = row.clamp(max=t - 1)
    bits = cache.view(torch.uint8)
    before = bits[at, :, row].transpose(1, 2).contiguous()
    ratio, per_row = (f.repeat_interleave(CACHE_BLOCK, dim=2)[..., None] for f in (held / now, now))
    value = torch.where(new[:, None, :, None], rows / per_row, before.view(cache.dtype).float() * ratio)
    changed = (new | old) & touched[:, 0].repeat_interleave(CACHE_BLOCK, dim=1)
    after = torch.where(changed[:, None, :, None], _to_e4m3(value).view(torch.uint8), before)
    bits[at, :, row] = after[at, :, row - first * CACHE_BLOCK]
    scale[at, :, block] = now[at, :, block - first]


def rotary_append(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    k_scale: Tensor,
    v_scale: Tensor,
    lengths: Tensor,
    cos: Tensor | None,
    sin: Tensor | None,
    interleave: bool,
) -> Tensor:
    """Oracle of :func:`priml_b200.ops.rotary_append`: the keys go to the cache from the fp32 rotation."""
    kf = k.float()
    if cos is not None and sin is not None:
        at = (lengths.long()[:, None] + torch.arange(q.shape[1], device=q.device)).clamp(0, cos.shape[0] - 1)
        c, n = cos.float()[at][:, :, None], sin.float()[at][:, :, None]
        q, kf = rotate(q, c, n, interleave), rotate(kf, c, n, interleave)
    cache_append(kf, k_cache, k_scale, lengths)
    cache_append(v.float(), v_cache, v_scale, lengths)
    return q


def cache_attention(
    q: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    k_scale: Tensor,
    v_scale: Tensor,
    lengths: Tensor,
    *,
    scale: float,
    window: int | None = None,
    offset: int = 0,
) -> Tensor:
    """fp32 oracle of attention over an 8-bit cache: ``[B, s, H, D]`` queries, the last ``s`` tokens of each sequence."""
    b, s, h, d = q.shape
    hkv, t = k_cache.shape[1], k_cache.shape[2]
    k, v = (
        c.float() * f.repeat_interleave(CACHE_BLOCK, dim=2)[:, :, :t, None] for c, f in ((k_cache, k_scale), (v_cache, v_scale))
    )
    n = (lengths.to(device=q.device, dtype=torch.long) + offset).clamp(0, t)
    pos = n[:, None] - s + torch.arange(s, device=q.device)
    key = torch.arange(t, device=q.device)
    ok = key <= pos[..., None]  # [B, s, T]
    if window is not None:
        ok &= key >= pos[..., None] - window
    # rows that no query sees may hold anything
    v = torch.where(ok.any(1)[:, None, :, None], v, torch.zeros_like(v))
    qf = q.float().reshape(b, s, hkv, h // hkv, d)
    z = torch.einsum("bskgd,bktd->bkgst", qf, k) * scale
    z = z.masked_fill(~ok[:, None, None], float("-inf"))
    p = torch.where(ok.any(-1)[:, None, None, :, None], z.softmax(dim=-1), torch.zeros_like(z))
    bad = v.isnan()
    o = torch.einsum("bkgst,bktd->bskgd", p, v.masked_fill(bad, 0.0))
    # a NaN reaches the queries that see its row, and no others
    o = o.masked_fill(torch.einsum("bst,bktd->bskd", ok.float(), bad.float())[:, :, :, None] > 0, float("nan"))
    return o.reshape(b, s, h, d).to(q.dtype)


def mla_decode(
    q: Tensor, c_kv: Tensor, k_pe: Tensor, *, scale: float, lengths: Tensor | None = None
) -> Tensor:
    """fp32 oracle of latent-space MLA decode: ``q [B, H, 576] = [q_abs | q_pe]`` over
    ``c_kv [B, T, 512]`` and ``k_pe [B, T, 64]``; returns the softmax-weighted latent rows ``[B, H, 512]``."""
    lat = c_kv.shape[-1]
    c = c_kv.float()
    s = (torch.einsum("bhl,btl->bht", q[..., :lat].float(), c)
         + torch.einsum("bhr,btr->bht", q[..., lat:].float(), k_pe.float())) * scale  # fmt: skip
    if lengths is not None:
        pos = torch.arange(c.shape[1], device=q.device)
        ok = pos[None, :] < lengths.to(device=q.device, dtype=torch.long)[:, None]
        s = s.masked_fill(~ok[:, None, :], float("-inf"))
    p = torch.nan_to_num(s.softmax(dim=-1), nan=0.0)
    return torch.einsum("bht,btl->bhl", p, c).to(q.dtype)


def cross_entropy(logits: Tensor, targets: Tensor, *, ignore_index: int = -100, softcap: float | None = None) -> Tensor:
    """Unreduced token cross-entropy computed in fp32."""
    lf = logits.float()
    if softcap is not None:
        lf = softcap * torch.tanh(lf / softcap)
    return F.cross_entropy(lf.reshape(-1, lf.shape[-1]), targets.reshape(-1), ignore_index=ignore_index, reduction="none").reshape(
        targets.shape
    )


def linear_cross_entropy(
    hidden: Tensor,
    weight: Tensor,
    targets: Tensor,
    *,
    ignore_index: int = -100,
    softcap: float | None = None,
) -> Tensor:
    logits = linear(hidden, weight)
    return cross_entropy(logits, targets, ignore_index=ignore_index, softcap=softcap)


def adamw_(
    params: list[Tensor],
    grads: list[Tensor],
    exp_avgs: list[Tensor],
    exp_avg_sqs: list[Tensor],
    *,
    step: int,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
) -> None:
    """AdamW in the FusedAdamW operation order (``priml/optimizers/fused_adamw.py:42-83``):
    ``p *= 1 - lr*wd``; ``m = lerp(m, g, 1-b1)``; ``v = lerp(v, g*g, 1-b2)``;
    ``p -= m / (sqrt(v / bias2) + eps) * (lr / bias1)`` -- all in fp32."""
    bias1 = 1.0 - beta1**step
    bias2 = 1.0 - beta2**step
    with torch.no_grad():
        for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs, strict=True):
            g32 = g.float()
            p32 = p if p.dtype == torch.float32 else p.float()
            m32 = m if m.dtype == torch.float32 else m.float()  # moments of narrow parameters update in fp32
            v32 = v if v.dtype == torch.float32 else v.float()
            p32.mul_(1.0 - lr * weight_decay)
            m32.lerp_(g32, 1.0 - beta1)
            v32.lerp_(g32.square(), 1.0 - beta2)
            denom = (v32 / bias2).sqrt() + eps
            p32.sub_(m32 / denom * (lr / bias1))
            for lo, hi in ((p, p32), (m, m32), (v, v32)):
                if hi.data_ptr() != lo.data_ptr():
                    lo.copy_(hi)


def grouped_swiglu_mlp(x_sorted: Tensor, up_w: Tensor, down_w: Tensor, offsets: Tensor) -> Tensor:
    """Rows ``offsets[e]:offsets[e+1]`` through expert ``e``:
    ``down_w[e] @ swiglu(up_w[e] @ x)``; ``up_w [E, 2H, C]``, ``down_w [E, C, H]``.
    Rows past ``offsets[E]`` (padding of a padded buffer) come out zero."""
    bounds = offsets.tolist()
    pieces = []
    for e in range(up_w.shape[0]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            pieces.append(linear(swiglu(linear(x_sorted[lo:hi], up_w[e])), down_w[e]))
    tail = x_sorted.shape[0] - bounds[-1]  # rows past the last segment (padded buffers)
    if tail > 0:
        pieces.append(x_sorted.new_zeros(tail, down_w.shape[1]))
    if not pieces:
        return x_sorted.new_zeros(0, down_w.shape[1])
    return torch.cat(pieces, dim=0)
