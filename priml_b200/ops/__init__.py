"""Hot ops: hand-written sm_100a kernels on CUDA, pure-torch oracles elsewhere.

Every public op here dispatches on the device of its inputs:

* CUDA tensors run the in-tree extension ``priml_b200.ops._C`` (tcgen05/TMA
  GEMMs, attention, fused norm/rope/CE/optimizer kernels). When the extension
  is missing on a CUDA device the op raises -- there is no silent fallback.
* CPU tensors (and ``PRIML_B200_REFERENCE=1``) run :mod:`priml_b200.ops.reference`.
"""

from __future__ import annotations

import os

import torch
from torch import Tensor

from priml_b200.ops import reference
from priml_b200.ops._loader import native, native_available

__all__ = [
    "CACHE_BLOCK",
    "adamw_",
    "add_rms_norm",
    "attention",
    "cache_attention",
    "cross_entropy",
    "decode_attention",
    "grouped_swiglu_experts",
    "grouped_swiglu_mlp",
    "mla_decode",
    "linear",
    "linear_cross_entropy",
    "linear_swiglu",
    "native",
    "native_available",
    "reference",
    "reference_forced",
    "rms_norm",
    "rotary",
    "rotary_append",
    "swiglu",
    "swiglu_mlp",
    "use_native",
]


def use_native(*tensors: Tensor | None) -> bool:
    """True when these tensors should take the CUDA kernel path."""
    if os.environ.get("PRIML_B200_REFERENCE", "0") == "1":
        return False
    if any(t is not None and type(t).__name__ == "DTensor" for t in tensors):
        return False  # DTensor dispatch (tensor parallel on the decomposed path)
    return any(t is not None and t.is_cuda for t in tensors)


def reference_forced() -> bool:
    """True when ``PRIML_B200_REFERENCE=1`` pins every op to the torch oracle."""
    return os.environ.get("PRIML_B200_REFERENCE", "0") == "1"


def _compute_dtype(x: Tensor) -> torch.dtype:
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda")
    return x.dtype


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """``x @ weight.T (+ bias)``; weight ``[N, K]`` in its master dtype."""
    if use_native(x, weight) and _compute_dtype(x) == torch.bfloat16:
        from priml_b200.ops import functional

        return functional.linear(x, weight, bias)
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        return torch.nn.functional.linear(x, weight, bias)
    return reference.linear(x, weight, bias)


def rms_norm(x: Tensor, weight: Tensor | None, eps: float | None) -> Tensor:
    if use_native(x) and _compute_dtype(x) in (torch.bfloat16, torch.float32):
        from priml_b200.ops import functional

        return functional.rms_norm(x, weight, eps)
    return reference.rms_norm(x, weight, eps)


def add_rms_norm(x: Tensor, d: Tensor | None, weight: Tensor | None, eps: float | None) -> tuple[Tensor, Tensor]:
    """Residual add fused into RMSNorm: ``h = x + d`` (``x`` when ``d`` is None) and ``rmsnorm(h)``."""
    fusable = (
        x.shape[-1] % 8 == 0
        and x.dtype in (torch.bfloat16, torch.float32)
        and (d is None or (d.dtype in (torch.bfloat16, torch.float32) and d.shape == x.shape))
    )
    if fusable and use_native(x, d) and _compute_dtype(x) in (torch.bfloat16, torch.float32):
        from priml_b200.ops import functional

        return functional.add_rms_norm(x, d, weight, eps)
    h = x if d is None else x + d
    return h, reference.rms_norm(h, weight, eps)


def rotary(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, *, interleave: bool = False) -> tuple[Tensor, Tensor]:
    """RoPE of ``[B, S, H, D]`` q and ``[B, S, Hk, D]`` k by fp32 half-width factors.

    ``cos`` and ``sin`` are ``[S, 1, R/2]`` (one table), ``[B, S, 1, R/2]`` (positions per sequence) or
    have a head axis of their own; the first ``R`` channels of a head are rotated, the others copied.
    The pairs are channels ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with ``interleave``. The rotation is
    computed in fp32 and rounded once. On CUDA q and k take one kernel (bf16, fp16, fp32), and its
    transpose in the backward; odd head widths and factors that need a gradient take the torch operations,
    and so do calls under ``torch.func`` transforms, forward-mode AD, ``torch.compile``, tracing and fake tensors.
    """
    if use_native(q):
        from priml_b200.ops import functional

        if not interleave and q.dtype == torch.bfloat16 and cos.ndim == 3 and cos.shape[-1] * 2 == q.shape[-1] and cos.shape[-2] == 1:
            return functional.rotary(q, k, cos, sin)
        if functional.rotary_any_supported(q, k, cos, sin) and not functional.traced(q, k, cos, sin):
            return native().rotary(q, k, cos, sin, interleave)
    return reference.rotate(q, cos, sin, interleave), reference.rotate(k, cos, sin, interleave)


def attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    causal: bool = True,
    scale: float | None = None,
    window: int | None = None,
) -> Tensor:
    """Flash attention over ``[B, S, H, D]`` with native GQA (no K/V expansion)."""
    if use_native(q):
        from priml_b200.ops import functional

        if functional.attention_supported(q, k, v):
            return functional.attention(q, k, v, causal=causal, scale=scale, window=window)
    return reference.attention(q, k, v, causal=causal, scale=scale, window=window)


def linear_swiglu(x: Tensor, up_weight: Tensor) -> Tensor:
    """``silu(x @ Wg^T) * (x @ Wu^T)`` for ``up_weight = [Wg; Wu]`` (``[2H, C]``)."""
    if use_native(x) and _compute_dtype(x) == torch.bfloat16 and up_weight.shape[0] % 16 == 0 and x.shape[-1] % 8 == 0:
        from priml_b200.ops import functional

        return functional.linear_swiglu(x, up_weight)
    return swiglu(linear(x, up_weight))


def swiglu_mlp(x: Tensor, up_weight: Tensor, down_weight: Tensor) -> Tensor:
    """``down(silu(x Wg^T) * (x Wu^T))`` for ``up_weight = [Wg; Wu]`` ([2H, C]) and ``down_weight`` [C_out, H]."""
    if (
        use_native(x)
        and _compute_dtype(x) == torch.bfloat16
        and up_weight.shape[0] % 16 == 0
        and x.shape[-1] % 8 == 0
        and down_weight.shape[0] % 8 == 0
    ):
        from priml_b200.ops import functional

        return functional.swiglu_mlp(x, up_weight, down_weight)
    return linear(swiglu(linear(x, up_weight)), down_weight)


def swiglu(gate_up: Tensor) -> Tensor:
    if use_native(gate_up) and gate_up.dtype == torch.bfloat16:
        from priml_b200.ops import functional

        return functional.swiglu(gate_up)
    return reference.swiglu(gate_up)


def mla_decode(q: Tensor, c_kv: Tensor, k_pe: Tensor, *, scale: float, lengths: Tensor | None = None) -> Tensor:
    """Latent-space multi-head latent attention for one query token per sequence.

    ``q`` is ``[B, H, 576]``: the absorbed query ``q_nope @ W_UK`` (512) followed by the
    rotary query (64); ``c_kv [B, T, 512]`` and ``k_pe [B, T, 64]`` are the cached latent
    rows and shared rotary keys (any row / sequence strides with contiguous channels).
    Returns ``softmax(scale * q . [c_kv | k_pe]) @ c_kv`` per head, ``[B, H, 512]``; keys
    at or past ``lengths[b]`` are hidden. On CUDA (bf16) this is the tcgen05 kernel of
    ``ops/csrc/mla_decode.cu``.
    """
    if (
        use_native(q)
        and q.dtype == torch.bfloat16
        and c_kv.dtype == torch.bfloat16
        and k_pe.dtype == torch.bfloat16
        and q.shape[-1] == 576
        and c_kv.shape[-1] == 512
        and k_pe.shape[-1] == 64
        and c_kv.stride(-1) == 1
        and k_pe.stride(-1) == 1
        and all(st % 8 == 0 for st in (*c_kv.stride()[:-1], *k_pe.stride()[:-1]))
    ):
        return native().mla_decode(q.contiguous(), c_kv, k_pe, lengths, float(scale))
    return reference.mla_decode(q, c_kv, k_pe, scale=scale, lengths=lengths)


def decode_attention(
    q: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    lengths: Tensor,
    *,
    scale: float | None = None,
    window: int | None = None,
) -> Tensor:
    """One query token per sequence against a KV cache with per-sequence lengths.

    ``q`` is ``[B, H, D]``; the caches are ``[B, Hkv, T, D]`` whose first
    ``lengths[b]`` rows are visible to sequence ``b`` (the query's own key
    included); query head ``h`` reads KV head ``h // (H / Hkv)``. ``window``
    hides keys more than ``window`` positions behind the query. The lengths stay
    on the device, so a decode step that calls this needs no host sync and can be
    captured in a CUDA graph. Returns ``[B, H, D]``.
    """
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if (
        use_native(q)
        and q.dtype == torch.bfloat16
        and k_cache.dtype == torch.bfloat16
        and q.shape[-1] in (64, 128)
        and v_cache.shape[-1] == q.shape[-1]
    ):
        return native().decode_attn(
            q.contiguous(), k_cache, v_cache, lengths.to(torch.int32).contiguous(), float(scale),
            -1 if window is None else int(window),
        )  # fmt: skip
    return reference.decode_attention(q, k_cache, v_cache, lengths, scale=float(scale), window=window)


CACHE_BLOCK = reference.CACHE_BLOCK


def _check_cache(q: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor, v_scale: Tensor, lengths: Tensor) -> None:
    """Refuse caches that do not belong together, on any device."""
    b, d = q.shape[0], q.shape[-1]
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[0] != b or k_cache.shape[-1] != d:
        raise ValueError(f"caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} do not fit queries {tuple(q.shape)}.")
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError(f"an 8-bit cache holds float8_e4m3fn, not {k_cache.dtype} and {v_cache.dtype}.")
    want = (*k_cache.shape[:2], -(-k_cache.shape[2] // CACHE_BLOCK))
    for name, f in (("k", k_scale), ("v", v_scale)):
        if tuple(f.shape) != want or f.dtype != torch.float32:
            raise ValueError(f"{name} scales must be fp32 {want}, got {f.dtype} {tuple(f.shape)}.")
    if tuple(lengths.shape) != (b,) or lengths.is_floating_point():
        raise ValueError(f"lengths must be {b} integers, got {lengths.dtype} {tuple(lengths.shape)}.")
    if any(x.device != q.device for x in (k_cache, v_cache, k_scale, v_scale, lengths)):
        raise ValueError("the caches, their scales and the lengths must be on the queries' device.")


def _overlap(*tensors: Tensor) -> bool:
    """Whether two (sequence, head) planes of these tensors of one shape share memory; rows within a plane are packed."""
    x = tensors[0]
    if not x.numel():
        return False
    size, plane = x.element_size(), x[0, 0].numel() * x.element_size()
    if all(t.is_contiguous() for t in tensors):  # what most caches are: no need to look at every plane
        starts = sorted(t.data_ptr() for t in tensors)
        return any(b - a < x.numel() * size for a, b in zip(starts, starts[1:], strict=False))
    starts = sorted(
        t.data_ptr() + size * (i * t.stride(0) + j * t.stride(1))
        for t in tensors
        for i in range(t.shape[0])
        for j in range(t.shape[1])
    )
    return any(b - a < plane for a, b in zip(starts, starts[1:], strict=False))


def rotary_append(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    k_scale: Tensor,
    v_scale: Tensor,
    lengths: Tensor,
    *,
    cos: Tensor | None = None,
    sin: Tensor | None = None,
    interleave: bool = False,
) -> Tensor:
    """Rotate ``s`` new tokens per sequence and append their keys and values to 8-bit caches, in place.

    ``q`` is ``[B, s, H, D]``, ``k`` and ``v`` ``[B, s, Hkv, D]``; token ``i`` of sequence ``b`` takes
    cache row and position ``lengths[b] + i`` (int32, on the device; not changed here). ``cos`` and
    ``sin`` are tables ``[positions, R/2]`` that are read at those positions (the last row past their
    end); q and k are rotated as :func:`rotary` does it. Without them nothing is rotated.

    The caches are ``float8_e4m3fn`` ``[B, Hkv, T, D]``; ``k_scale`` / ``v_scale`` (fp32
    ``[B, Hkv, ceil(T / 32)]``) hold one power of two per 32 rows and head, the least one with which the
    rows stay within e4m3's range: a row stands for ``row * scale``. Appending to a block that holds rows
    already keeps its scale or, for larger values, raises it and requantises those rows. Values that are
    not finite are stored as NaN. Tokens past ``T`` are not stored. Returns the rotated q, or ``q`` itself
    where nothing is rotated.

    On CUDA with bf16 and 64 or 128 channels a head this is one kernel (``csrc/rotary.cu``); others take torch
    operations on the device.
    """
    if use_native(q) and q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[-1] in (64, 128):
        return native().rotary_append(q, k, v, k_cache, v_cache, k_scale, v_scale, lengths, cos, sin, interleave)
    if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together.")
    if k.shape[2] != k_cache.shape[1]:
        raise ValueError(f"{k.shape[2]} key heads for a cache of {k_cache.shape[1]}.")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together.")
    if cos is not None and (cos.ndim != 2 or cos.shape != sin.shape or not 2 <= 2 * cos.shape[1] <= q.shape[-1] or cos.shape[0] < 1):
        raise ValueError(f"cos and sin must be [positions, R/2] tables with 2 <= R <= {q.shape[-1]}, got {tuple(cos.shape)}.")
    _check_cache(q, k_cache, v_cache, k_scale, v_scale, lengths)
    if _overlap(k_cache) or _overlap(v_cache) or _overlap(k_scale) or _overlap(v_scale):
        raise ValueError("caches and scales must not overlap themselves.")
    if _overlap(k_cache, v_cache) or _overlap(k_scale, v_scale):
        raise ValueError("keys and values need caches and scales of their own.")
    if any(x.requires_grad for x in (q, k, v)) and torch.is_grad_enabled():
        raise RuntimeError("rotary_append has no gradient: call it under torch.no_grad().")
    return reference.rotary_append(q, k, v, k_cache, v_cache, k_scale, v_scale, lengths, cos, sin, interleave)


def cache_attention(
    q: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    k_scale: Tensor,
    v_scale: Tensor,
    lengths: Tensor,
    *,
    scale: float | None = None,
    window: int | None = None,
    offset: int = 0,
) -> Tensor:
    """Attention of each sequence's last tokens over its 8-bit cache (see :func:`rotary_append`).

    ``q`` is ``[B, H, D]`` (one token per sequence) or ``[B, s, H, D]`` (a chunk). ``n = min(lengths[b] + offset, T)``
    rows of sequence ``b`` are filled, the chunk's own included: query ``i`` stands at position ``n - s + i``
    (so a chunk that ran past the cache's end stands at the last ``s`` rows) and sees the rows up to its own,
    with ``window`` only those not more than ``window`` behind it. A query that sees no row gives zeros; rows
    that a query does not see may hold anything; a NaN among the values reaches its own channel of the queries
    that see its row. Query head ``h`` reads KV head ``h // (H / Hkv)``. The lengths stay on the device, so the
    call can be captured in a CUDA graph. Returns ``q``'s shape.

    On CUDA with bf16 queries and 64 or 128 channels a head this runs ``csrc/cache_attention*.cu``; others take
    torch operations on the device. The kernels round the weights to f16 (half a step is 2**-11 of one) and keep a
    query's channels exactly down to 2**-30 of the largest one.
    """
    if window is not None and window < 0:
        window = None
    if not 0 <= offset < 1 << 31:
        raise ValueError(f"offset must be a token count, got {offset}.")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if use_native(q) and q.dtype == torch.bfloat16 and q.shape[-1] in (64, 128):
        return native().cache_attn(
            q, k_cache, v_cache, k_scale, v_scale, lengths, offset, scale, -1 if window is None else int(window)
        )
    if q.ndim not in (3, 4):
        raise ValueError(f"q must be [B, H, D] or [B, s, H, D], got {tuple(q.shape)}.")
    q4 = q[:, None] if q.ndim == 3 else q
    _check_cache(q4, k_cache, v_cache, k_scale, v_scale, lengths)
    if k_cache.shape[1] < 1 or q4.shape[2] % k_cache.shape[1]:
        raise ValueError(f"{q4.shape[2]} query heads are not a multiple of {k_cache.shape[1]} KV heads.")
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("cache_attention has no gradient: call it under torch.no_grad().")
    out = reference.cache_attention(
        q4, k_cache, v_cache, k_scale, v_scale, lengths, scale=scale, window=window, offset=offset
    )
    return out[:, 0] if q.ndim == 3 else out


def cross_entropy(logits: Tensor, targets: Tensor, *, ignore_index: int = -100, softcap: float | None = None) -> Tensor:
    """Unreduced token CE in fp32 of ``[..., V]`` logits, optionally soft-capped by ``softcap * tanh(x / softcap)``.

    bf16 CUDA logits with ``V % 8 == 0`` run the CE kernels (one read of the row for the
    log-sum-exp, one read and one write for the gradient).
    """
    if (
        use_native(logits)
        and logits.dtype == torch.bfloat16
        and logits.shape[-1] % 8 == 0
        and (softcap is None or softcap > 0)
    ):
        from priml_b200.ops import functional

        return functional.cross_entropy(logits, targets, ignore_index=ignore_index, softcap=softcap)
    return reference.cross_entropy(logits, targets, ignore_index=ignore_index, softcap=softcap)


def linear_cross_entropy(
    hidden: Tensor,
    weight: Tensor,
    targets: Tensor,
    *,
    ignore_index: int = -100,
    softcap: float | None = None,
) -> Tensor:
    """Unreduced CE of ``hidden @ weight.T`` in fp32, optionally soft-capped.

    On CUDA the bf16 logits are written once by the GEMM; the CE kernels read them
    for the log-sum-exp (with the cap applied on the fly) and overwrite them with
    d(logits) in the backward, so no fp32 or capped copy of the logits exists.
    """
    if use_native(hidden) and _compute_dtype(hidden) == torch.bfloat16:
        from priml_b200.ops import functional

        return functional.linear_cross_entropy(hidden, weight, targets, ignore_index=ignore_index, softcap=softcap)
    return reference.linear_cross_entropy(hidden, weight, targets, ignore_index=ignore_index, softcap=softcap)


def grouped_swiglu_mlp(x_sorted: Tensor, up_w: Tensor, down_w: Tensor, offsets: Tensor) -> Tensor:
    """Grouped SwiGLU experts over expert segments ``offsets[e]:offsets[e+1]`` (device-side
    offsets; on CUDA the segments must start on multiples of 128, as the padded plan lays them out)."""
    if use_native(x_sorted):
        from priml_b200.ops import grouped

        return grouped.grouped_swiglu_mlp(x_sorted, up_w, down_w, offsets)
    return reference.grouped_swiglu_mlp(x_sorted, up_w, down_w, offsets)


def grouped_swiglu_experts(x: Tensor, weights: Tensor, indices: Tensor, up_w: Tensor, down_w: Tensor) -> Tensor:
    """Routed SwiGLU experts: padded device-side dispatch, grouped expert MLP, weighted combine."""
    from priml_b200.ops import grouped

    return grouped.grouped_swiglu_experts(x, weights, indices, up_w, down_w)


def adamw_(
    params: list[Tensor],
    grads: list[Tensor],
    exp_avgs: list[Tensor],
    exp_avg_sqs: list[Tensor],
    **hyper: float,
) -> None:
    if params and use_native(params[0]):
        from priml_b200.ops import functional

        functional.adamw_(params, grads, exp_avgs, exp_avg_sqs, **hyper)
        return
    reference.adamw_(params, grads, exp_avgs, exp_avg_sqs, **hyper)  # type: ignore[arg-type]
