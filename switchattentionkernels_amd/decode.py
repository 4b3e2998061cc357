"""Routed decode: one new query token per sequence against its KV cache.

The reference is prefill-only.  This applies its routing rule to the last row
of a sequence (F:145-155): with ``n = cache_lens[b]`` the new token sits at
position ``n - 1`` -- its own K/V already appended -- and attends keys
``[0, n)`` when routed full, else the last ``window_size`` of them.  Output
follows the prefill's conventions: bf16 O and fp32 LSE in the log2
convention (V:15, V:236-241).  ``switch_gqa_decode_quantized_forward`` does the
same over an 8-bit cache (``cache.py``), ``switch_gqa_decode_shared_forward`` for
sequences that continue shared prefixes.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .cache import (_CODES, SwitchKVCache, _all_tensors, check_cache, check_lens,
                    check_weights)

LOG2E = 1.4426950408889634


def switch_gqa_decode_forward(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              cache_lens: torch.Tensor, full_mask: torch.Tensor, *,
                              window_size: int = 1024,
                              sm_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routed decode step.

    ``q``: bf16 ``[B, 1, Hq, 128]`` (or ``[B, Hq, 128]``); ``k_cache`` /
    ``v_cache``: bf16 ``[B, L, Hkv, 128]``; ``cache_lens``: int32 ``[B]``
    (valid cache rows, new token included; clamped to ``[0, L]``);
    ``full_mask``: bool ``[B]``, True = full attention over the cache.
    Returns ``(O [B, 1, Hq, 128] bf16, LSE [B, 1, Hq] fp32)``.
    """
    squeeze = q.ndim == 3
    if squeeze:
        q = q.unsqueeze(1)
    for t in (q, k_cache, v_cache):
        if t.dtype != torch.bfloat16:
            raise TypeError("Switch Attention decode requires BF16 Q and KV cache")
        if not t.is_cuda:
            raise ValueError("Q and KV cache must be tensors on a supported accelerator device")
        if not t.is_contiguous():
            raise ValueError("Q and KV cache must be contiguous")
    if q.ndim != 4 or q.shape[1] != 1 or k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("q must be [B,1,Hq,128] and the caches [B,L,Hkv,128] of one shape")
    batch, _, heads, dim = (int(x) for x in q.shape)
    _, cache_len, kv_heads, kdim = (int(x) for x in k_cache.shape)
    if dim != 128 or kdim != 128:
        raise ValueError("the decode kernel is specialized for head_dim=128")
    if k_cache.shape[0] != batch:
        raise ValueError("Q and KV cache batch sizes must match")
    if kv_heads == 0 or heads % kv_heads or heads // kv_heads > 8:
        raise ValueError("query heads must be a multiple (at most 8x) of KV heads")
    if cache_len == 0:
        raise ValueError("the KV cache must hold at least one position")
    if window_size <= 0:
        raise ValueError("window_size must be positive")
    dev = q.device
    if (cache_lens.dtype != torch.int32 or cache_lens.shape != (batch,)
            or cache_lens.device != dev):
        raise ValueError("cache_lens must be an int32 [B] tensor on the device of Q")
    if full_mask.dtype != torch.bool or full_mask.shape != (batch,) or full_mask.device != dev:
        raise ValueError("full_mask must be a bool [B] tensor on the device of Q")
    if not (k_cache.device == v_cache.device == dev):
        raise ValueError("Q and KV cache must be on the same device")
    scale = ((1.0 / dim) ** 0.5 if sm_scale is None else float(sm_scale)) * LOG2E
    lens = cache_lens.contiguous()
    full = full_mask.contiguous()
    with _lib.on_device(dev):
        out, lse = _lib.native().decode_forward(q, k_cache, v_cache, lens, full, int(window_size),
                                                scale, _lib.stream_handle(dev), _lib.like(q))
    if squeeze:
        return out[:, 0], lse[:, 0]
    return out, lse


def _check_quantized(q, cache: SwitchKVCache, cache_lens, full_mask):
    """(cache_lens, full_mask) for the kernels, or raise."""
    check_cache(cache)
    if q.dtype != torch.bfloat16:
        raise TypeError("Switch Attention decode requires BF16 Q")
    if not q.is_contiguous():
        raise ValueError("Q must be contiguous")
    if q.ndim != 4 or q.shape[1] != 1 or q.shape[3] != 128:
        raise ValueError("q must be [B,1,Hq,128]")
    batch, _, heads, _ = (int(x) for x in q.shape)
    if cache.k.shape[0] != batch:
        raise ValueError("Q and KV cache batch sizes must match")
    kv_heads = int(cache.k.shape[2])
    if heads == 0 or heads % kv_heads or heads // kv_heads > 8:
        raise ValueError("query heads must be a multiple (at most 8x) of KV heads")
    dev = cache.k.device
    if q.device != dev:
        raise ValueError("Q and KV cache must be on the same device")
    lens = check_lens(cache_lens, batch, dev, "cache_lens")
    if full_mask.dtype != torch.bool or full_mask.shape != (batch,) or full_mask.device != dev:
        raise ValueError("full_mask must be a bool [B] tensor on the device of Q")
    return lens, full_mask.contiguous()


def switch_gqa_decode_quantized_forward(
        q: torch.Tensor, cache: SwitchKVCache, cache_lens: torch.Tensor, full_mask: torch.Tensor, *,
        window_size: int = 1024, sm_scale: Optional[float] = None,
        key_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routed decode step over an 8-bit cache: ``switch_gqa_decode_forward`` with
    ``cache`` (``SwitchKVCache``) in the place of the bf16 caches.

    With ``key_weights`` (fp32 ``[B, Hkv, L]``) each attended key's softmax
    weight, summed over the query heads of its KV head, is added there in
    place; other entries keep their value.  A sequence without keys gives O =
    NaN and LSE = -inf and adds nothing.
    """
    squeeze = q.ndim == 3
    if squeeze:
        q = q.unsqueeze(1)
    lens, full = cache_lens, full_mask
    if not _all_tensors(q, cache.k, cache.v, cache.k_scales, cache.v_scales, lens, full) or \
            not _lib.native().decode_ok(q, cache.k, cache.v, cache.k_scales, cache.v_scales,
                                        int(cache.block_size), lens, full):
        lens, full = _check_quantized(q, cache, cache_lens, full_mask)
    if window_size <= 0:
        raise ValueError("window_size must be positive")
    dev = q.device
    if key_weights is not None:
        check_weights(key_weights, cache)
        if not _lib.native().apart((key_weights,), (q, cache.k, cache.v, cache.k_scales,
                                                    cache.v_scales, lens, full)):
            raise ValueError("key_weights must not share memory with the other arguments")
    scale = (128 ** -0.5 if sm_scale is None else float(sm_scale)) * LOG2E
    with _lib.on_device(dev):
        out, lse = _lib.native().cache_decode(q, cache.k, cache.v, cache.k_scales, cache.v_scales,
                                              lens, full, key_weights,
                                              min(int(window_size), 2 ** 31 - 1), cache.block_size,
                                              _CODES[cache.k.dtype], scale,
                                              _lib.stream_handle(dev), _lib.like(q))
    if squeeze:
        return out[:, 0], lse[:, 0]
    return out, lse


SHARED_MAX_SEQS = 1024       # SWATTN_SHARED_MAX_SEQS
SHARED_MAX_PREFIXES = 1024   # SWATTN_SHARED_MAX_PREFIXES


def _check_shared(q, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, cache_lens,
                  full_mask):
    """(prefix_lens, prefix_ids, cache_lens, full_mask) for the kernels, or raise."""
    rows = (q, k_prefix, v_prefix, k_cache, v_cache)
    if not _all_tensors(*rows) or any(t.dtype != torch.bfloat16 for t in rows):
        raise TypeError("Switch Attention decode requires BF16 Q, prefixes and KV cache")
    for name, t in (("prefix_lens", prefix_lens), ("prefix_ids", prefix_ids), ("cache_lens", cache_lens),
                    ("full_mask", full_mask)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
    dev = q.device
    if not q.is_cuda or any(t.device != dev for t in rows):
        raise ValueError("Q, prefixes and KV cache must be on one supported accelerator device")
    if any(not t.is_contiguous() or t.data_ptr() % 16 for t in rows):
        raise ValueError("Q, prefixes and KV cache must be contiguous and 16-byte aligned")
    if q.ndim != 4 or q.shape[1] != 1 or k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("q must be [B,1,Hq,128] and the caches [B,L,Hkv,128] of one shape")
    if k_prefix.ndim != 4 or k_prefix.shape != v_prefix.shape:
        raise ValueError("the prefixes must be [P,Lp,Hkv,128] of one shape")
    if any(t.shape[3] != 128 for t in rows):
        raise ValueError("the decode kernel is specialized for head_dim=128")
    batch, heads, kv_heads = int(q.shape[0]), int(q.shape[2]), int(k_cache.shape[2])
    if k_cache.shape[0] != batch:
        raise ValueError("Q and KV cache batch sizes must match")
    if kv_heads == 0 or heads == 0 or heads % kv_heads or heads // kv_heads > 8:
        raise ValueError("query heads must be a multiple (at most 8x) of KV heads")
    if k_prefix.shape[2] != kv_heads:
        raise ValueError("the prefixes must have the cache's KV heads")
    if any(t.numel() == 0 for t in rows):
        raise ValueError("the batch, the prefixes and the KV cache must hold at least one position")
    if batch > SHARED_MAX_SEQS or k_prefix.shape[0] > SHARED_MAX_PREFIXES:
        raise ValueError("at most 1024 sequences and 1024 prefixes")
    lens = check_lens(cache_lens, batch, dev, "cache_lens")
    ids = check_lens(prefix_ids, batch, dev, "prefix_ids")
    if (prefix_lens.dtype != torch.int32 or prefix_lens.shape != (k_prefix.shape[0],)
            or prefix_lens.device != dev):
        raise ValueError("prefix_lens must be an int32 [P] tensor on the device of Q")
    if full_mask.dtype != torch.bool or full_mask.shape != (batch,) or full_mask.device != dev:
        raise ValueError("full_mask must be a bool [B] tensor on the device of Q")
    return prefix_lens.contiguous(), ids, lens, full_mask.contiguous()


def switch_gqa_decode_shared_forward(
        q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, prefix_lens: torch.Tensor,
        prefix_ids: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
        cache_lens: torch.Tensor, full_mask: torch.Tensor, *, window_size: int = 1024,
        sm_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routed decode step of sequences that continue shared prefixes:
    ``switch_gqa_decode_forward`` where the rows of a system prompt or a document are kept
    once, and read once for every 128 query rows of a KV head that attend them.

    ``q``: bf16 ``[B, 1, Hq, 128]`` (or ``[B, Hq, 128]``); ``k_prefix`` / ``v_prefix``: bf16
    ``[P, Lp, Hkv, 128]``, of which prefix i holds the first ``prefix_lens[i]`` rows (int32
    ``[P]``, clamped to ``[0, Lp]``); ``prefix_ids``: int32 ``[B]``, the prefix that each
    sequence continues (outside ``[0, P)``: none); ``k_cache`` / ``v_cache``: bf16 ``[B, L,
    Hkv, 128]``, each sequence's own rows behind its prefix, ``cache_lens[b]`` of them, the
    new token's among them (int32 ``[B]``, clamped to ``[0, L]``); ``full_mask``: bool
    ``[B]``.  With ``n`` rows of prefix and cache together a sequence attends all of them
    when routed full, else the last ``window_size``.  Up to 1024 sequences and 1024 prefixes,
    of fewer than 2^31 rows of all KV heads (``include/swattn_shared.h`` has the bounds).

    Returns ``(O [B, 1, Hq, 128] bf16, LSE [B, 1, Hq] fp32)``; a sequence without any row
    gives O = NaN and LSE = -inf.
    """
    squeeze = isinstance(q, torch.Tensor) and q.ndim == 3
    if squeeze:
        q = q.unsqueeze(1)
    if window_size <= 0:
        raise ValueError("window_size must be positive")
    scale = (128 ** -0.5 if sm_scale is None else float(sm_scale)) * LOG2E
    if not abs(scale) < 2.0 ** 127:
        raise ValueError("sm_scale must be finite")
    call, how = _lib.native().shared_decode, (min(int(window_size), 2 ** 31 - 1), scale)
    try:
        out = call(q, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, cache_lens, full_mask,
                   *how, _lib.like(q))
    except TypeError:   # not tensors
        out = None
    if out is None:
        prefix_lens, prefix_ids, cache_lens, full_mask = _check_shared(
            q, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, cache_lens, full_mask)
        out = call(q, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, cache_lens, full_mask,
                   *how, _lib.like(q))
    if squeeze:
        return out[0][:, 0], out[1][:, 0]
    return out
