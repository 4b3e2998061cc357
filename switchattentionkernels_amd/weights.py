"""The attention weight that each key received from a prefill's queries.

The sums that an eviction goes by (``switch_kv_cache_evict``) start with the
prompt: ``switch_gqa_prefill_key_weights`` computes them from the forward's
LSE, and decode steps add to them (``switch_gqa_decode_quantized_forward``).
The reference's forward (V:103-249) exports the log2 LSE (V:236-241) but no
weights.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .backward import _check_monotone
from .metadata import SwitchAttentionMetadata, _is_untouched
from .prefill import (ERR_OVERLAP, LOG2E, MSG_DISJOINT, _check_lists, _check_metadata,
                      _is_untouched_compaction, _note_sync, _prepare_indices, _raise_for, check_qkv)

WAITS_FOR_LISTS = "waits for the check of the index lists"


def switch_gqa_prefill_key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor,
                                   full_query_indices: torch.Tensor,
                                   local_query_indices: torch.Tensor, *,
                                   metadata: Optional[SwitchAttentionMetadata] = None,
                                   window_size: int = 1024,
                                   sm_scale: Optional[float] = None) -> torch.Tensor:
    """Softmax weight of every key, summed over the queries that see it and over
    the query heads of its KV head: fp32 ``[B, Hkv, Skv]``, 0 for a key that no
    query sees.

    The arguments are those of ``switch_gqa_prefill_forward`` (or, with packed
    sequences, their metadata) without V, and ``lse`` is its result.  Like the
    backward, it needs each list's key bounds non-decreasing along the list: true for metadata
    of ``build_switch_attention_metadata`` that was not modified since, checked for any other.
    Lists and bounds that need a check make the call wait for it, and a capture refuse it.

    Rows that are padding add to the keys before them like any other; a row whose ``lse`` is
    set to +inf adds nothing (its Q must be finite).
    """
    check_qkv(q, k, k)
    if window_size <= 0:
        raise ValueError("window_size must be positive")
    if (lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.device != q.device
            or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous FP32 tensor shaped [B, Sq, Hq]")
    batch, q_len, _, dim = q.shape
    kv_len = k.shape[1]
    if metadata is not None and batch != 1:
        raise ValueError("position metadata requires batch size 1; pack sequences with cu_seqlens")
    if kv_len == 0 and q_len > 0:
        raise ValueError("K must hold at least one position")
    scale = (1.0 / dim) ** 0.5 if sm_scale is None else float(sm_scale)
    if not math.isfinite(scale):
        raise ValueError("sm_scale must be finite")
    if metadata is not None:
        _check_metadata(metadata, q_len, kv_len, q.device)
    total_q, dev = batch * q_len, q.device
    fs, ls, ends = (None, None, None) if metadata is None else (
        metadata.full_starts, metadata.local_starts, metadata.causal_ends)
    full, local, unchecked = full_query_indices, local_query_indices, False
    if (metadata is None and 0 not in k.shape and full.ndim == 1 and local.ndim == 1
            and full.numel() + local.numel() == total_q > 0 and full.device == local.device == dev
            and not _is_untouched_compaction(full, local, total_q)):
        # The lists' values are checked by the call itself, beside its first kernel.
        _lib.refuse_capture(dev, WAITS_FOR_LISTS)
        full, local = _prepare_indices(full, device=dev), _prepare_indices(local, device=dev)
        _note_sync(dev)
        unchecked = True
    else:
        if not _is_untouched_compaction(full, local, total_q):
            _lib.refuse_capture(dev, WAITS_FOR_LISTS)
        full, local = _check_lists(full, local, total_q, dev)
        if metadata is not None and not _is_untouched(metadata):
            _lib.refuse_capture(dev, "waits for the check of the metadata's bounds")
            _check_monotone(metadata, full, local, "the sums of attention weights")
    if 0 in k.shape:
        return torch.zeros(batch, k.shape[2], kv_len, dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        out, flags = _lib.native().prefill_key_weights(q, k, lse, full, local, fs, ls, ends,
                                                       min(int(window_size), 2 ** 31 - 1),
                                                       scale * LOG2E, unchecked,
                                                       _lib.stream_handle(dev))
    if flags:
        _raise_for(flags, "full")
        _raise_for(flags, "local")
        if flags & ERR_OVERLAP:
            raise ValueError(MSG_DISJOINT)
    return out
