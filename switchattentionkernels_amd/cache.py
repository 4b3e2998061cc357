"""A KV cache in 8 bits: quantised appends, reads, and eviction by accumulated
attention weight.

The reference is prefill-only and keeps no cache.  ``SwitchKVCache`` holds one
layer's keys and values as one-byte codes with a scale for each block of
tokens and KV head, half the memory and half the traffic of the bf16 caches of
``switch_gqa_decode_forward``:

* ``build_switch_kv_cache`` makes an empty one;
* ``switch_kv_cache_append`` quantises new rows, a prompt's or one token's, behind
  each sequence's valid rows;
* ``switch_kv_cache_read`` gives rows back in bf16, for a prefill over what is
  cached;
* ``switch_gqa_decode_quantized_forward`` (``decode.py``) attends it;
* ``switch_kv_cache_evict`` keeps the newest rows and the heaviest of the others,
  by the sums that ``switch_gqa_prefill_key_weights`` (``weights.py``) starts
  and the decode step adds to.

Lengths are the caller's, as for ``switch_gqa_decode_forward``: int32 ``[B]`` on
the device.  Scales written here are powers of two: for a block's largest
magnitude ``a`` the smallest ``2^e >= 2^-100`` with ``a <= qmax * 2^e`` (qmax 448
for e4m3, 127 for int8).  Scaling is then exact and every value is rounded once,
to the nearest code that stands for a finite bf16 number.  A block that takes a NaN or an
infinity reads as NaN.

All device work runs in ``libswattn.so`` (``include/swattn_cache.h``) on torch's
current stream.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .metadata import _as_cu

BLOCK_SIZES = (16, 32, 64, 128)
HOST_MAX_SEQS = 256   # SWATTN_CACHE_HOST_MAX_SEQS
_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}   # SWATTN_CODE_*


@dataclass(frozen=True)
class SwitchKVCache:
    """Codes and scales of one layer's cache.

    ``k``/``v``: ``torch.float8_e4m3fn`` or ``torch.int8`` ``[B, L, Hkv, 128]``;
    ``k_scales``/``v_scales``: fp32 ``[B, Hkv, ceil(L / block_size)]``; row ``r`` of
    head ``h`` stands for ``code * scale[b, h, r // block_size]``.  All
    contiguous, on one device.  Rows behind a sequence's length, and scales of
    blocks without a valid row, may hold anything.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    block_size: int


def build_switch_kv_cache(batch: int, capacity: int, kv_heads: int, *, device,
                          dtype: torch.dtype = torch.float8_e4m3fn,
                          block_size: int = 64) -> SwitchKVCache:
    """An empty cache of ``capacity`` rows for each of ``batch`` sequences (its
    memory is not cleared: nothing reads behind a sequence's length)."""
    if dtype not in _CODES:
        raise TypeError("the cache holds float8_e4m3fn or int8 codes")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if batch < 1 or capacity < 1 or kv_heads < 1:
        raise ValueError("the cache needs at least one sequence, row and KV head")
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError("the cache must be on a supported accelerator device")
    codes = [torch.empty(batch, capacity, kv_heads, 128, dtype=dtype, device=dev) for _ in range(2)]
    scales = [torch.empty(batch, kv_heads, -(-capacity // block_size), dtype=torch.float32,
                          device=dev) for _ in range(2)]
    return SwitchKVCache(*codes, *scales, block_size)


def _parts(cache: SwitchKVCache):
    return cache.k, cache.v, cache.k_scales, cache.v_scales


def _all_tensors(*args) -> bool:
    for t in args:
        if not isinstance(t, torch.Tensor):
            return False
    return True


def check_cache(cache: SwitchKVCache) -> None:
    """Raise unless ``cache`` is whole: types, shapes, one device.  In Python only
    where one of the conditions fails."""
    tensors = _parts(cache)
    if (not _all_tensors(*tensors)
            or not _lib.native().cache_ok(*tensors, int(cache.block_size))):
        _validate_cache(cache)


def _validate_cache(cache: SwitchKVCache) -> None:
    k, v, ks, vs = cache.k, cache.v, cache.k_scales, cache.v_scales
    if k.dtype not in _CODES or v.dtype != k.dtype:
        raise TypeError("the cache holds float8_e4m3fn or int8 codes, K and V alike")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("the cache's scales must be FP32")
    if not k.is_cuda:
        raise ValueError("the cache must be on a supported accelerator device")
    if cache.block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if k.ndim != 4 or k.shape != v.shape or k.shape[3] != 128 or 0 in k.shape:
        raise ValueError("the cache's codes must be [B,L,Hkv,128], K and V alike, and not empty")
    want = (k.shape[0], k.shape[2], -(-k.shape[1] // cache.block_size))
    if tuple(ks.shape) != want or tuple(vs.shape) != want:
        raise ValueError("the cache's scales must be [B,Hkv,ceil(L/block_size)]")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("the cache's tensors must be contiguous")
    if not (k.device == v.device == ks.device == vs.device):
        raise ValueError("the cache's tensors must be on the same device")


def check_lens(lens: torch.Tensor, batch: int, device, name: str) -> torch.Tensor:
    if lens.dtype != torch.int32 or lens.shape != (batch,) or lens.device != device:
        raise ValueError(f"{name} must be an int32 [B] tensor on the device of the cache")
    return lens.contiguous()


def check_weights(weights: torch.Tensor, cache: SwitchKVCache) -> None:
    b, n, h, _ = cache.k.shape
    if weights.dtype != torch.float32:
        raise TypeError("key_weights must be FP32")
    if weights.shape != (b, h, n) or weights.device != cache.k.device:
        raise ValueError("key_weights must be [B,Hkv,L] on the device of the cache")
    if not weights.is_contiguous():
        raise ValueError("key_weights must be contiguous")


def _append_arguments(cache, k, v, cache_lens, row_counts, cu_seqlens):
    """(cache_lens, row_counts, offsets on the device, offsets on the host, most
    rows of a sequence), checked."""
    check_cache(cache)
    batch, capacity, heads, _ = cache.k.shape
    dev = cache.k.device
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError("Switch Attention caches are filled from BF16 K/V")
    if k.device != dev or v.device != dev:
        raise ValueError("K/V must be on the device of the cache")
    if k.ndim != 4 or k.shape != v.shape or tuple(k.shape[2:]) != (heads, 128):
        raise ValueError("K/V must be [B,T,Hkv,128] of one shape, with the cache's KV heads")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("K/V must be contiguous")
    lens = check_lens(cache_lens, batch, dev, "cache_lens")
    rows = int(k.shape[1])
    cu, host_cu = None, []
    if cu_seqlens is not None:
        if row_counts is not None:
            raise ValueError("row_counts and cu_seqlens exclude each other")
        if k.shape[0] != 1:
            raise ValueError("packed K/V must have batch size 1")
        if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda:
            _lib.refuse_capture(dev, "reads cu_seqlens back from the device")
        offsets = _as_cu(cu_seqlens, rows, "cu_seqlens")
        if len(offsets) != batch + 1:
            raise ValueError("cu_seqlens must hold one sequence for each of the cache's")
        if batch <= HOST_MAX_SEQS:
            host_cu = offsets
        else:
            _lib.refuse_capture(dev, f"copies cu_seqlens of more than {HOST_MAX_SEQS} sequences to the device")
            cu = torch.tensor(offsets, dtype=torch.int32, device=dev)
        most = max(b - a for a, b in zip(offsets, offsets[1:]))
    else:
        if k.shape[0] != batch:
            raise ValueError("K/V and cache batch sizes must match")
        if row_counts is not None:
            row_counts = check_lens(row_counts, batch, dev, "row_counts")
        most = rows
    if most > capacity:
        raise ValueError("more rows than the cache holds")
    if not _lib.native().apart(_parts(cache), (k, v, lens)):
        raise ValueError("K, V and the cache's tensors must not overlap in memory")
    return lens, row_counts, cu, host_cu, most


def switch_kv_cache_append(cache: SwitchKVCache, k: torch.Tensor, v: torch.Tensor,
                           cache_lens: torch.Tensor, *,
                           row_counts: Optional[torch.Tensor] = None,
                           cu_seqlens=None) -> torch.Tensor:
    """Quantise new rows into the cache, behind each sequence's ``cache_lens[b]``
    valid ones; returns the new lengths, int32 ``[B]`` (``cache_lens`` itself is
    left as it is).

    ``k``/``v``: bf16 ``[B, T, Hkv, 128]`` with T at most the capacity, of which
    sequence b appends its first ``row_counts[b]`` (int32 ``[B]`` on the device,
    clamped to ``[0, T]``; default all).  Or, with ``cu_seqlens`` (int list or
    tensor of ``B + 1`` offsets), packed ``[1, total, Hkv, 128]`` as for
    ``switch_gqa_prefill_varlen_forward``, each sequence at most the capacity.  The host
    needs these offsets: a device tensor is read back, which waits for the stream; a captured
    call keeps the offsets it was captured with (of up to 256 sequences, from a list or a host
    tensor; others are refused under capture).
    Rows that do not fit the cache any more are dropped, and the new length is
    the capacity.  A block that already held rows takes the larger scale of its
    own and its new rows', and its rows are rounded again where it grows.
    """
    lens, cu, host_cu = cache_lens, None, []
    tensors = _parts(cache)
    if cu_seqlens is None and _all_tensors(*tensors, k, v, lens) and _lib.native().append_ok(
            *tensors, int(cache.block_size), k, v, lens, row_counts):
        most = k.shape[1]
    else:
        lens, row_counts, cu, host_cu, most = _append_arguments(cache, k, v, cache_lens, row_counts,
                                                                cu_seqlens)
    dev = cache.k.device
    with _lib.on_device(dev):
        return _lib.native().cache_append(k, v, cu, host_cu, row_counts, lens, *tensors, most,
                                          cache.block_size, _CODES[cache.k.dtype],
                                          _lib.stream_handle(dev))


def switch_kv_cache_read(cache: SwitchKVCache, starts: Union[int, torch.Tensor], rows: int, *,
                         cache_lens: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rows`` rows of each sequence from row ``starts`` on (an int, or int32 ``[B]``
    on the device) as ``(k, v)``, bf16 ``[B, rows, Hkv, 128]``.

    Rows at or behind ``cache_lens[b]`` (default: the capacity), or before 0,
    come out as 0.  With the power-of-two scales that this package writes the
    values are exact in bf16.
    """
    first, tensors = 0, _parts(cache)
    if not isinstance(starts, torch.Tensor):
        first, starts = int(starts), None
    if rows < 0 or not _all_tensors(*tensors) or not _lib.native().read_ok(
            *tensors, int(cache.block_size), starts, cache_lens):
        check_cache(cache)
        if rows < 0:
            raise ValueError("rows must not be negative")
        batch, dev = cache.k.shape[0], cache.k.device
        if starts is not None:
            starts = check_lens(starts, batch, dev, "starts")
        if cache_lens is not None:
            cache_lens = check_lens(cache_lens, batch, dev, "cache_lens")
    if not 0 <= first < 2 ** 31:
        raise ValueError("starts must not be negative")
    dev = cache.k.device
    with _lib.on_device(dev):
        return _lib.native().cache_read(*tensors, starts, first, cache_lens, int(rows),
                                        cache.block_size, _CODES[cache.k.dtype],
                                        _lib.stream_handle(dev))


def switch_kv_cache_evict(cache: SwitchKVCache, cache_lens: torch.Tensor, key_weights: torch.Tensor,
                          *, budget: int, recent: int, capacity: Optional[int] = None,
                          out: Optional[SwitchKVCache] = None,
                          out_weights: Optional[torch.Tensor] = None
                          ) -> Tuple[SwitchKVCache, torch.Tensor, torch.Tensor]:
    """Cut every sequence of more than ``budget`` rows to that many, in another cache.

    For each KV head on its own, the newest ``recent`` rows stay and those
    ``budget - recent`` of the older ones with the largest ``key_weights`` (fp32
    ``[B, Hkv, L]``; NaN counts as largest, of equal weights the lower row
    stays).  Kept rows keep their order, so that a local query still finds its
    window at the end where ``recent`` is at least the window.  Shorter
    sequences are copied whole.  Each block of the destination gets the scale
    that its rows need.

    Returns ``(cache, cache_lens, key_weights)``: the destination, its lengths
    and the kept rows' weights, 0 behind them.  The destination is new, of
    ``capacity`` rows (default: as many as ``cache``), or ``out`` with
    ``out_weights`` (same batch, heads, dtype and block size, at least
    ``budget`` rows), which must not share memory with the source: two caches
    in turn let a captured decode loop go on.
    """
    lens, tensors = cache_lens, _parts(cache)
    if not _all_tensors(*tensors, lens, key_weights) or not _lib.native().evict_ok(
            *tensors, int(cache.block_size), lens, key_weights):
        check_cache(cache)
        lens = check_lens(cache_lens, cache.k.shape[0], cache.k.device, "cache_lens")
        check_weights(key_weights, cache)
    batch, n, heads, _ = cache.k.shape
    dev = cache.k.device
    budget, recent = int(budget), int(recent)
    if budget < 1:
        raise ValueError("budget must be positive")
    if not 0 <= recent <= budget:
        raise ValueError("recent must lie in [0, budget]")
    if (out is None) != (out_weights is None):
        raise ValueError("out and out_weights go together")
    if out is not None and capacity is not None:
        raise ValueError("capacity and out exclude each other")
    if out is None:
        rows = n if capacity is None else int(capacity)
        if rows < budget:
            raise ValueError("the destination must hold at least budget rows")
        with _lib.on_device(dev):
            *made, out_weights, new_lens = _lib.native().cache_evict_new(
                *tensors, key_weights, lens, rows, cache.block_size, _CODES[cache.k.dtype], budget,
                recent, _lib.stream_handle(dev))
        return SwitchKVCache(*made, cache.block_size), new_lens, out_weights
    check_cache(out)
    if (out.k.shape[0], out.k.shape[2]) != (batch, heads) or out.k.device != dev:
        raise ValueError("out must have the cache's batch size, KV heads and device")
    if out.k.dtype != cache.k.dtype or out.block_size != cache.block_size:
        raise ValueError("out must have the cache's dtype and block_size")
    if out.k.shape[1] < budget:
        raise ValueError("the destination must hold at least budget rows")
    check_weights(out_weights, out)
    if not _lib.native().apart(_parts(out) + (out_weights,), tensors + (key_weights, lens)):
        raise ValueError("the destination's tensors must not share memory, with the source or "
                         "each other")
    with _lib.on_device(dev):
        new_lens = _lib.native().cache_evict(*tensors, key_weights, lens, *_parts(out),
                                             out_weights, cache.block_size, _CODES[cache.k.dtype],
                                             budget, recent, _lib.stream_handle(dev))
    return out, new_lens, out_weights
