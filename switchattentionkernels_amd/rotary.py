"""What stands between a layer's projections and its attention: per-head norms of
queries and keys and their rotation by positions, in one pass.

The reference starts at finished Q and K.  These make them from a projection's
slices, contiguous as the attention wants them:

* ``switch_qk_rotary_forward`` normalises (optionally) and rotates;
* ``switch_qk_rotary_backward`` gives the gradients, ``switch_qk_rotary`` is the
  forward as a node of autograd's graph;
* ``switch_qk_rotary_append`` rotates new tokens of a serving batch, with the keys and
  values going into bf16 caches (those of ``switch_gqa_decode_forward``).

For every head row x of 128 dims: ``y = w x / sqrt(mean(x^2) + eps)`` where the tensor
has a weight w (else ``y = x``), then for every pair (a, b) of the first
``2 * inv_freq.numel()`` dims ``(a cos t - b sin t, b cos t + a sin t)`` with t the pair's
frequency times the token's position.  Sums and products are in fp32 and every value
is rounded once, to bf16; angles are as good at position 2^31 as at 0.

All device work runs in ``libswattn.so`` (``include/swattn_rotary.h``) on torch's
current stream.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .cache import check_lens

MAX_AXES = 4   # SWATTN_ROTARY_MAX_AXES


def _validate_rows(name: str, x: torch.Tensor, device) -> None:
    if not isinstance(x, torch.Tensor) or x.dtype != torch.bfloat16:
        raise TypeError("Switch Attention rotary requires BF16 Q/K/V")
    if not x.is_cuda or x.device != device:
        raise ValueError("Q/K/V must be on one supported accelerator device")
    if x.ndim != 4 or x.shape[3] != 128 or x.shape[0] == 0 or x.shape[2] == 0:
        raise ValueError(f"{name} must be [B,S,H,128] with at least one sequence and head")
    if x.layout != torch.strided or x.numel() and (
            x.stride(3) != 1 or any(s % 8 for s, n in zip(x.stride(), x.shape[:3]) if n > 1)
            or x.data_ptr() % 16):
        raise ValueError(f"{name}'s head rows must be contiguous and start at multiples of 16 bytes")


def _validate(q, k, positions, inv_freq, sections, q_weight, k_weight, eps) -> None:
    """Raise for the first argument that is not as documented."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("Switch Attention rotary requires BF16 Q/K/V")
    dev = q.device
    _validate_rows("q", q, dev)
    _validate_rows("k", k, dev)
    if q.shape[:2] != k.shape[:2]:
        raise ValueError("Q and K must have the same batch size and length")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype not in (torch.float32, torch.float64):
        raise TypeError("inv_freq must be an FP32 or FP64 tensor")
    if (inv_freq.ndim != 1 or inv_freq.device != dev or inv_freq.numel() % 8
            or not 8 <= inv_freq.numel() <= 64):
        raise ValueError("inv_freq must be 1-D on the device of Q, with 8 to 64 frequencies, a "
                         "multiple of 8")
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 1 or sum(sections) != inv_freq.numel():
        raise ValueError("sections must be 1 to 4 positive counts that add up to the frequencies")
    want = (len(sections),) + tuple(q.shape[:2])
    if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32:
        raise TypeError("positions must be an int32 tensor")
    if tuple(positions.shape) != want or positions.device != dev:
        raise ValueError("positions must be [axes,B,S] (or [B,S] for one axis) on the device of Q")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or w.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{name} must be an FP32 or BF16 tensor")
        if tuple(w.shape) != (128,) or w.device != dev:
            raise ValueError(f"{name} must be [128] on the device of Q")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight must have the same type")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")


def _arguments(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, look=None):
    """The same arguments, checked (``look``: at q, k and the weights as they came, too),
    positions ``[axes,B,S]`` and all but q and k contiguous."""
    if isinstance(positions, torch.Tensor) and positions.ndim == 2:
        positions = positions.unsqueeze(0)
    if sections is None:
        sections = [inv_freq.numel()] if isinstance(inv_freq, torch.Tensor) else [0]
    else:
        sections = [int(n) for n in sections]
    _validate(q, k, positions, inv_freq, sections, q_weight, k_weight, eps)
    if look is not None:
        look(q, k, q_weight, k_weight)
    return (q, k, positions.contiguous(), inv_freq.contiguous(), sections,
            *(None if w is None else w.contiguous() for w in (q_weight, k_weight)), eps)


def _quick(call, *args):
    """What the native call gives: None where its arguments need a look, which also holds
    for those that it cannot take at all."""
    try:
        return call(*args)
    except TypeError:
        return None


def switch_qk_rotary_forward(
        q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
        sections: Optional[Sequence[int]] = None, interleaved: bool = False,
        q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
        eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated queries and keys, new contiguous tensors in the shapes of
    ``q`` and ``k``.

    ``q``: bf16 ``[B, S, Hq, 128]``; ``k``: bf16 ``[B, S, Hkv, 128]``.  Head rows are
    contiguous; the other strides are free in steps of 16 bytes, so that slices of a fused
    projection need no copy.
    ``positions``: int32 ``[B, S]``, any sign, or with several axes ``[axes, B, S]``
    (time, height and width of image tokens, say).  ``inv_freq``: fp32 or fp64, 8 to 64
    frequencies in radians per position, a multiple of 8, on the device; twice as many
    dims are rotated, the others stay.  With axes ``sections`` says how many of the
    frequencies, in order, belong to each (up to four).  Pair i is dims
    ``(i, i + inv_freq.numel())``, or with ``interleaved`` ``(2 i, 2 i + 1)``.
    ``q_weight`` / ``k_weight``: fp32 or bf16 ``[128]``, of one type; where one is given,
    its rows are normalised first (each head by itself).
    """
    return _rotate(_lib.native().rotary_forward, q, k, positions, inv_freq, sections, interleaved,
                   q_weight, k_weight, eps)


def _rotate(call, q, k, positions, inv_freq, sections, interleaved, q_weight, k_weight, eps, look=None):
    interleaved, eps = bool(interleaved), float(eps)
    made = (_lib.like_contiguous(q), _lib.like_contiguous(k))
    out = _quick(call, q, k, positions, inv_freq, sections, interleaved, q_weight, k_weight, eps, *made)
    if out is None:
        q, k, positions, inv_freq, sections, q_weight, k_weight, eps = _arguments(
            q, k, positions, inv_freq, sections, q_weight, k_weight, eps, look)
        out = call(q, k, positions, inv_freq, sections, interleaved, q_weight, k_weight, eps, *made)
    return out


def switch_qk_rotary_backward(
        grad_q: torch.Tensor, grad_k: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
        positions: torch.Tensor, inv_freq: torch.Tensor, *, sections: Optional[Sequence[int]] = None,
        interleaved: bool = False, q_weight: Optional[torch.Tensor] = None,
        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_grads: bool = True):
    """Gradients of ``switch_qk_rotary_forward``'s outputs, given theirs (``grad_q`` and
    ``grad_k``: contiguous bf16 in the outputs' shapes) and that call's arguments.

    Returns ``(dq, dk, dq_weight, dk_weight)``: dq and dk bf16 and contiguous, the weights'
    gradients in the weights' type, None where there is no weight (or without
    ``weight_grads``).  They are summed in fp32 in a fixed order.
    """
    interleaved, eps, call = bool(interleaved), float(eps), _lib.native().rotary_backward
    out = _quick(call, grad_q, grad_k, q, k, positions, inv_freq, sections, interleaved, q_weight,
                 k_weight, eps, bool(weight_grads))
    if out is None:
        q, k, positions, inv_freq, sections, q_weight, k_weight, eps = _arguments(
            q, k, positions, inv_freq, sections, q_weight, k_weight, eps)
        for name, g, x in (("grad_q", grad_q, q), ("grad_k", grad_k, k)):
            if (not isinstance(g, torch.Tensor) or g.shape != x.shape or g.dtype != torch.bfloat16
                    or g.device != x.device or not g.is_contiguous() or g.numel() and g.data_ptr() % 16):
                raise ValueError(f"{name} must be a contiguous BF16 tensor shaped like {name[-1].upper()}")
        out = call(grad_q, grad_k, q, k, positions, inv_freq, sections, interleaved, q_weight, k_weight,
                   eps, bool(weight_grads))
    return out


def switch_qk_rotary(q, k, positions, inv_freq, *, sections: Optional[Sequence[int]] = None,
                     interleaved: bool = False, q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``switch_qk_rotary_forward`` with autograd support for q, k and the weights (once:
    gradients of gradients raise).  The graph keeps the rows of a tensor that has a weight;
    without one they may be freed or changed before the backward.

    Under capture the leaves among them, and those that they are views of, must not belong to
    an eager graph that still lives (such a call raises: the captured backward would end the
    process).  Leaves further back are the caller's to look after."""
    native = _lib.native()
    return _rotate(native.rotary_autograd, q, k, positions, inv_freq, sections, interleaved, q_weight,
                   k_weight, eps, native.rotary_leaves)


def _validate_append(q, k, v, k_cache, v_cache, lens, counts) -> None:
    dev = q.device
    _validate_rows("v", v, dev)
    if v.shape != k.shape:
        raise ValueError("K and V must have identical shapes")
    for t in (k_cache, v_cache):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16:
            raise TypeError("the caches must be BF16")
        if t.device != dev:
            raise ValueError("the caches must be on the device of Q")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("the caches must be contiguous and 16-byte aligned")
    if (k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] == 0
            or k_cache.shape[0] != k.shape[0] or k_cache.shape[2:] != k.shape[2:]):
        raise ValueError("the caches must be [B,L,Hkv,128] of one shape, with K's batch size and heads")
    for name, t in (("cache_lens", lens), ("row_counts", counts)):
        if not isinstance(t, torch.Tensor) and not (t is None and name == "row_counts"):
            raise TypeError(f"{name} must be a tensor")
    check_lens(lens, q.shape[0], dev, "cache_lens")
    if counts is not None:
        check_lens(counts, q.shape[0], dev, "row_counts")


def switch_qk_rotary_append(
        q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
        v_cache: torch.Tensor, cache_lens: torch.Tensor, positions: torch.Tensor,
        inv_freq: torch.Tensor, *, row_counts: Optional[torch.Tensor] = None,
        sections: Optional[Sequence[int]] = None, interleaved: bool = False,
        q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
        eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``switch_qk_rotary_forward`` of T new tokens for each of B sequences, with the keys
    written into ``k_cache`` and the values ``v`` (as they are, shaped like ``k``) into
    ``v_cache`` (bf16 ``[B, L, Hkv, 128]``, contiguous), behind each sequence's
    ``cache_lens[b]`` valid rows (int32 ``[B]`` on the device, clamped to ``[0, L]``).

    Returns ``(q, cache_lens)``: the rotated queries and the new lengths (the argument
    stays as it is).  Of sequence b the first ``row_counts[b]`` tokens are appended (int32
    ``[B]`` on the device, clamped to ``[0, T]``; default all); rows that do not fit the
    cache any more are dropped and the new length is the capacity.  Other rows of the
    caches keep their contents, and the q rows of tokens that are not appended are
    rotated like the rest.  ``positions`` are the tokens' own, whatever the cache holds.
    A captured call writes the same q and lengths at each replay; copy the lengths where the
    next replay reads them.
    """
    interleaved, eps, call = bool(interleaved), float(eps), _lib.native().rotary_append
    made = _lib.like_contiguous(q)
    out = _quick(call, q, k, v, k_cache, v_cache, cache_lens, row_counts, positions, inv_freq, sections,
                 interleaved, q_weight, k_weight, eps, made)
    if out is None:
        q, k, positions, inv_freq, sections, q_weight, k_weight, eps = _arguments(
            q, k, positions, inv_freq, sections, q_weight, k_weight, eps)
        _validate_append(q, k, v, k_cache, v_cache, cache_lens, row_counts)
        lens = cache_lens.contiguous()
        counts = None if row_counts is None else row_counts.contiguous()
        read = [q, k, v, lens, positions, inv_freq]
        read += [t for t in (counts, q_weight, k_weight) if t is not None]
        if not _lib.native().rotary_apart((k_cache, v_cache), read):
            raise ValueError("the caches must not share memory with each other or the other arguments")
        out = call(q, k, v, k_cache, v_cache, lens, counts, positions, inv_freq, sections, interleaved,
                   q_weight, k_weight, eps, made)
    return out
