"""Prompts of different lengths through the 8-bit cache: appended, summed up, evicted and
decoded, padded and packed."""

import math

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (build_switch_attention_metadata, build_switch_kv_cache,
                                        build_switch_query_indices,
                                        switch_gqa_decode_quantized_forward,
                                        switch_gqa_prefill_forward, switch_gqa_prefill_key_weights,
                                        switch_kv_cache_append, switch_kv_cache_evict)

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS, T, HQ, HKV, W = [200, 1, 333, 64, 310], 333, 8, 2, 60
CU = [0, 200, 201, 534, 598, 908]
BUDGET, RECENT, BLOCK = 100, 60, 32


def _prompts():
    gen = torch.Generator().manual_seed(3)
    rows = [[torch.randn(n, h, 128, generator=gen).to(torch.bfloat16) for h in (HQ, HKV, HKV)] for n in LENS]
    masks = [torch.rand(n, generator=gen) < 0.4 for n in LENS]
    return gen, rows, masks


def _padded(gen, rows, masks, cache, sums):
    b = len(LENS)
    q, k, v = (torch.stack([torch.cat([r[i], 3 * torch.randn(T - n, *r[i].shape[1:], generator=gen).to(torch.bfloat16)])
                            for r, n in zip(rows, LENS)]).to(DEV) for i in range(3))
    mask = torch.stack([torch.cat([m, torch.rand(T - n, generator=gen) < 0.5]) for m, n in zip(masks, LENS)])
    full, local = build_switch_query_indices(mask.to(DEV))
    counts = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    _, lse = switch_gqa_prefill_forward(q, k, v, full, local, window_size=W)
    real = [lse[i, :n].cpu() for i, n in enumerate(LENS)]
    lens = switch_kv_cache_append(cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV), row_counts=counts)
    lse[torch.arange(T, device=DEV) >= counts[:, None]] = math.inf
    sums[:, :, :T] += switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=W)
    return lens, real


def _packed(gen, rows, masks, cache, sums):
    q, k, v = (torch.cat([r[i] for r in rows])[None].to(DEV) for i in range(3))
    full, local = build_switch_query_indices(torch.cat(masks).to(DEV))
    md = build_switch_attention_metadata(CU[-1], CU[-1], device=DEV, window_size=W, cu_seqlens=CU)
    _, lse = switch_gqa_prefill_forward(q, k, v, full, local, metadata=md)
    lens = switch_kv_cache_append(cache, k, v, torch.zeros(len(LENS), dtype=torch.int32, device=DEV), cu_seqlens=CU)
    got = switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
    for b, (first, end) in enumerate(zip(CU, CU[1:])):
        sums[b, :, :end - first] += got[0, :, first:end]
    return lens, [lse[0, a:e].cpu() for a, e in zip(CU, CU[1:])]


@pytest.mark.parametrize("form", [_padded, _packed])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_prompts_of_different_lengths(form, dtype):
    gen, rows, masks = _prompts()
    cache = build_switch_kv_cache(len(LENS), 400, HKV, device=DEV, dtype=dtype, block_size=BLOCK)
    sums = torch.zeros(len(LENS), HKV, 400, device=DEV)
    lens, lses = form(gen, rows, masks, cache, sums)
    assert lens.tolist() == LENS
    # Each prompt by itself in 64 bits: a weight's score is off by at most 130 * 2^-24 * c *
    # |q| |k| and 2^-23 of the LSE or that, in log2 units, the exponential by 2^-22.  A lane adds
    # one weight of a block of 32 rows, at most 42 of them, then come the lanes and chunks: 2^-18.
    for b, ((q, k, _), mask, lse) in enumerate(zip(rows, masks, lses)):
        n = LENS[b]
        i = torch.arange(n)
        want = C.key_weights(q, k, lse, torch.where(mask, 0, (i - W + 1).clamp(min=0)), i + 1).t()
        d = 128 ** -0.5 * math.log2(math.e) * float(q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max())
        eps = math.log(2) * (130 * 2.0 ** -24 * d + 2.0 ** -23 * max(d, float(lse.abs().max()))) + 2.0 ** -22 + 2.0 ** -18
        got = sums[b, :, :n].double().cpu()
        assert ((got - want).abs() <= eps * want).all(), b
        assert not sums[b, :, n:].any()
        assert abs(float(got.sum()) - n * HQ) <= eps * n * HQ
    # What the budget keeps goes by those sums.
    k, v = (C.cache_values(c, s, BLOCK) for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)))
    _, ends, rk, rv, _, _, rw = C.evict(k, v, sums.cpu().numpy(), LENS, BUDGET, RECENT, BLOCK, dtype)
    kept, after, left = switch_kv_cache_evict(cache, lens, sums, budget=BUDGET, recent=RECENT, capacity=BUDGET)
    assert after.tolist() == ends
    kk, vv = (C.cache_values(c, s, BLOCK) for c, s in ((kept.k, kept.k_scales), (kept.v, kept.v_scales)))
    for b, end in enumerate(ends):
        assert np.array_equal(kk[b, :end], rk[b, :end]) and np.array_equal(vv[b, :end], rv[b, :end])
        assert np.array_equal(left[b, :, :end].cpu().numpy(), rw[b, :, :end].astype(np.float32))
    # A step over it adds one weight per head.  A weight is off by its score's and the LSE's
    # error, 130 * 2^-24 of c |q| |k| each (log2 units), and 2^-20; O by one rounding more.
    q = torch.randn(len(LENS), 1, HQ, 128, generator=gen).to(torch.bfloat16).to(DEV)
    before = left.clone()
    out, _ = switch_gqa_decode_quantized_forward(q, kept, after, torch.ones(len(LENS), dtype=torch.bool, device=DEV),
                                                 key_weights=left)
    kk, vv = ([x[b, :end] for b, end in enumerate(ends)] for x in (kk, vv))
    k_max, v_max = max(np.linalg.norm(x, axis=-1).max() for x in kk), max(np.abs(x).max() for x in vv)
    eps = 2 * math.log(2) * 130 * 2.0 ** -24 * 128 ** -0.5 * math.log2(math.e) * k_max * float(q.float().norm(dim=-1).max()) + 2.0 ** -20
    for b, end in enumerate(ends):
        want = C.decode(q[b:b + 1, 0].cpu(), kk[b][None], vv[b][None], [end], [True], BUDGET)[0]
        assert (np.abs(out[b, 0].double().cpu().numpy() - want[0]) <= 2.0 ** -8 * np.abs(want[0]) + eps * v_max).all()
    total = (left - before).double().sum(-1)
    assert (total - HQ // HKV).abs().max() <= HQ // HKV * eps + 2.0 ** -23 * float(left.sum(-1).max())
