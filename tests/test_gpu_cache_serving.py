"""The 8-bit cache's operators together, as a serving program runs them: a prompt in
chunks over what is cached, the prompt's attention sums, eviction, decode steps with
appends, and random cases of each operator.  Every step is compared with a plain
64-bit evaluation on the values that the cache stands for (``oracle/cache.py``).
"""

import math

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (SwitchKVCache, build_switch_kv_cache,
                                        build_switch_query_indices, merge_attention_partials,
                                        shard_attention_metadata,
                                        switch_gqa_decode_quantized_forward,
                                        switch_gqa_prefill_forward,
                                        switch_gqa_prefill_key_weights, switch_kv_cache_append,
                                        switch_kv_cache_evict, switch_kv_cache_read)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rows_attention(q, k, v, start, end):
    """(O, LSE, P) in 64 bits: q [S, Hq, 128], k, v [N, Hkv, 128], bounds per row."""
    s, hq, _ = q.shape
    n, hkv = k.shape[:2]
    c = 128 ** -0.5 * math.log2(math.e)
    j = np.arange(n)
    see = (j >= start[:, None]) & (j < end[:, None])
    out, lse, weights = np.zeros((s, hq, 128)), np.zeros((s, hq)), np.zeros((n, hkv))
    for h in range(hq):
        x = np.where(see, c * (q[:, h] @ k[:, h // (hq // hkv)].T), -np.inf)
        m = x.max(axis=1, keepdims=True)
        p = np.exp2(x - m)
        lse[:, h] = (m + np.log2(p.sum(axis=1, keepdims=True)))[:, 0]
        p /= p.sum(axis=1, keepdims=True)
        out[:, h] = p @ v[:, h // (hq // hkv)]
        weights[:, h // (hq // hkv)] += p.sum(axis=0)
    return out, lse, weights


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_chunked_prompt_eviction_and_decode(dtype):
    """The prefill's products are bf16 MFMA with P in bf16: O within 2^-7 of the values
    it is a mean of (2^-8 from P's rounding and 2^-8 from the result's); merging
    rounds each part's O to bf16 once more.  The LSE and the sums have no such
    rounding: 1e-4 in log2 units, and ln 2 of that relative to a weight, cover 128
    fp32 terms many times over (128 * 2^-24 * the largest sum of |q_i k_i|, 60)."""
    gen = torch.Generator().manual_seed(17)
    hq, hkv, w, n, steps = 8, 2, 100, 700, 6
    cache = build_switch_kv_cache(1, n, hkv, device=DEV, dtype=dtype, block_size=32)
    lens = _int32([0])
    sums = torch.zeros(1, hkv, n, device=DEV)
    r = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)  # noqa: E731
    held_k, held_v = np.zeros((0, hkv, 128)), np.zeros((0, hkv, 128))
    want_sums = np.zeros((n, hkv))
    at = 0
    for size in (1, 250, 130, 129):
        q, k, v = r(1, size, hq, 128), r(1, size, hkv, 128), r(1, size, hkv, 128)
        mask = (torch.rand(size, generator=gen) < 0.4).to(DEV)
        full, local = build_switch_query_indices(mask)
        after = switch_kv_cache_append(cache, k, v, lens)
        # All queries attend what the cache holds, their own chunk included.
        hk, hv = switch_kv_cache_read(cache, 0, at + size, cache_lens=after)
        pos = torch.arange(at, at + size, dtype=torch.int32, device=DEV)
        cut = max(at // 2, 1)
        parts = []
        for a, b in ((0, cut), (cut, at + size)) if at else ((0, size),):
            md = shard_attention_metadata(pos, kv_start=a, kv_end=b, window_size=w)
            parts.append(switch_gqa_prefill_forward(q, hk[:, a:b].contiguous(), hv[:, a:b].contiguous(),
                                                    full, local, metadata=md))
        out, lse = merge_attention_partials(*zip(*parts)) if len(parts) > 1 else parts[0]
        md = shard_attention_metadata(pos, kv_start=0, kv_end=at + size, window_size=w)
        got = switch_gqa_prefill_key_weights(q, hk, lse, full, local, metadata=md)
        sums[:, :, :at + size] += got
        held_k, held_v = hk[0].double().cpu().numpy(), hv[0].double().cpu().numpy()
        i = np.arange(at, at + size)
        start = np.where(mask.cpu().numpy(), 0, np.maximum(i - w + 1, 0))
        ro, rl, rw = _rows_attention(q[0].double().cpu().numpy(), held_k, held_v, start, i + 1)
        assert np.abs(out[0].double().cpu().numpy() - ro).max() <= 2.0 ** -7 * 2 * np.abs(held_v).max()
        assert np.abs(lse[0].double().cpu().numpy() - rl).max() <= 1e-4
        assert (np.abs(got[0].double().cpu().numpy().T - rw) <= 1e-4 * rw + 1e-12).all()
        want_sums[:at + size] += rw
        at += size
        lens = after
    assert lens.tolist() == [at] == [510]
    budget, recent = 200, 120
    cache, lens, sums = switch_kv_cache_evict(cache, lens, sums, budget=budget, recent=recent, capacity=300)
    # Which rows stay: by the sums as computed, which the check above holds to the formula.
    heavy = np.argsort(-want_sums[:at - recent].T, axis=1, kind="stable")[:, :budget - recent]
    k = C.cache_values(cache.k, cache.k_scales, 32)[0]
    kept = sums[0, :, :budget].double().cpu().numpy()
    for h in range(hkv):
        rows = np.concatenate([np.sort(heavy[h]), np.arange(at - recent, at)])
        assert np.abs(kept[h] - want_sums[rows, h]).max() <= 2e-4 * want_sums.max()
        # Rounded again at most once, to a scale that the block's largest value needs.
        assert np.abs(k[:budget, h] - held_k[rows, h]).max() <= np.abs(held_k).max() * 2.0 ** -4
    full = torch.tensor([True], device=DEV)
    for i in range(steps):
        q, kn, vn = r(1, 1, hq, 128), r(1, 1, hkv, 128), r(1, 1, hkv, 128)
        lens = switch_kv_cache_append(cache, kn, vn, lens)
        before = sums.double().cpu().numpy()
        out, lse = switch_gqa_decode_quantized_forward(q, cache, lens, full, window_size=w, key_weights=sums)
        m = int(lens[0])
        assert m == budget + i + 1
        kk = C.cache_values(cache.k, cache.k_scales, 32)[0, :m]
        vv = C.cache_values(cache.v, cache.v_scales, 32)[0, :m]
        first = 0 if bool(full[0]) else m - w
        ro, rl, rw = _rows_attention(q[0].double().cpu().numpy(), kk, vv, np.array([first]), np.array([m]))
        assert np.abs(out[0].double().cpu().numpy() - ro).max() <= (2.0 ** -8 + 1e-4) * np.abs(vv).max()
        assert np.abs(lse[0].double().cpu().numpy() - rl).max() <= 1e-4
        assert np.abs(sums.double().cpu().numpy()[0, :, :m] - before[0, :, :m] - rw.T).max() <= 1e-4
        assert np.array_equal(sums.double().cpu().numpy()[0, :, m:], before[0, :, m:])
        full = ~full


@pytest.mark.parametrize("seed", range(24))
def test_random_cases(seed):
    """Random shapes, lengths, blocks and codes through append, read, decode and
    evict."""
    g = torch.Generator().manual_seed(1000 + seed)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=g))]  # noqa: E731
    rint = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    dtype, block = pick(torch.float8_e4m3fn, torch.int8), pick(16, 32, 64, 128)
    b, h, grp, n = rint(1, 9), pick(1, 2, 3, 8), rint(1, 8), rint(1, 700)
    print(f"seed {seed}: {dtype} block {block} B{b} Hkv{h} G{grp} L{n}", flush=True)
    raw = [torch.randint(0, 256, (b, n, h, 128), generator=g, dtype=torch.uint8) for _ in range(2)]
    cache = SwitchKVCache(*(x.to(DEV).view(dtype) for x in raw),
                          *(torch.full((b, h, -(-n // block)), math.nan, device=DEV) for _ in range(2)), block)
    lens = [0] * b
    for _ in range(rint(1, 4)):
        t = rint(0, n)
        counts = [rint(0, t) for _ in range(b)]
        size = 10.0 ** rint(-3, 3)
        k, v = ((torch.randn(b, t, h, 128, generator=g) * size).to(torch.bfloat16) for _ in range(2))
        was = cache.k.clone(), cache.k_scales.clone(), cache.v.clone(), cache.v_scales.clone()
        after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), _int32(lens), row_counts=_int32(counts))
        for codes, sc, old, old_sc, x in ((cache.k, cache.k_scales, was[0], was[1], k),
                                          (cache.v, cache.v_scales, was[2], was[3], v)):
            values, scales, ends = C.append(old, old_sc, block, [x[i, :counts[i]].float().numpy() for i in range(b)], lens)
            assert after.tolist() == ends
            got = C.cache_values(codes, sc, block)
            for i, end in enumerate(ends):
                assert np.array_equal(got[i, :end], values[i, :end])
                assert torch.equal(codes.view(torch.uint8)[i, end:], old.view(torch.uint8)[i, end:])
            assert np.array_equal(sc.cpu().numpy(), scales, equal_nan=True)
        lens = after.tolist()
    vals = [C.cache_values(c, s, block) for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]
    for i in range(b):
        for x in vals:
            x[i, lens[i]:] = 0.0
    rk, rv = switch_kv_cache_read(cache, 0, n, cache_lens=_int32(lens))
    assert np.array_equal(rk.double().cpu(), vals[0]) and np.array_equal(rv.double().cpu(), vals[1])
    # Decode, at a scale that keeps scores moderate whatever the keys' magnitude.
    q = torch.randn(b, 1, grp * h, 128, generator=g).to(torch.bfloat16)
    full = [bool(rint(0, 1)) for _ in range(b)]
    window, scale = rint(1, n + 5), 128 ** -0.5 / max(np.abs(vals[0]).max(), 1e-3)
    w = torch.rand(b, h, n, generator=g).to(DEV)
    before = w.double().cpu().numpy()
    o, lse = switch_gqa_decode_quantized_forward(q.to(DEV), cache, _int32(lens), torch.tensor(full, device=DEV),
                                                 window_size=window, sm_scale=scale, key_weights=w)
    ro, rl, rw, dots = C.decode(q[:, 0], vals[0], vals[1], lens, full, window, scale)
    ds = 130 * 2.0 ** -24 * dots
    eps = 2 * math.log(2) * ds + 2.0 ** -20          # as in test_gpu_cache.py
    live = np.array(lens) > 0
    go, gl = o[:, 0].double().cpu().numpy(), lse[:, 0].double().cpu().numpy()
    assert np.isnan(go[~live]).all() and np.isneginf(gl[~live]).all()
    if live.any():
        bound = 2.0 ** -8 * np.abs(ro[live]) + (eps + 2.0 ** -16) * np.abs(vals[1]).max()
        assert (np.abs(go[live] - ro[live]) <= bound).all()
        assert (np.abs(gl[live] - rl[live]) <= ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(rl[live])).all()
    got = w.double().cpu().numpy()
    assert (np.abs(got - before - rw) <= eps * rw + 2.0 ** -23 * (before + rw)).all()
    budget = rint(1, n)
    recent = rint(0, budget)
    out, after, ow = switch_kv_cache_evict(cache, _int32(lens), w, budget=budget, recent=recent, capacity=rint(budget, n))
    kept, ends, ek, ev, sk, sv, ew = C.evict(vals[0], vals[1], w.cpu().numpy(), lens, budget, recent, block, dtype)
    assert after.tolist() == ends
    for i, end in enumerate(ends):
        for codes, sc, want in ((out.k, out.k_scales, ek), (out.v, out.v_scales, ev)):
            assert np.array_equal(C.cache_values(codes, sc, block)[i, :end], want[i, :end])
        assert np.array_equal(ow[i, :, :end].cpu().numpy(), ew[i, :, :end].astype(np.float32)) and not ow[i, :, end:].any()
