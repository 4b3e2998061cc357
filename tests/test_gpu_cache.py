"""The 8-bit KV cache on the GPU: append, read, decode with attention sums,
eviction, against plain evaluations (``oracle/cache.py``).

Codes and scales are exact (power-of-two scales, one rounding to nearest), so
appended, read and evicted values are compared for equality.  The decode's
bounds are derived where they are used (``_bounds``).
"""

import math

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (SwitchKVCache, build_switch_kv_cache,
                                        switch_gqa_decode_quantized_forward,
                                        switch_kv_cache_append, switch_kv_cache_evict,
                                        switch_kv_cache_read)

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
DTYPES = [E4M3, INT8]


def _rows(gen, *shape, spread=1.0):
    x = torch.randn(*shape, generator=gen) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=gen))
    return x.to(torch.bfloat16)


def _garbage_cache(gen, b, n, h, dtype, block):
    """Every byte set: codes of NaN among them, scales NaN, infinite, negative."""
    raw = [torch.randint(0, 256, (b, n, h, 128), generator=gen, dtype=torch.uint8) for _ in range(2)]
    for r in raw:
        r[torch.rand(r.shape, generator=gen) < 0.2] = 0x7f
    bad = torch.tensor([math.nan, math.inf, -1.0, 3.0])
    sc = [bad[torch.randint(0, 4, (b, h, -(-n // block)), generator=gen)] for _ in range(2)]
    return SwitchKVCache(*(r.to(DEV).view(dtype) for r in raw), *(s.to(DEV) for s in sc), block)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _filled(gen, b, n, h, dtype, block, lens, spread=0.5):
    """A garbage cache with rows [0, lens[b]) appended."""
    cache = _garbage_cache(gen, b, n, h, dtype, block)
    t = max(max(lens), 0)
    k, v = _rows(gen, b, t, h, 128, spread=spread), _rows(gen, b, t, h, 128, spread=spread)
    after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), _int32([0] * b), row_counts=_int32(lens))
    assert after.tolist() == [min(max(x, 0), n) for x in lens]
    return cache


def _same(a, b):
    return np.array_equal(np.asarray(a), np.asarray(b), equal_nan=True)


def _check_append(cache, before, new_k, new_v, lens, after):
    """The whole cache against the oracle, bytes that may not change included."""
    for codes, scales, was, was_s, new in ((cache.k, cache.k_scales, *before[0], new_k),
                                           (cache.v, cache.v_scales, *before[1], new_v)):
        values, sc, ends = C.append(was, was_s, cache.block_size, new, lens)
        assert after.tolist() == ends
        got = C.cache_values(codes, scales, cache.block_size)
        for b, end in enumerate(ends):
            assert _same(got[b, :end], values[b, :end]), f"values of sequence {b}"
            assert torch.equal(codes.view(torch.uint8)[b, end:], was.view(torch.uint8)[b, end:])
        assert _same(scales.cpu(), sc), "scales"


def _snapshot(cache):
    return (cache.k.clone(), cache.k_scales.clone()), (cache.v.clone(), cache.v_scales.clone())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_padded_rows_and_tokens(dtype, block):
    """Chunks of any length at any place of a block, single tokens that make a
    block's scale grow, rows that no longer fit, lengths out of range."""
    gen = torch.Generator().manual_seed(block + (dtype == INT8))
    b, n, h = 7, 3 * block + 5, 3
    cache = _filled(gen, b, n, h, dtype, block, [0, 1, block, block - 1, n - 1, n, -4])
    lens = _int32([0, 1, block, block - 1, n - 1, n, -4])
    for t in (block + 3, 1, 1, 2, 17 % block + 1, 1):
        k, v = _rows(gen, b, t, h, 128, spread=1.5), _rows(gen, b, t, h, 128, spread=1.5)
        counts = torch.randint(0, t + 1, (b,), generator=gen, dtype=torch.int32) if t > 1 else None
        before = _snapshot(cache)
        was = lens.clone()
        after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), lens,
                                       row_counts=None if counts is None else counts.to(DEV))
        assert torch.equal(lens, was)
        take = [t] * b if counts is None else counts.tolist()
        _check_append(cache, before, [k[i, :take[i]].float().numpy() for i in range(b)],
                      [v[i, :take[i]].float().numpy() for i in range(b)], lens.tolist(), after)
        lens = after


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_packed(dtype):
    gen = torch.Generator().manual_seed(5)
    n, h, block = 300, 2, 32
    cu = [0, 130, 130, 131, 300, 447]      # an empty sequence, one token, one that overflows
    cache = _garbage_cache(gen, 5, n, h, dtype, block)
    lens = _int32([0, 7, 33, 31, 200])
    # Rows that the first calls' lengths count must exist.
    fill = _rows(gen, 5, 200, h, 128)
    switch_kv_cache_append(cache, fill.to(DEV), fill.to(DEV), _int32([0] * 5), row_counts=lens)
    k, v = _rows(gen, 1, cu[-1], h, 128), _rows(gen, 1, cu[-1], h, 128)
    for as_tensor in (False, True):
        before = _snapshot(cache)
        after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), lens,
                                       cu_seqlens=torch.tensor(cu) if as_tensor else cu)
        part = lambda x: [x[0, a:b].float().numpy() for a, b in zip(cu, cu[1:])]  # noqa: E731
        _check_append(cache, before, part(k), part(v), lens.tolist(), after)


def test_append_packed_many_sequences():
    """More sequences than offsets travel as kernel arguments."""
    gen = torch.Generator().manual_seed(15)
    b, n, h, block = 300, 20, 1, 16
    counts = torch.randint(0, 6, (b,), generator=gen).tolist()
    lens = torch.randint(0, 18, (b,), generator=gen).tolist()
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    for m in (256, 257, 300):
        cache = _filled(gen, m, n, h, E4M3, block, lens[:m])
        k = _rows(gen, 1, cu[m], h, 128)
        before = _snapshot(cache)
        after = switch_kv_cache_append(cache, k.to(DEV), (-k).to(DEV), _int32(lens[:m]), cu_seqlens=cu[:m + 1])
        part = [k[0, x:y].float().numpy() for x, y in zip(cu[:m], cu[1:m + 1])]
        _check_append(cache, before, part, [-x for x in part], lens[:m], after)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_non_finite_value_makes_its_block_nan(dtype, bad):
    gen = torch.Generator().manual_seed(9)
    b, n, h, block = 2, 100, 2, 32
    cache = _garbage_cache(gen, b, n, h, dtype, block)
    lens = _int32([0, 40])
    switch_kv_cache_append(cache, *(_rows(gen, b, 40, h, 128).to(DEV) for _ in range(2)), _int32([0, 0]))
    k, v = _rows(gen, b, 50, h, 128), _rows(gen, b, 50, h, 128)
    k[0, 40, 1, 3] = bad          # sequence 0, row 40 (block 1), head 1
    v[1, 0, 0, 127] = bad         # sequence 1, row 40 (block 1, begun), head 0
    before = _snapshot(cache)
    after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), lens)
    _check_append(cache, before, list(k.float().numpy()), list(v.float().numpy()), lens.tolist(), after)
    rk, rv = switch_kv_cache_read(cache, 0, n, cache_lens=after)
    assert torch.isnan(rk[0, 32:50, 1]).all() and torch.isnan(rk).sum() == 18 * 128
    assert torch.isnan(rv[1, 32:64, 0]).all() and torch.isnan(rv).sum() == 32 * 128
    # One more token leaves the block as it is.
    one = _rows(gen, b, 1, h, 128).to(DEV)
    switch_kv_cache_append(cache, one, one, _int32([50, 60]))
    rk2, rv2 = switch_kv_cache_read(cache, 0, n, cache_lens=_int32([51, 61]))
    assert torch.isnan(rk2[0, 32:51, 1]).all() and torch.isnan(rv2[1, 32:61, 0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_extremes_and_zeros(dtype):
    """Zeros, subnormals, the largest bf16 numbers, values at rounding ties."""
    x = torch.zeros(1, 6, 1, 128)
    x[0, 1] = torch.finfo(torch.bfloat16).max
    x[0, 2] = 1e-40
    x[0, 3] = torch.linspace(-448, 448, 128)
    x[0, 4] = torch.arange(128) + 0.5
    x[0, 5] = 2.0 ** -103
    x = x.to(torch.bfloat16)
    for rows in ([0], [1], [2], [3], [4], [5], [0, 2], [3, 4], [2, 5], [0, 1, 2, 3]):
        cache = build_switch_kv_cache(1, 20, 1, device=DEV, dtype=dtype, block_size=16)
        before = _snapshot(cache)
        part = x[:, rows].contiguous()
        after = switch_kv_cache_append(cache, part.to(DEV), (-part).to(DEV), _int32([0]))
        (bk, bks), (bv, bvs) = before
        for codes, scales, was, was_s, new in ((cache.k, cache.k_scales, bk, bks, part),
                                               (cache.v, cache.v_scales, bv, bvs, -part)):
            values, sc, _ = C.append(was, was_s, 16, [new[0].float().numpy()], [0])
            got = C.cache_values(codes, scales, 16)
            assert _same(got[0, :len(rows)], values[0, :len(rows)]), rows
            assert float(scales[0, 0, 0]) == sc[0, 0, 0]
        assert after.tolist() == [len(rows)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_to_scales_made_elsewhere(dtype):
    """A begun block whose scale is no power of two, and larger or smaller than
    what the new rows need."""
    gen = torch.Generator().manual_seed(3)
    for size in (0.01, 30.0):
        cache = _filled(gen, 1, 64, 2, dtype, 32, [40])
        cache.k_scales.mul_(1.3)
        cache.v_scales.mul_(0.7)
        k = (_rows(gen, 1, 3, 2, 128) * size).to(torch.bfloat16)
        before = _snapshot(cache)
        after = switch_kv_cache_append(cache, k.to(DEV), (-k).to(DEV), _int32([40]))
        _check_append(cache, before, [k[0].float().numpy()], [-k[0].float().numpy()], [40], after)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 128])
def test_read_ranges(dtype, block):
    gen = torch.Generator().manual_seed(11)
    b, n, h = 5, 201, 3
    lens = [201, 0, 64, 130, 1]
    cache = _filled(gen, b, n, h, dtype, block, lens)
    for starts, rows, use_lens in (([0, 0, 0, 0, 0], 201, True), ([3, 100, 63, 129, 0], 77, True),
                                   ([-2, -500, 2 ** 31 - 1, 5, 0], 9, True), ([200, 0, 50, 100, 0], 1, True),
                                   ([0, 0, 0, 0, 0], 0, True)):
        ln = _int32(lens) if use_lens else None
        k, v = switch_kv_cache_read(cache, _int32(starts), rows, cache_lens=ln)
        for got, codes, sc in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
            assert _same(got.double().cpu(), C.read(codes, sc, block, starts, rows, lens))
    full = _filled(gen, b, n, h, dtype, block, [n] * b)
    k, _ = switch_kv_cache_read(full, 7, n)
    assert _same(k.double().cpu(), C.read(full.k, full.k_scales, block, [7] * b, n))


# ---------------------------------------------------------------------------
# Decode
# ---------------------------------------------------------------------------
def _bounds(dots, out, v_max):
    """A score is a sum of 128 exact products in fp32, scaled twice: off by at most
    130 * 2^-24 * sum |q_i k_i| c (`dots`), in log2 units; the weight by that times
    ln 2, twice (its score's and the LSE's), and 2^-20 for exp2, the sums and the
    merges.  p enters the product with V as two bf16 halves, 2^-17.  O is then
    rounded to bf16, 2^-8 relative."""
    ds = 130 * 2.0 ** -24 * dots
    eps = 2 * math.log(2) * ds + 2.0 ** -20
    return ds + 2.0 ** -20, eps, 2.0 ** -8 * np.abs(out) + (eps + 2.0 ** -16) * v_max + 1e-30


def _check_decode(cache, q, lens, full, window, weights, sm_scale=None):
    before = None if weights is None else weights.clone()
    o, lse = switch_gqa_decode_quantized_forward(q, cache, _int32(lens), torch.tensor(full, device=DEV),
                                                 window_size=window, sm_scale=sm_scale, key_weights=weights)
    k = C.cache_values(cache.k, cache.k_scales, cache.block_size)
    v = C.cache_values(cache.v, cache.v_scales, cache.block_size)
    ro, rl, rw, dots = C.decode(q[:, 0].cpu(), k, v, lens, full, window, sm_scale)
    live = [i for i, n in enumerate(lens) if n > 0]
    v_max = max([np.nanmax(np.abs(v[i, :lens[i]])) for i in live], default=1.0)
    d_lse, eps, d_o = _bounds(dots, ro, v_max)
    go, gl = o[:, 0].double().cpu().numpy(), lse[:, 0].double().cpu().numpy()
    for i in range(len(lens)):
        if i not in live:
            assert np.isnan(go[i]).all() and (gl[i] == -math.inf).all()
            continue
        assert np.array_equal(np.isnan(go[i]), np.isnan(ro[i]))
        ok = ~np.isnan(ro[i])
        assert (np.abs(go[i] - ro[i])[ok] <= d_o[i][ok]).all(), \
            (i, np.nanmax(np.abs(go[i] - ro[i])), np.nanmax(d_o[i]))
        assert np.array_equal(np.isnan(gl[i]), np.isnan(rl[i]))
        if not np.isnan(rl[i]).any():
            assert (np.abs(gl[i] - rl[i]) <= d_lse + 2.0 ** -22 * np.abs(rl[i])).all()
    if weights is not None:
        got, was = weights.double().cpu().numpy(), before.double().cpu().numpy()
        want = was + rw
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= (eps * rw + 2.0 ** -23 * np.abs(want) + 1e-30)[ok]).all()
        untouched = rw == 0
        assert torch.equal(weights.cpu()[torch.from_numpy(untouched)], before.cpu()[torch.from_numpy(untouched)])


def _q(gen, b, hq):
    return torch.randn(b, 1, hq, 128, generator=gen).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_decode_groups(dtype, group):
    """Every group size, lengths at the ends of steps and blocks, garbage behind."""
    gen = torch.Generator().manual_seed(group)
    n, h, block = 467, 2, [16, 32, 64, 128][group % 4]
    lens = [467, 1, 0, 31, 32, 33, 128, 129, 300, 16]
    full = [True, False, True, True, False, True, False, False, True, False]
    cache = _filled(gen, len(lens), n, h, dtype, block, lens)
    w = torch.rand(len(lens), h, n, generator=gen).to(DEV)
    _check_decode(cache, _q(gen, len(lens), group * h), lens, full, 100, w)
    _check_decode(cache, _q(gen, len(lens), group * h), lens, full, 1, w)
    _check_decode(cache, _q(gen, len(lens), group * h), lens, full, 2 ** 32 + 1, None)


@pytest.mark.parametrize("dtype,batch,n,hq,hkv,window,p,weights", [
    (E4M3, 1, 4096, 32, 8, 1024, 1.0, True),
    (INT8, 1, 1, 8, 2, 7, 1.0, True),
    (E4M3, 3, 2500, 40, 8, 333, 0.5, True),
    (INT8, 24, 700, 4, 1, 256, 0.25, True),
    (E4M3, 2, 9001, 16, 2, 5000, 0.0, False),
    (INT8, 70, 1500, 8, 2, 64, 0.1, True),
])
def test_decode_shapes(dtype, batch, n, hq, hkv, window, p, weights):
    gen = torch.Generator().manual_seed(n)
    lens = torch.randint(0, n + 1, (batch,), generator=gen).tolist()
    lens[0] = n
    full = (torch.rand(batch, generator=gen) < p).tolist()
    cache = _filled(gen, batch, n, hkv, dtype, 64, lens)
    w = torch.zeros(batch, hkv, n, device=DEV) if weights else None
    _check_decode(cache, _q(gen, batch, hq), lens, full, window, w, sm_scale=0.11 if batch == 3 else None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_many_sequences(dtype):
    """More sequences than a workgroup plans for itself."""
    gen = torch.Generator().manual_seed(77)
    batch, n = 1100, 60
    lens = torch.randint(0, n + 1, (batch,), generator=gen).tolist()
    full = (torch.rand(batch, generator=gen) < 0.5).tolist()
    cache = _filled(gen, batch, n, 1, dtype, 16, lens)
    w = torch.zeros(batch, 1, n, device=DEV)
    _check_decode(cache, _q(gen, batch, 2), lens, full, 20, w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_lengths_out_of_range_and_strided_arguments(dtype):
    gen = torch.Generator().manual_seed(6)
    lens = [90, 17, 44]
    cache = _filled(gen, 3, 90, 2, dtype, 32, lens)
    q = _q(gen, 3, 4)
    full = torch.tensor([True, False, True], device=DEV)
    want = switch_gqa_decode_quantized_forward(q, cache, _int32(lens), full, window_size=9)
    over = torch.stack([_int32([1000, 17, 44]), _int32([0, 0, 0])], dim=1)[:, 0]
    strided = torch.stack([full, ~full], dim=1)[:, 0]
    got = switch_gqa_decode_quantized_forward(q[:, 0], cache, over, strided, window_size=9)
    assert got[0].shape == (3, 4, 128) and got[1].shape == (3, 4)
    assert torch.equal(got[0], want[0][:, 0]) and torch.equal(got[1], want[1][:, 0])
    o, lse = switch_gqa_decode_quantized_forward(q, cache, _int32([-5, 17, 0]), full, window_size=9)
    assert torch.isnan(o[0]).all() and torch.isneginf(lse[2]).all() and torch.equal(o[1], want[0][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_nan_blocks_show(dtype):
    """A NaN block makes the rows that attend it NaN, in one split of many too, and
    no others."""
    gen = torch.Generator().manual_seed(8)
    n, h = 3000, 2
    lens = [3000, 3000, 2000, 2990]
    cache = _filled(gen, 4, n, h, dtype, 64, lens)
    cache.k_scales[0, 0, 3] = math.nan       # full, head 0: NaN
    cache.v_scales[1, 1, 40] = math.nan      # local, outside of its window: not seen
    cache.v_scales[2, 1, 31] = math.nan      # its last block
    cache.k_scales[3, 0, 46:] = math.nan     # every block in its window
    w = torch.zeros(4, h, n, device=DEV)
    full = [True, False, True, False]
    o, lse = switch_gqa_decode_quantized_forward(_q(gen, 4, 8), cache, _int32(lens),
                                                 torch.tensor(full, device=DEV), window_size=40,
                                                 key_weights=w)
    nan = torch.isnan(o[:, 0]).view(4, h, 4, 128).all(3).all(2).cpu()
    assert nan.tolist() == [[True, False], [False, False], [False, True], [True, False]]
    assert torch.isnan(o[:, 0]).view(4, h, -1).any(2).cpu().equal(nan)
    lse_nan = torch.isnan(lse[:, 0]).view(4, h, 4).cpu()
    assert lse_nan[0, 0].all() and lse_nan[3, 0].all() and lse_nan.sum() == 8
    assert torch.isnan(w[0, 0]).all() and torch.isnan(w[2]).sum() == 0


def test_decode_nan_codes_and_queries_stay_where_they_are():
    """A NaN code of a cache made elsewhere: a key's in its head's rows, a value's in
    its dimension; a NaN or infinite query in its own row."""
    gen = torch.Generator().manual_seed(28)
    n, h, grp = 300, 2, 4
    cache = _filled(gen, 2, n, h, E4M3, 32, [300, 300])
    q = _q(gen, 2, h * grp)
    full = torch.tensor([True, True], device=DEV)
    clean, clean_lse = switch_gqa_decode_quantized_forward(q, cache, _int32([300, 300]), full)
    keep = cache.v[0, 7, 1, 5].clone().view(torch.uint8)
    cache.v.view(torch.uint8)[0, 7, 1, 5] = 0x7f
    o, lse = switch_gqa_decode_quantized_forward(q, cache, _int32([300, 300]), full)
    assert torch.isnan(o[0, 0, grp:, 5]).all() and torch.isnan(o).sum() == grp and torch.equal(lse, clean_lse)
    cache.v.view(torch.uint8)[0, 7, 1, 5] = keep
    cache.k.view(torch.uint8)[1, 299, 0, 127] = 0xff
    o, lse = switch_gqa_decode_quantized_forward(q, cache, _int32([300, 300]), full)
    assert torch.isnan(o[1, 0, :grp]).all() and torch.isnan(lse).sum() == grp
    assert torch.equal(o[0], clean[0]) and torch.equal(o[1, 0, grp:], clean[1, 0, grp:])
    o, lse = switch_gqa_decode_quantized_forward(q, cache, _int32([300, 299]), full)   # behind the end
    assert not torch.isnan(o).any() and not torch.isnan(lse).any()
    for bad in (math.nan, math.inf):
        q2 = q.clone()
        q2[0, 0, 2, 9] = bad
        w = torch.zeros(2, h, n, device=DEV)
        o, lse = switch_gqa_decode_quantized_forward(q2, cache, _int32([300, 299]), full, key_weights=w)
        others = torch.ones(h * grp, dtype=torch.bool, device=DEV)
        others[2] = False
        assert torch.isnan(o[0, 0, 2]).all() and torch.equal(o[0, 0, others], clean[0, 0, others])
        assert not torch.isnan(o[1]).any() and not torch.isnan(w[0, 1]).any() and not torch.isnan(w[1]).any()
    values, _ = switch_kv_cache_read(cache, 0, n)
    assert torch.isnan(values[1, 299, 0, 127]) and torch.isnan(values).sum() == 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_score_jumps_and_large_scales(dtype):
    """Running maxima that move many times, far apart, and caches whose values are
    very large or small."""
    gen = torch.Generator().manual_seed(12)
    n, h = 1500, 1
    k = torch.randn(1, n, h, 128, generator=gen) * torch.linspace(0.01, 6, n)[None, :, None, None]
    v = torch.randn(1, n, h, 128, generator=gen) * 1e-20
    for flip in (False, True):
        cache = build_switch_kv_cache(1, n, h, device=DEV, dtype=dtype, block_size=16)
        kk = (k.flip(1) if flip else k).contiguous().to(torch.bfloat16)
        switch_kv_cache_append(cache, kk.to(DEV), v.to(torch.bfloat16).to(DEV), _int32([0]))
        _check_decode(cache, _q(gen, 1, 8), [n], [True], 5, torch.zeros(1, h, n, device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(dtype):
    """A cache of more than 2^32 bytes per tensor: its last rows."""
    n, h, block = 4_300_000, 8, 64
    cache = build_switch_kv_cache(1, n, h, device=DEV, dtype=dtype, block_size=block)
    gen = torch.Generator().manual_seed(1)
    t = 200
    k, v = _rows(gen, 1, t, h, 128), _rows(gen, 1, t, h, 128)
    start = n - t - 3                     # no multiple of a block
    start -= start % block                # rows before it must be valid or absent: begin a block
    after = switch_kv_cache_append(cache, k.to(DEV), v.to(DEV), _int32([start]))
    assert after.tolist() == [start + t]
    rk, rv = switch_kv_cache_read(cache, _int32([start]), t + 5, cache_lens=after)
    small = build_switch_kv_cache(1, t, h, device=DEV, dtype=dtype, block_size=block)
    switch_kv_cache_append(small, k.to(DEV), v.to(DEV), _int32([0]))
    sk, sv = switch_kv_cache_read(small, 0, t)
    assert torch.equal(rk[:, :t], sk) and torch.equal(rv[:, :t], sv) and not rk[:, t:].any()
    q = _q(gen, 1, 32)
    local = torch.tensor([False], device=DEV)
    w = torch.zeros(1, h, n, device=DEV)
    got = switch_gqa_decode_quantized_forward(q, cache, after, local, window_size=t, key_weights=w)
    ws = torch.zeros(1, h, t, device=DEV)
    want = switch_gqa_decode_quantized_forward(q, small, _int32([t]), local, window_size=t, key_weights=ws)
    assert torch.allclose(got[1], want[1], rtol=0, atol=2.0 ** -18)
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0 ** -7, atol=2.0 ** -12)
    assert torch.allclose(w[:, :, start:start + t], ws, rtol=2.0 ** -16, atol=0) and not w[:, :, :start].any()


# ---------------------------------------------------------------------------
# Evict
# ---------------------------------------------------------------------------
def _check_evict(cache, lens, w, budget, recent, **kw):
    out, after, ow = switch_kv_cache_evict(cache, _int32(lens), w, budget=budget, recent=recent, **kw)
    block = cache.block_size
    k = C.cache_values(cache.k, cache.k_scales, block)
    v = C.cache_values(cache.v, cache.v_scales, block)
    kept, ends, rk, rv, sk, sv, rw = C.evict(k, v, w.cpu().numpy(), lens, budget, recent, block,
                                             cache.k.dtype)
    assert after.tolist() == ends
    gk, gv = (C.cache_values(c, s, block) for c, s in ((out.k, out.k_scales), (out.v, out.v_scales)))
    for b, end in enumerate(ends):
        assert _same(gk[b, :end], rk[b, :end]) and _same(gv[b, :end], rv[b, :end]), b
        nb = -(-end // block)
        assert _same(out.k_scales[b, :, :nb].double().cpu(), sk[b, :, :nb])
        assert _same(out.v_scales[b, :, :nb].double().cpu(), sv[b, :, :nb])
        assert _same(ow[b, :, :end].cpu(), rw[b, :, :end].astype(np.float32))
        assert not ow[b, :, end:].any()
    return out, after, ow


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_evict_budgets(dtype, block):
    gen = torch.Generator().manual_seed(block)
    n, h = 333, 3
    lens = [333, 0, 100, 101, 1, 332, 99]
    cache = _filled(gen, len(lens), n, h, dtype, block, lens)
    w = torch.exp(2 * torch.randn(len(lens), h, n, generator=gen)).to(DEV)
    for budget, recent in ((100, 0), (100, 100), (100, 31), (1, 0), (1, 1), (333, 5), (64, 63), (129, 17)):
        before = _snapshot(cache)
        _check_evict(cache, lens, w, budget, recent, capacity=budget)
        assert all(torch.equal(a.view(torch.uint8), c.view(torch.uint8)) for pair, now in
                   zip(before, _snapshot(cache)) for a, c in zip(pair, now)), "the source is left as it is"
    _check_evict(cache, lens, w, 50, 20)                       # destination of the same capacity
    _check_evict(cache, lens, w, 50, 20, capacity=1001)        # and a larger one


@pytest.mark.parametrize("kind", ["equal", "zeros", "signed zeros", "two values", "nan", "negative", "inf"])
def test_evict_ties_and_odd_weights(kind):
    """Equal weights keep the lower rows; NaN counts as largest; -0 equals 0."""
    gen = torch.Generator().manual_seed(2)
    n, h = 9001, 2
    lens = [9001, 5000, 4097]
    cache = _filled(gen, 3, n, h, INT8, 128, lens)
    w = torch.rand(3, h, n, generator=gen)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "zeros":
        w.zero_()
    elif kind == "signed zeros":
        w = torch.where(w < 0.5, 0.0, -0.0)
    elif kind == "two values":
        w = torch.where(w < 0.3, 1.0, 2.0)
    elif kind == "nan":
        w[w < 0.1] = math.nan
        w[0, 0, 7] = -math.nan
    elif kind == "negative":
        w = torch.round((w - 0.5) * 50)
    else:
        w[w < 0.2] = math.inf
        w[w > 0.9] = -math.inf
        w[(w > 0.5) & (w < 0.6)] = 1e-42
    _check_evict(cache, lens, w.to(DEV), 4097, 100, capacity=4100)
    _check_evict(cache, lens, w.to(DEV), 700, 0, capacity=700)


@pytest.mark.parametrize("n,budget,recent", [(16385, 4000, 1000), (32768, 32767, 3), (32768, 1, 0),
                                             (50001, 20000, 64), (70000, 300, 299)])
def test_evict_long_caches(n, budget, recent):
    """Every way of holding the weights during the search; equal ones among them."""
    gen = torch.Generator().manual_seed(n)
    lens = [n, n - 1, budget + 1]
    cache = _filled(gen, 3, n, 1, INT8, 128, lens)
    w = torch.exp(2 * torch.randn(3, 1, n, generator=gen))
    w[1] = torch.round(w[1])
    _check_evict(cache, lens, w.to(DEV), budget, recent, capacity=budget)


@pytest.mark.parametrize("bits", [1, 10, 21, 31])
def test_evict_weights_that_differ_in_their_last_bits(bits):
    """The search ends after one, two or all three digits of a weight."""
    gen = torch.Generator().manual_seed(bits)
    cache = _filled(gen, 2, 3000, 2, INT8, 64, [3000, 1500])
    low = torch.randint(0, 2 ** bits, (2, 2, 3000), generator=gen)
    w = ((0x3f800000 if bits < 23 else 0) + low).clamp_max(0x7f800000).to(torch.int32).view(torch.float32)
    for budget in (1, 777, 1499):
        _check_evict(cache, [3000, 1500], w.to(DEV), budget, 0, capacity=1500)


@pytest.mark.parametrize("dtype", DTYPES)
def test_evict_carries_nan_blocks_and_foreign_scales(dtype):
    gen = torch.Generator().manual_seed(4)
    cache = _filled(gen, 1, 256, 1, dtype, 32, [256])
    cache.k_scales.mul_(1.7)
    cache.v_scales[0, 0, 2] = math.nan
    _check_evict(cache, [256], torch.rand(1, 1, 256, generator=gen).to(DEV), 100, 10)


def test_evict_into_a_given_cache_and_lengths_out_of_range():
    gen = torch.Generator().manual_seed(14)
    cache = _filled(gen, 3, 120, 2, E4M3, 32, [120, 60, 30])
    w = torch.rand(3, 2, 120, generator=gen).to(DEV)
    out, ow = build_switch_kv_cache(3, 77, 2, device=DEV, block_size=32), torch.empty(3, 2, 77, device=DEV)
    got, after, gw = _check_evict(cache, [120, 60, 30], w, 50, 10, out=out, out_weights=ow)
    assert got is out and gw is ow
    a, la, wa = switch_kv_cache_evict(cache, _int32([999, 60, -1]), w, budget=50, recent=10)
    assert la.tolist() == [50, 50, 0] and torch.equal(wa[:2, :, :50], ow[:2, :, :50]) and not wa[2].any()
    assert torch.equal(a.k.view(torch.uint8)[:2, :50], out.k.view(torch.uint8)[:2, :50])


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_calls_equal_their_parts(dtype):
    """Reads and evictions of 250 to 400 MB against the same in parts of less than 100."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    b, n, h, block = 4, 16000, 8, 32
    codes = [torch.randint(0, 0x7f, (b, n, h, 128), generator=gen, device=DEV, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.rand(b, h, n // block, generator=gen, device=DEV) + 0.5 for _ in range(2)]
    cache = SwitchKVCache(*(x.view(dtype) for x in codes), *scales, block)
    lens = _int32([16000, 15990, 15001, 300])
    whole = switch_kv_cache_read(cache, 0, n, cache_lens=lens)
    for a in range(0, n, 4000):
        for x, y in zip(whole, switch_kv_cache_read(cache, a, 4000, cache_lens=lens)):
            assert torch.equal(x[:, a:a + 4000], y)
    weights = torch.rand(b, h, n, generator=gen, device=DEV)
    kept, after, w = switch_kv_cache_evict(cache, lens, weights, budget=15000, recent=100, capacity=15010)
    for i in range(b):
        one = SwitchKVCache(*(x[i:i + 1] for x in (cache.k, cache.v, cache.k_scales, cache.v_scales)), block)
        k1, a1, w1 = switch_kv_cache_evict(one, lens[i:i + 1], weights[i:i + 1], budget=15000, recent=100,
                                           capacity=15010)
        m = int(a1[0])
        assert m == min(int(lens[i]), 15000) == int(after[i]) and torch.equal(w[i], w1[0])
        for x, y in ((kept.k, k1.k), (kept.v, k1.v)):
            assert torch.equal(x.view(torch.uint8)[i, :m], y.view(torch.uint8)[0, :m])
        nb = -(-m // block)
        assert torch.equal(kept.k_scales[i, :, :nb], k1.k_scales[0, :, :nb])
        assert torch.equal(kept.v_scales[i, :, :nb], k1.v_scales[0, :, :nb])


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_31_bits(dtype):
    """A cache of 2 x 2.2 GB: its last rows against those of a small cache, and keys of
    zeros before them, whose scores are 0 and whose values add nothing."""
    gen = torch.Generator().manual_seed(9)
    n, h, block, hq = 2_150_003, 8, 64, 8
    at = n - 500
    base = (at - 100) // block * block        # the small cache holds rows [base, n)
    big = build_switch_kv_cache(1, n, h, device=DEV, dtype=dtype, block_size=block)
    small = build_switch_kv_cache(1, n - base, h, device=DEV, dtype=dtype, block_size=block)
    for c in (big, small):
        for x in (c.k, c.v):
            x.view(torch.uint8).zero_()
        c.k_scales.fill_(2.0 ** -100)
        c.v_scales.fill_(2.0 ** -100)
    k, v = _rows(gen, 1, 480, h, 128).to(DEV), _rows(gen, 1, 480, h, 128).to(DEV)
    lb, ls = (switch_kv_cache_append(c, k, v, _int32([x])) for c, x in ((big, at), (small, at - base)))
    assert lb.tolist() == [at + 480] and ls.tolist() == [at + 480 - base]
    rb = switch_kv_cache_read(big, base, n - base, cache_lens=lb)
    rs = switch_kv_cache_read(small, 0, n - base, cache_lens=ls)
    assert all(torch.equal(x, y) for x, y in zip(rb, rs)) and rb[0][0, at - base:at - base + 480].any()
    # A window inside the small cache: both are within the bounds of the same values.
    q = _q(gen, 1, hq)
    full = torch.tensor([False], device=DEV)
    _check_decode(small, q, ls.tolist(), [False], 490, None)
    ob, eb = switch_gqa_decode_quantized_forward(q, big, lb, full, window_size=490)
    os_, es = switch_gqa_decode_quantized_forward(q, small, ls, full, window_size=490)
    assert (ob.float() - os_.float()).abs().max() <= 2 * 2.0 ** -8 * v.float().abs().max()
    assert (eb - es).abs().max() <= 1e-4
    # All keys: `at` scores of 0 beside the others'.
    sums = torch.zeros(1, h, n, device=DEV)
    ob, eb = switch_gqa_decode_quantized_forward(q, big, lb, ~full, key_weights=sums)
    kk, vv = (x[0, at - base:at - base + 480].double().cpu() for x in rs)
    sc = (q[0, 0].double().cpu()[:, None] * kk.transpose(0, 1)).sum(-1) * 128 ** -0.5
    total = at + sc.exp().sum(-1)
    assert (eb[0, 0].double().cpu() - total.log2()).abs().max() <= 1e-4
    want = (sc.exp() / total[:, None])[:, None] @ vv.transpose(0, 1)
    # P's two bf16 halves keep 16 bits: far below the output's own rounding.
    assert ((ob[0, 0].double().cpu() - want[:, 0]).abs() <= 2.0 ** -8 * want[:, 0].abs() + 1e-4 * want.abs().max()).all()
    ws = sums[0].double().cpu()
    assert (ws[:, at:at + 480] * total[:, None] / sc.exp() - 1).abs().max() <= 1e-4
    assert (ws[:, :at] * total[:, None] - 1).abs().max() <= 1e-4 and not ws[:, at + 480:].any()
    # The heaviest rows are the last ones and a few zeros before them.
    weights = torch.zeros(1, h, n, device=DEV)
    weights[:, :, 5], weights[:, :, at + 3], weights[:, :, at + 77] = 3.0, 2.0, 1.0
    kept, lk, wk = switch_kv_cache_evict(big, lb, weights, budget=103, recent=100, capacity=128)
    gk = switch_kv_cache_read(kept, 0, 103)
    rows = [0, at + 3 - base, at + 77 - base] + list(range(at + 380 - base, at + 480 - base))
    assert lk.tolist() == [103] and wk[0, :, :3].tolist() == [[3.0, 2.0, 1.0]] * h and not wk[0, :, 3:].any()
    for got, was in zip(gk, rs):
        x = was[0, rows].float()
        x[0] = 0
        # Rounded to the scale of the largest value of its block at most once more.
        step = 2.0 ** -4 * x.abs() + 2.0 ** -9 * x.abs().amax() if dtype == E4M3 else 2.0 ** -6 * x.abs().amax()
        assert ((got[0].float() - x).abs() <= step).all() and not got[0, 0].any()


# ---------------------------------------------------------------------------
# As a program uses them
# ---------------------------------------------------------------------------
def _serve(dtype, steps, gen_seed, graph):
    """Prompt, then tokens with sums, evicting in turn between two caches."""
    g = torch.Generator(device=DEV).manual_seed(gen_seed)
    b, n, h, hq, w = 4, 300, 2, 8, 50
    cache = build_switch_kv_cache(b, n, h, device=DEV, dtype=dtype, block_size=32)
    sums = torch.zeros(b, h, n, device=DEV)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    prompt = rnd(b, 200, h, 128), rnd(b, 200, h, 128)
    lens = switch_kv_cache_append(cache, *prompt, _int32([0] * b), row_counts=_int32([200, 7, 64, 0]))
    k, v, q = rnd(b, 1, h, 128), rnd(b, 1, h, 128), rnd(b, 1, hq, 128)
    full = torch.tensor([True, False, True, False], device=DEV)

    def step():
        after = switch_kv_cache_append(cache, k, v, lens)
        out = switch_gqa_decode_quantized_forward(q, cache, after, full, window_size=w, key_weights=sums)
        lens.copy_(after)
        return out

    if graph:
        state = [t.clone() for t in (lens, sums, cache.k_scales, cache.v_scales)]
        codes = cache.k.clone(), cache.v.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            held = step()
        for t, was in zip((lens, sums, cache.k_scales, cache.v_scales), state):
            t.copy_(was)
        for t, was in zip((cache.k, cache.v), codes):
            t.view(torch.uint8).copy_(was.view(torch.uint8))
    outs = []
    for i in range(steps):
        for t in (k, v, q):
            t.copy_(rnd(*t.shape))
        if graph:
            captured.replay()
            outs.append([t.clone() for t in held])
        else:
            outs.append(step())
        if i % 4 == 3:   # evict eagerly between steps and copy back under the captured pointers
            kept, after, ws = switch_kv_cache_evict(cache, lens, sums, budget=100, recent=50)
            cache.k.view(torch.uint8).copy_(kept.k.view(torch.uint8))
            cache.v.view(torch.uint8).copy_(kept.v.view(torch.uint8))
            cache.k_scales.copy_(kept.k_scales)
            cache.v_scales.copy_(kept.v_scales)
            sums.copy_(ws)
            lens.copy_(after)
    torch.cuda.synchronize()
    return outs, lens, sums


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_steps_equal_eager_ones(dtype):
    eager, lens_e, sums_e = _serve(dtype, 9, 21, False)
    graph, lens_g, sums_g = _serve(dtype, 9, 21, True)
    assert lens_e.tolist() == lens_g.tolist() == [101, 16, 73, 9]
    assert torch.equal(sums_e, sums_g)
    for (oe, le), (og, lg) in zip(eager, graph):
        assert torch.equal(oe, og) and torch.equal(le, lg)


def test_two_streams_match_sequential():
    want = [_serve(E4M3, 5, s, False) for s in (31, 32)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for st, seed in zip(streams, (31, 32)):
        with torch.cuda.stream(st):
            got.append(_serve(E4M3, 5, seed, False))
    torch.cuda.synchronize()
    for (oa, la, sa), (ob, lb, sb) in zip(want, got):
        assert torch.equal(sa, sb) and la.tolist() == lb.tolist()
        for x, y in zip(oa, ob):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
