"""The largest bf16 numbers in an 8-bit cache: finite values read back as finite ones.

bf16 ends at 255 * 2^120.  Its largest numbers need a scale of 2^120 (e4m3, qmax 448) or
2^122 (int8, qmax 127), and the code nearest to them, 256 or 64, would stand for 2^128,
an infinity in fp32 and bf16.  The largest code below is 240 or 63: off by 15 / 255 at most.
"""

import math

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (build_switch_kv_cache, switch_gqa_decode_quantized_forward,
                                        switch_kv_cache_append, switch_kv_cache_evict,
                                        switch_kv_cache_read)

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 240 * 2.0 ** 120, INT8: 63 * 2.0 ** 122}


def _int32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _append(cache, x, at):
    x = x.to(DEV)
    return switch_kv_cache_append(cache, x, -x, _int32(at))


def _near(got, x, dtype):
    """Within half a step of the code, or TOP for what lies nearer to 2^128."""
    got, x = got.double().cpu(), x.double()
    assert torch.isfinite(got).all()
    half = 2.0 ** -4 * x.abs() if dtype == E4M3 else torch.tensor(2.0 ** 121, dtype=torch.float64)
    assert ((got - x).abs() <= torch.where(x.abs() > TOP[dtype], x.abs() - TOP[dtype], half)).all()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_largest_values_stay_finite(dtype, block):
    big = torch.arange(128, 256).double() * 2.0 ** 120            # every bf16 number from 2^127 on
    x = torch.stack([big, -big, big.flip(0), big * 0.5])[None, :, None].to(torch.bfloat16)
    assert torch.isfinite(x).all() and x.max() == torch.finfo(torch.bfloat16).max
    cache = build_switch_kv_cache(1, 200, 1, device=DEV, dtype=dtype, block_size=block)
    lens = _append(cache, x, 0)
    k, v = switch_kv_cache_read(cache, 0, 4)
    _near(k, x, dtype)
    _near(v, -x, dtype)
    assert k.max() == TOP[dtype] and k.min() == -TOP[dtype]
    # Moved to another cache they stay as they are, and so does what shares their block.
    kept, after, _ = switch_kv_cache_evict(cache, lens, torch.ones(1, 1, 200, device=DEV), budget=3, recent=1)
    ek, ev = switch_kv_cache_read(kept, 0, 3, cache_lens=after)
    assert torch.equal(ek[0], k[0, [0, 1, 3]]) and torch.equal(ev[0], v[0, [0, 1, 3]])


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_held_rows_that_are_rounded_again_stay_finite(dtype):
    """Rows below the largest values, whose scale then grows to theirs: 127 * 2^121 of
    int8 would become 64 * 2^122."""
    first = {E4M3: 1.75 * 2.0 ** 127, INT8: 127 * 2.0 ** 121}[dtype]
    x = torch.full((1, 3, 1, 128), first).to(torch.bfloat16)
    cache = build_switch_kv_cache(1, 40, 1, device=DEV, dtype=dtype, block_size=32)
    _append(cache, x, 0)
    assert torch.equal(switch_kv_cache_read(cache, 0, 3)[0].cpu(), x)
    top = torch.full((1, 1, 1, 128), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    before = (cache.k.clone(), cache.k_scales.clone())
    lens = _append(cache, top, 3)
    values, scales, _ = C.append(*before, 32, [top[0].float().numpy()], [3])
    assert np.array_equal(C.cache_values(cache.k, cache.k_scales, 32)[0, :4], values[0, :4])
    assert float(cache.k_scales[0, 0, 0]) == scales[0, 0, 0]
    k, v = switch_kv_cache_read(cache, 0, 4, cache_lens=lens)
    _near(k, torch.cat([x, top], 1), dtype)
    _near(v, -torch.cat([x, top], 1), dtype)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("scale", [1.3 * 2.0 ** 121, 1.9 * 2.0 ** 123, 1.5 * 2.0 ** 126, 1.99 * 2.0 ** 127])
def test_scales_made_elsewhere_up_to_the_largest(dtype, scale):
    """A begun block keeps its own scale where it is larger than the new rows' (2^120, 2^122);
    the new rows stay finite in it."""
    cache = build_switch_kv_cache(1, 32, 1, device=DEV, dtype=dtype, block_size=32)
    zero = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    _append(cache, zero, 0)
    cache.k_scales[0, 0, 0] = cache.v_scales[0, 0, 0] = scale
    x = (torch.linspace(-1, 1, 128).double() * torch.finfo(torch.bfloat16).max).to(torch.bfloat16).view(1, 1, 1, 128)
    before = (cache.k.clone(), cache.k_scales.clone())
    lens = _append(cache, x, 1)
    values, _, _ = C.append(*before, 32, [x[0].float().numpy()], [1])
    own = float(before[1][0, 0, 0])
    assert float(cache.k_scales[0, 0, 0]) == max(own, 2.0 ** (120 if dtype == E4M3 else 122))
    assert np.array_equal(C.cache_values(cache.k, cache.k_scales, 32)[0, :2], values[0, :2])
    k, v = switch_kv_cache_read(cache, 0, 2, cache_lens=lens)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


def test_a_decode_over_the_largest_keys_is_finite():
    """Scores of the largest finite keys and small queries, weights of the largest
    values that a single key has."""
    cache = build_switch_kv_cache(1, 16, 1, device=DEV, dtype=INT8, block_size=16)
    x = torch.full((1, 1, 1, 128), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    lens = _append(cache, x, 0)
    q = torch.full((1, 1, 2, 128), 2.0 ** -120, dtype=torch.bfloat16, device=DEV)
    out, lse = switch_gqa_decode_quantized_forward(q, cache, lens, torch.tensor([True], device=DEV))
    assert (out == -TOP[INT8]).all() and torch.isfinite(lse).all() and math.isfinite(float(lse.max()))


def test_a_held_minus_128_keeps_the_nearest_code():
    """A block made elsewhere that holds -128 takes the scale of new rows, 2^e: -128 stays
    only where the old scale is less than 1/256 below it."""
    for own, code in ((1.0 - 2.0 ** -10, -128), (127.75 / 128, -128), (127.25 / 128, -127), (0.6, -77)):
        cache = build_switch_kv_cache(1, 32, 1, device=DEV, dtype=INT8, block_size=32)
        _append(cache, torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16), 0)
        cache.k[0, :2] = -128
        cache.k_scales.fill_(own)
        x = torch.full((1, 1, 1, 128), 100.0, dtype=torch.bfloat16)
        _append(cache, x, 2)
        assert float(cache.k_scales[0, 0, 0]) == 1.0 and (cache.k[0, :2] == code).all() and (cache.k[0, 2] == 100).all()
