"""Evictions of caches that are mostly empty: every way of holding the weights during the
search, few rows of it taken, with weights of -inf beside the rows behind the end."""

import math

import pytest
import torch

from switchattentionkernels_amd import build_switch_kv_cache, switch_kv_cache_evict

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("capacity", [1000, 4096, 4097, 5000, 16384, 16385, 32768, 32769, 40000])
@pytest.mark.parametrize("low", [0.0, -1.0, -math.inf])
def test_few_rows_of_a_large_cache(capacity, low):
    gen = torch.Generator().manual_seed(capacity)
    lens = [capacity, 301, 300, 299, 777, capacity // 2 + 1]
    budget, recent = 300, 20
    cache = build_switch_kv_cache(len(lens), capacity, 1, device=DEV, dtype=torch.int8, block_size=128)
    for x in (cache.k, cache.v):
        x.zero_()
    cache.k_scales.fill_(1.0)
    cache.v_scales.fill_(1.0)
    w = torch.rand(len(lens), 1, capacity, generator=gen)
    w[torch.rand(w.shape, generator=gen) < 0.7] = low           # many equal ones
    w[1, 0, :301] = low                                         # none else
    _, after, left = switch_kv_cache_evict(cache, torch.tensor(lens, dtype=torch.int32, device=DEV), w.to(DEV),
                                           budget=budget, recent=recent, capacity=budget)
    assert after.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        x = w[b, 0, :n]
        if n > budget:
            heavy = torch.sort(x[:n - recent], descending=True, stable=True).indices[:budget - recent]
            x = torch.cat([x[heavy.sort().values], x[n - recent:]])
        assert torch.equal(left[b, 0, :len(x)].cpu(), x) and not left[b, 0, len(x):].any()
