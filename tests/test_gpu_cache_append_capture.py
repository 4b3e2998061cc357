"""Appends of packed rows to an 8-bit KV cache under capture."""

import pytest
import torch

from switchattentionkernels_amd import (build_switch_kv_cache, switch_kv_cache_append,
                                        switch_kv_cache_read)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_packed_appends_under_capture():
    """Offsets of a list or a host tensor are kept; those that the host would have to
    read from or copy to the device are refused."""
    gen = torch.Generator().manual_seed(5)
    cu, t = [0, 3, 20, 20, 60], 60
    k = torch.randn(1, t, 2, 128, generator=gen).to(torch.bfloat16).to(DEV)
    zero = torch.zeros(4, dtype=torch.int32, device=DEV)
    cache = build_switch_kv_cache(4, 64, 2, device=DEV)
    many = build_switch_kv_cache(300, 4, 2, device=DEV)
    on_device = torch.tensor(cu, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    offsets = list(cu)
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="from the device and cannot be captured"):
            switch_kv_cache_append(cache, k, k, zero, cu_seqlens=on_device)
        with pytest.raises(RuntimeError, match="256 sequences to the device and cannot be captured"):
            switch_kv_cache_append(many, k, k, torch.zeros(300, dtype=torch.int32, device=DEV),
                                   cu_seqlens=[min(i, t) for i in range(301)])
        after = switch_kv_cache_append(cache, k, k, zero, cu_seqlens=offsets)
    offsets[1] = 7                                          # of no effect on the captured call
    for _ in range(2):
        k.copy_(torch.randn(k.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        assert after.tolist() == [3, 17, 0, 40]
        got, _ = switch_kv_cache_read(cache, 0, 64, cache_lens=after)
        eager = build_switch_kv_cache(4, 64, 2, device=DEV)
        want, _ = switch_kv_cache_read(eager, 0, 64, cache_lens=switch_kv_cache_append(
            eager, k, k, zero, cu_seqlens=torch.tensor(cu)))
        assert torch.equal(got, want)
