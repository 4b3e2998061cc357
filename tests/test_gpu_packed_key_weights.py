"""Attention sums of packed sequences: which calls wait, which can be captured, and the
refusals of those that cannot."""

import copy
import dataclasses
import pickle

import pytest
import torch

from switchattentionkernels_amd import (build_switch_attention_metadata, build_switch_query_indices,
                                        shard_attention_metadata, switch_gqa_prefill_forward,
                                        switch_gqa_prefill_key_weights)

pytestmark = pytest.mark.gpu
DEV = "cuda"
CU = [0, 1, 300, 300, 377, 890]


def _packed(seed, t=CU[-1], hq=8, hkv=2):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(1, t, h, 128, generator=gen).to(torch.bfloat16).to(DEV) for h in (hq, hkv))
    full, local = build_switch_query_indices((torch.rand(t, generator=gen) < 0.4).to(DEV))
    return gen, q, k, full, local


def _metadata(t=CU[-1], cu=CU):
    return build_switch_attention_metadata(t, t, device=DEV, window_size=60, cu_seqlens=cu)


def _sums(q, k, full, local, md):
    _, lse = switch_gqa_prefill_forward(q, k, k, full, local, metadata=md)
    return switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)


def test_packed_sums_are_captured():
    gen, q, k, full, local = _packed(1)
    md = _metadata()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _sums(q, k, full, local, md)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _sums(q, k, full, local, md)
    for _ in range(3):
        for x in (q, k):
            x.copy_(torch.randn(x.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        want = _sums(q, k, full, local, md)
        torch.cuda.synchronize()
        assert torch.equal(held, want) and abs(float(held.double().sum()) / (CU[-1] * 8) - 1) < 1e-5


@pytest.fixture
def waits_allowed_again():
    yield
    torch.cuda.set_sync_debug_mode("default")


def test_packed_sums_wait_only_for_a_check(waits_allowed_again):
    _, q, k, full, local = _packed(2)
    built = _metadata()
    many = list(range(0, 301)) + [CU[-1]]                  # more sequences than kernel arguments hold
    sets = [(built, False), (copy.copy(built), False), (copy.deepcopy(built), True), (_metadata(cu=many), False),
            (dataclasses.replace(built), False), (pickle.loads(pickle.dumps(built)), True),
            (shard_attention_metadata(torch.arange(CU[-1], dtype=torch.int32, device=DEV), kv_start=0,
                                      kv_end=CU[-1], window_size=60), True)]
    mixed = dataclasses.replace(built, local_starts=_metadata().local_starts)
    swapped = dataclasses.replace(built, full_starts=built.local_starts)
    for md, waits in sets + [(mixed, True), (swapped, True)]:
        want = _sums(q, k, full, local, md)
        _, lse = switch_gqa_prefill_forward(q, k, k, full, local, metadata=md)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        if waits:
            with pytest.raises(RuntimeError, match="synchroniz"):
                switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
            torch.cuda.set_sync_debug_mode("default")
        else:
            got = switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
            torch.cuda.set_sync_debug_mode("default")
            assert torch.equal(got, want)


def test_bounds_that_were_modified_are_checked():
    _, q, k, full, local = _packed(3)
    lse = torch.zeros(1, CU[-1], 8, device=DEV)
    for field in ("full_starts", "local_starts", "causal_ends"):
        for way in ("in place", "in place, then copied", "replaced"):
            md = _metadata()
            x = getattr(md, field)
            bad = x.flip(0)
            if way == "replaced":
                md = dataclasses.replace(md, **{field: bad})
            else:
                x.copy_(bad)
                if "copied" in way:
                    md = copy.deepcopy(md)
            with pytest.raises(ValueError, match="non-decreasing along each index list for the sums"):
                switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
    with torch.inference_mode():
        md = _metadata()
        md.causal_ends.copy_(md.causal_ends.flip(0))
    with pytest.raises(ValueError, match="non-decreasing"):
        switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
    md = _metadata()
    md.q_positions.zero_()                                  # no bound of the sums
    assert torch.equal(_sums(q, k, full, local, md), _sums(q, k, full, local, _metadata()))


def test_sums_that_need_a_check_refuse_a_capture():
    _, q, k, full, local = _packed(4)
    md = _metadata()
    _, lse = switch_gqa_prefill_forward(q, k, k, full, local, metadata=md)
    want = switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
    other = copy.deepcopy(md)
    own = full.clone(), local.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="check of the metadata's bounds and cannot be captured"):
            switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=other)
        with pytest.raises(RuntimeError, match="check of the index lists and cannot be captured"):
            switch_gqa_prefill_key_weights(q, k, lse, *own, metadata=md)
        with pytest.raises(RuntimeError, match="check of the index lists and cannot be captured"):
            switch_gqa_prefill_key_weights(q, k, lse, *own, window_size=60)
        held = switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md)
    for _ in range(2):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
