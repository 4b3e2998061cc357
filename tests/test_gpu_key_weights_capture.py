"""Attention sums with lists that the compaction did not make, under capture."""

import threading

import pytest
import torch

from switchattentionkernels_amd import (build_switch_query_indices, switch_gqa_prefill_forward,
                                        switch_gqa_prefill_key_weights)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_the_first_call_of_a_thread_refuses_a_capture_too():
    """A thread's first call with lists of its own would allocate pinned memory, which a
    capture does not survive."""
    gen, s = torch.Generator().manual_seed(6), 890
    q, k = (torch.randn(1, s, h, 128, generator=gen).to(torch.bfloat16).to(DEV) for h in (8, 2))
    full, local = build_switch_query_indices((torch.rand(s, generator=gen) < 0.4).to(DEV))
    _, lse = switch_gqa_prefill_forward(q, k, k, full, local, window_size=60)
    want = switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=60)
    own = full.clone(), local.clone()
    torch.cuda.synchronize()
    graph, held, errors = torch.cuda.CUDAGraph(), [], []

    def capture():
        try:
            with torch.cuda.graph(graph):
                with pytest.raises(RuntimeError, match="check of the index lists and cannot be captured"):
                    switch_gqa_prefill_key_weights(q, k, lse, *own, window_size=60)
                held.append(switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=60))
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    thread = threading.Thread(target=capture)
    thread.start()
    thread.join()
    assert not errors, errors
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want)
