"""Lengths, routes and prefix numbers that are no tensors are refused by name."""

import pytest
import torch

from switchattentionkernels_amd import switch_gqa_decode_shared_forward, switch_qk_rotary_append

pytestmark = pytest.mark.gpu
DEV = "cuda"
WRONG = [None, [1, 1], 1]


def _rows(*shape):
    return torch.zeros(*shape, 128, dtype=torch.bfloat16, device=DEV)


def _ones(n=2):
    return torch.ones(n, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("name", ["prefix_lens", "prefix_ids", "cache_lens", "full_mask"])
def test_decode(name):
    ok = dict(q=_rows(2, 1, 4), k_prefix=_rows(1, 5, 2), v_prefix=_rows(1, 5, 2), prefix_lens=_ones(1), prefix_ids=_ones(),
              k_cache=_rows(2, 3, 2), v_cache=_rows(2, 3, 2), cache_lens=_ones(), full_mask=_ones() == 1)
    switch_gqa_decode_shared_forward(**ok)
    for wrong in WRONG:
        with pytest.raises(TypeError, match=name):
            switch_gqa_decode_shared_forward(**dict(ok, **{name: wrong}))


def test_append():
    ok = dict(q=_rows(2, 1, 4), k=_rows(2, 1, 2), v=_rows(2, 1, 2), k_cache=_rows(2, 3, 2), v_cache=_rows(2, 3, 2),
              cache_lens=_ones(), positions=torch.zeros(2, 1, dtype=torch.int32, device=DEV), inv_freq=torch.ones(64, device=DEV))
    switch_qk_rotary_append(**ok)
    for wrong in WRONG:
        with pytest.raises(TypeError, match="cache_lens"):
            switch_qk_rotary_append(**dict(ok, cache_lens=wrong))
        if wrong is not None:
            with pytest.raises(TypeError, match="row_counts"):
                switch_qk_rotary_append(**dict(ok, row_counts=wrong))
