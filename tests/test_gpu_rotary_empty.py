"""Calls of no tokens whose rows are slices: nothing is read, so no stride matters."""

import pytest
import torch

from switchattentionkernels_amd import (switch_qk_rotary, switch_qk_rotary_append, switch_qk_rotary_backward,
                                        switch_qk_rotary_forward)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_no_tokens_of_any_strides():
    wide = lambda h: torch.empty(2, 0, h, 132, dtype=torch.bfloat16, device=DEV)[..., :128]  # noqa: E731
    q, k = wide(4).requires_grad_(), wide(2).requires_grad_()
    assert q.stride(2) % 8 != 0
    pos = torch.zeros(1, 2, 0, dtype=torch.int32, device=DEV)
    freq = torch.ones(64, device=DEV)
    w = torch.ones(128, device=DEV)
    how = dict(q_weight=w, k_weight=w)
    for call in (switch_qk_rotary_forward, switch_qk_rotary):
        a, b = call(q, k, pos, freq, **how)
        assert a.shape == q.shape and b.shape == k.shape
    dq, dk, dwq, dwk = switch_qk_rotary_backward(a.detach(), b.detach(), q, k, pos, freq, **how)
    assert dq.shape == q.shape and dk.shape == k.shape and not dwq.any() and not dwk.any()
    kc, vc = (torch.ones(2, 3, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lens = torch.tensor([1, 5], dtype=torch.int32, device=DEV)
    out, after = switch_qk_rotary_append(q.detach(), k.detach(), k.detach(), kc, vc, lens, pos, freq, **how)
    assert after.tolist() == [1, 3] and out.shape == q.shape and bool((kc == 1).all() and (vc == 1).all())
