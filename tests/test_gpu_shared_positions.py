"""A serving loop as it is documented, with prefix numbers and lengths outside their ranges:
positions that follow what the decode attends."""

import torch
import pytest

from switchattentionkernels_amd import (switch_gqa_decode_forward, switch_gqa_decode_shared_forward,
                                        switch_qk_rotary_append, switch_qk_rotary_forward)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def test_tokens_stand_behind_what_they_attend():
    gen = torch.Generator().manual_seed(3)
    rows = lambda *s: torch.randn(*s, 128, generator=gen).to(BF16).to(DEV)  # noqa: E731
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    P, Lp, cap, hq, hkv = 2, 70, 9, 8, 2
    prefix_lens, prefix_ids = int32([45, 99]), int32([0, -1, 1, 2, 2 ** 31 - 1, -2 ** 31, 1])
    held = [45, 0, 70, 0, 0, 0, 70]              # rows of its prefix that each sequence has
    B = len(held)
    inv_freq = 1e4 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)
    k0, v_prefix = rows(P, Lp, hkv), rows(P, Lp, hkv)
    at = torch.arange(Lp, dtype=torch.int32, device=DEV).expand(P, Lp)
    _, k_prefix = switch_qk_rotary_forward(k0, k0, at, inv_freq)
    k_cache, v_cache = (torch.zeros(B, cap, hkv, 128, dtype=BF16, device=DEV) for _ in range(2))
    one_k, one_v = (torch.zeros(B, Lp + cap, hkv, 128, dtype=BF16, device=DEV) for _ in range(2))
    for b, n in enumerate(held):
        if n:
            one_k[b, :n], one_v[b, :n] = k_prefix[prefix_ids[b], :n], v_prefix[prefix_ids[b], :n]
    lens, one_lens = int32([0] * B), int32(held)
    for step in range(4):
        q, k, v = rows(B, 1, hq), rows(B, 1, hkv), rows(B, 1, hkv)
        has = (prefix_ids >= 0) & (prefix_ids < P)
        behind = torch.where(has, prefix_lens.clamp(0, Lp)[prefix_ids.clamp(0, P - 1)], 0)
        assert behind.tolist() == held
        at = (behind + lens)[:, None]
        qr, lens = switch_qk_rotary_append(q, k, v, k_cache, v_cache, lens, at, inv_freq)
        qr2, one_lens = switch_qk_rotary_append(q, k, v, one_k, one_v, one_lens, one_lens[:, None].clone(), inv_freq)
        assert torch.equal(qr, qr2)
        full = torch.rand(B, generator=gen).to(DEV) < 0.5
        o, lse = switch_gqa_decode_shared_forward(qr, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, lens,
                                                  full, window_size=30)
        want, want_lse = switch_gqa_decode_forward(qr, one_k, one_v, one_lens, full, window_size=30)
        assert (o.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()
        assert (lse - want_lse).abs().max() <= 1e-4
