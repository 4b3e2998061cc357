"""Scores below fp32's range in the decode over an 8-bit cache: -inf in fp32, a weight of
0 in the formula.  A wave meets 32 keys at a time, so that its first ones may all be such."""

import math

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import SwitchKVCache, switch_gqa_decode_quantized_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,far", [(torch.float8_e4m3fn, -448.0), (torch.int8, -127.0)])
@pytest.mark.parametrize("first,last", [(0, 200), (0, 699), (100, 700), (32, 64), (1, 700)])
def test_scores_of_minus_infinity_weigh_nothing(dtype, far, first, last):
    """Keys [first, last) of 700 have a score of about -1e39; head 1 does not see it."""
    gen = torch.Generator().manual_seed(first + last)
    n, g = 700, 2
    k = torch.randint(-8, 9, (1, n, 1, 128), generator=gen).float() / (4 if dtype != torch.int8 else 1)
    v = torch.randint(-8, 9, (1, n, 1, 128), generator=gen).float()
    k[..., 0] = 0
    k[0, first:last, 0, 0] = far
    q = torch.randn(1, 1, g, 128, generator=gen).to(torch.bfloat16)
    q[..., 0, 0], q[..., 1, 0] = 3e38, 0.0
    ones = torch.ones(1, 1, -(-n // 64), device=DEV)
    cache = SwitchKVCache(k.to(dtype).to(DEV), v.to(dtype).to(DEV), ones, ones.clone(), 64)
    lens, full = torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([True], device=DEV)
    w = torch.zeros(1, 1, n, device=DEV)
    out, lse = switch_gqa_decode_quantized_forward(q.to(DEV), cache, lens, full, key_weights=w)
    want, want_lse, want_w, _ = C.decode(q[:, 0], k.double().numpy(), v.double().numpy(), [n], [True], n)
    # Scores that are not far: 130 * 2^-24 * c * sum |q_i k_i|, d below, in log2 units; weights
    # ln 2 of that, twice, and 2^-20; O one rounding more.
    near = k[0, :, 0, 1:].abs() @ q[0, 0, :, 1:].float().abs().t()
    d = 130 * 2.0 ** -24 * 128 ** -0.5 * math.log2(math.e) * float(near.max())
    eps = 2 * math.log(2) * d + 2.0 ** -20
    assert np.isfinite(want).all()
    assert (np.abs(out[:, 0].double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + 8 * eps).all()
    assert (np.abs(lse[:, 0].double().cpu().numpy() - want_lse) <= d + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse)).all()
    assert (np.abs(w.double().cpu().numpy() - want_w) <= eps * want_w + 1e-30).all()


def test_nothing_but_such_scores_is_not_a_number():
    k = torch.full((1, 40, 1, 128), -100, dtype=torch.int8, device=DEV)
    ones = torch.ones(1, 1, 1, device=DEV)
    cache = SwitchKVCache(k, k.clone(), ones, ones.clone(), 64)
    q = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 3e38
    out, _ = switch_gqa_decode_quantized_forward(q, cache, torch.tensor([40], dtype=torch.int32, device=DEV),
                                                 torch.tensor([True], device=DEV))
    assert torch.isnan(out).all()
