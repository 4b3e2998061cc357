"""Norms of rows whose squares leave fp32's range, against 64 bits: bf16 has fp32's
exponents, so that a finite row's mean square can lie anywhere from 2^-266 to 2^256."""

import numpy as np
import pytest
import torch

from oracle import rotary as R
from switchattentionkernels_amd import switch_qk_rotary_backward, switch_qk_rotary_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Exponents of the rows; gradients of the smallest stay below bf16's largest number.
EXPONENTS = [-122, -110, -100, -90, -80, -75, -63, -52, -50, -49, -48, -47, -46, -45, -44, -40, -20, 0, 20, 40, 55, 58, 59,
             60, 61, 62, 63, 64, 65, 66, 80, 100, 120, 126]


def _case(seed):
    gen = torch.Generator().manual_seed(seed)
    n = len(EXPONENTS)
    size = torch.exp2(torch.tensor(EXPONENTS, dtype=torch.float64)).view(1, n, 1, 1)
    rows = lambda h: (torch.randn(1, n, h, 128, generator=gen, dtype=torch.float64) * size).clamp(-3.38e38, 3.38e38).to(torch.bfloat16)  # noqa: E731
    q, k = rows(3), rows(1)
    q[0, :, 2] = torch.randn(n, 128, generator=gen).to(torch.bfloat16)   # one large value among small ones
    q[0, :, 2, 5] = size.flatten().to(torch.bfloat16)
    w = [1 + 0.3 * torch.randn(128, generator=gen) for _ in range(2)]
    pos = torch.randint(-999, 999, (1, 1, n), generator=gen, dtype=torch.int32)
    freq = 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    grads = [torch.randn(x.shape, generator=gen).clamp(-3, 3).to(torch.bfloat16) for x in (q, k)]
    return q, k, w, pos, freq, grads


@pytest.mark.parametrize("eps", [0.0, 1e-35, 1e-6, 1e30])
def test_forward_and_gradients(eps):
    q, k, w, pos, freq, grads = _case(1)
    up = [x.to(DEV) for x in (q, k, pos, freq)]
    how = dict(q_weight=w[0].to(DEV), k_weight=w[1].to(DEV), eps=eps)
    eps = float(np.float32(eps))
    got = switch_qk_rotary_forward(*up, **how)
    back = switch_qk_rotary_backward(*(g.to(DEV) for g in grads), *up, **how)
    unit = R.unit(pos.numpy(), freq.numpy(), [64])
    for i, x in enumerate((q, k)):
        want, off = R.forward(R.np64(x), R.np64(w[i]), eps, *unit, False)
        g = R.np64(got[i])
        bad = ~(np.abs(g - want) <= off + R.BF16_HALF_STEP * (np.abs(want) + off) + 1e-40).all(axis=(0, 2, 3))
        assert not bad.any(), [e for e, b in zip(EXPONENTS, bad) if b]
        dx, off, dw, dw_off = R.backward(R.np64(grads[i]), R.np64(x), R.np64(w[i]), eps, *unit, False)
        g = R.np64(back[i])
        bad = ~(np.abs(g - dx) <= off + R.BF16_HALF_STEP * (np.abs(dx) + off) + 1e-40).all(axis=(0, 2, 3))
        assert not bad.any(), [e for e, b in zip(EXPONENTS, bad) if b]
        assert R.near(R.np64(back[2 + i]), dw, dw_off, R.U)
