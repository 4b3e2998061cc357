"""Sine and cosine relative to themselves: a pair whose other value is 0 shows each of them
alone, where the angle is small or a little beside a quarter turn.

A product a sin t, rounded once: the fraction of turns per position is held to 2^-65, so
that the angle is off by 2^-65 * 2 pi / f of itself (below 2^-30 for the smallest frequency
here, and for angles that lie 2^-30 beside a quarter turn); what is left behind the nearest
quarter turn is made of two conversions, two constants and a sum (3 U of it), the series
costs 4 U, the product 1 U.  12 U in all with room, then half a step of bf16.
"""

import math

import numpy as np
import pytest
import torch

from oracle import rotary as R
from switchattentionkernels_amd import switch_qk_rotary_backward, switch_qk_rotary_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"
POSITIONS = [0, 1, -1, 2, -7, 31, 100, -1000]


def _frequencies(kind):
    if kind == "small":      # a base of 1e8, positions stretched by 32
        return 1e8 ** (-torch.arange(64, dtype=torch.float64) / 64) / 32
    quarters = [k * math.pi / 2 * (1 + s * 2.0 ** -j) for k in (1, 2, 3, 4) for j in (10, 20, 29) for s in (1, -1)]
    return torch.tensor(quarters, dtype=torch.float64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind,dtype", [("small", torch.float64), ("small", torch.float32), ("quarters", torch.float64)])
def test_values_beside_zeros(kind, dtype, interleaved):
    freq = _frequencies(kind).to(dtype)
    n = freq.numel()
    i = torch.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(1, len(POSITIONS), 2, 128, generator=gen).to(torch.bfloat16)
    x[:, :, 0, b], x[:, :, 1, a] = 0.0, 0.0     # head 0: (a cos, a sin), head 1: (-b sin, b cos)
    angle = np.array(POSITIONS, dtype=np.longdouble)[:, None] * freq.numpy().astype(np.longdouble)
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    pos = torch.tensor([[POSITIONS]], dtype=torch.int32, device=DEV)
    up = x.to(DEV)
    for back, got in ((1, switch_qk_rotary_forward(up, up, pos, freq.to(DEV), interleaved=interleaved)),
                      (-1, switch_qk_rotary_backward(up, up, up, up, pos, freq.to(DEV), interleaved=interleaved)[:2])):
        want = R.np64(x)
        xa, xb = want[0, :, 0, a], want[0, :, 1, b]
        want[0, :, 0, a], want[0, :, 0, b] = xa * cos.T, back * xa * sin.T
        want[0, :, 1, a], want[0, :, 1, b] = -back * xb * sin.T, xb * cos.T
        for t in got:
            g = R.np64(t)
            room = (R.BF16_HALF_STEP + 12 * R.U) * np.abs(want) + 1e-40
            worst = np.unravel_index((np.abs(g - want) - room).argmax(), g.shape)
            assert (np.abs(g - want) <= room).all(), (worst, g[worst], want[worst])
