"""How many bits of a weight reach the product with V in the decode over an 8-bit
cache: two keys whose terms nearly cancel.

Key 0 scores 0 and key 1 scores -t, t = log2(1.75) - log2(1 + d), |d| from 2^-13 to
2^-12: its weight is w = (1 + d) / 1.75.  With values -a and 1.75 a

    O = a (1.75 w - 1) / (1 + w) = a d / (1 + w),

so that an error e of w is off by 1.75 a e / (1 + w), 1.75 e / |d| relative to O.

* 24 bits: t is a sum of three bf16 numbers times codes of 1 (exact products), scaled
  once: off by at most 4 * 2^-24, 3 * 2^-24 of w; the exponential by one last place,
  2^-23 of w; the three parts of a weight and their sums with terms of at most a by
  4 * 2^-24 a.  All of it: (3 + 2 + 4) * 2^-24 * 1.75 a w / (1 + w) at most, below
  2^-20 a.  O is rounded to bf16, 2^-8 of it.
* 17 bits: e is up to 2^-18, for the terms up to 2^-18 * 1.75 a / 1.57, more than
  2^-18 a: above 2^-20 a and 2^-8 |O| <= 2^-20 a / 1.57 together.  Of 512 weights many
  come near it.
"""

import math

import pytest
import torch

from switchattentionkernels_amd import SwitchKVCache, switch_gqa_decode_quantized_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,a", [(torch.float8_e4m3fn, 256.0), (torch.int8, 64.0)])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_weights_keep_24_bits(dtype, a, group):
    b, h = 512 // group, 1
    gen = torch.Generator().manual_seed(group)
    d = (1 + torch.rand(b, group, generator=gen, dtype=torch.float64)) * 2.0 ** -13
    d = torch.where(torch.rand(b, group, generator=gen) < 0.5, d, -d)
    left = math.log2(1.75) - torch.log2(1 + d)
    q = torch.zeros(b, 1, group, 128, dtype=torch.bfloat16)
    for i in range(3):                       # dims 0, 1, 2: t in three parts
        q[:, 0, :, i] = left.to(torch.bfloat16)
        left = left - q[:, 0, :, i].double()
    k, v = torch.zeros(b, 2, h, 128), torch.zeros(b, 2, h, 128)
    k[:, 1, :, :3] = -1.0
    v[:, 0], v[:, 1] = -a, 1.75 * a
    scales = torch.ones(b, h, 1, device=DEV)
    cache = SwitchKVCache(k.to(dtype).to(DEV), v.to(dtype).to(DEV), scales, scales.clone(), 16)
    lens = torch.full((b,), 2, dtype=torch.int32, device=DEV)
    full = torch.ones(b, dtype=torch.bool, device=DEV)
    sm_scale = math.log(2.0)                 # scores in the exp2 domain, but for its rounding to fp32
    out, _ = switch_gqa_decode_quantized_forward(q.to(DEV), cache, lens, full, sm_scale=sm_scale)
    c = torch.tensor(sm_scale * 1.4426950408889634, dtype=torch.float32).double()
    w = torch.exp2(-c * q[:, 0, :, :3].double().sum(-1))
    want = (a * (1.75 * w - 1) / (1 + w))[..., None].expand(b, group, 128)
    off = (out[:, 0].double().cpu() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * a).all(), (off.max().item(), want.abs().max().item())
