"""``switch_gqa_prefill_key_weights`` against 64 bits where rows are cut into long chunks:
64 blocks of 32 rows and more, the local list's half as long, and longer ones where the
parts of a call would take more than 64 MiB.

A weight's error is that of its score, a sum of 128 exact products in fp32, scaled once
and reduced by the LSE: 130 * 2^-24 * d + 2^-23 * max(|LSE|, d), d = c * max |q| |k| >=
c * sum |q_i k_i|, times ln 2, and 2^-22 for the exponential (``eps``).  A lane adds one
weight of a block, at most `blocks` of them a part; five more additions join the lanes and
one each the parts, of which a key has no more than there are chunks: (blocks + 5 +
chunks) * 2^-24 of a sum of positive numbers.

That stays below 2^-11, while a block of 32 rows that is dropped or counted twice moves
a key's sum by 32 of at most group * (p S + W) weights, 2^-10 and more in each case here.
"""

import math

import pytest
import torch

from switchattentionkernels_amd import (build_switch_attention_metadata, build_switch_query_indices,
                                        switch_gqa_prefill_forward, switch_gqa_prefill_key_weights)

pytestmark = pytest.mark.gpu
DEV = "cuda"
C = 128 ** -0.5 * math.log2(math.e)


def _chunk(total, hq, hkv):
    """Blocks a chunk of the full list has: enough of them for 1024 workgroups, at most
    128, unless the parts of the call exceed 64 MiB."""
    axis, pairs = -(-total * (hq // hkv) // 32), -(-total // 256) * hkv
    chunk = min(128, -(-axis * pairs // 1024) + 1)
    most = max(2, 2 ** 26 // (pairs * 1024))
    return max(chunk, -(-3 * axis // (2 * most))), axis


def _want(q, k, lse, start, end, keys):
    """float64 [Hkv, len(keys)] for rows q [R, Hq, 128] and flattened keys."""
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.zeros(hkv, len(keys), dtype=torch.float64, device=DEV)
    j = torch.arange(keys.start, keys.stop, device=DEV)
    see = (j >= start[:, None]) & (j < end[:, None])
    for h in range(hq):
        kh = k[keys.start:keys.stop, h // (hq // hkv)].double().t().contiguous()
        s = torch.matmul(q[:, h].double(), kh).mul_(C).sub_(lse[:, h].double()[:, None])
        out[h // (hq // hkv)] += torch.where(see, torch.exp2(s), 0.0).sum(0)
    return out


@pytest.mark.parametrize("b,s,hq,hkv,w,p,cu,least,step", [
    (1, 16384, 32, 8, 1024, 0.25, None, 128, 1),              # the longest chunks, every key
    (1, 4099, 32, 8, 500, 0.3, None, 70, 1),                  # an odd half
    (2, 4500, 16, 4, 700, 0.2, None, 128, 1),
    (1, 9001, 40, 8, 333, 0.5, [0, 1, 2500, 2500, 6007, 9001], 128, 1),   # packed
    (1, 65536, 16, 4, 300, 0.05, None, 192, 16),              # parts at their limit; every 16th tile
])
def test_long_chunks(b, s, hq, hkv, w, p, cu, least, step):
    gen = torch.Generator(device=DEV).manual_seed(s)
    t = b * s
    chunk, axis = _chunk(t, hq, hkv)
    assert chunk == least
    q, k = (torch.randn(b, s, h, 128, generator=gen, device=DEV).to(torch.bfloat16) for h in (hq, hkv))
    full, local = build_switch_query_indices(torch.rand(b, s, generator=gen, device=DEV) < p)
    assert full.numel() * (hq // hkv) > 32 * chunk and local.numel() * (hq // hkv) > 32 * chunk
    md = None if cu is None else build_switch_attention_metadata(s, s, device=DEV, window_size=w, cu_seqlens=cu)
    _, lse = switch_gqa_prefill_forward(q, k, k, full, local, metadata=md, window_size=w)
    torch.cuda.synchronize()
    torch.full((2 ** 25,), math.nan, device=DEV)              # what a workspace may hold
    got = switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md, window_size=w)
    assert torch.equal(got, switch_gqa_prefill_key_weights(q, k, lse, full, local, metadata=md, window_size=w))
    # 2^-24 of the forward's LSE and scores each way, their errors independent from row to row.
    assert abs(got.double().sum().item() / (t * hq) - 1) < 1e-5
    i = torch.arange(t, device=DEV)
    first = torch.zeros(t, dtype=torch.long, device=DEV)      # of the row's sequence
    for x in (range(0, t, s) if cu is None else cu[:-1]):
        first = torch.where(i >= x, x, first)
    start = first.clone()
    start[local.long()] = torch.maximum(first, i - w + 1)[local.long()]
    d = C * float(q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max())
    eps = math.log(2) * (130 * 2.0 ** -24 * d + 2.0 ** -23 * max(float(lse.abs().max()), d)) + 2.0 ** -22
    bound = eps + (chunk + 5 + axis // (chunk // 2) + 2) * 2.0 ** -24
    assert bound < 2.0 ** -11
    flat = got.transpose(1, 2).reshape(t, hkv).t()            # [Hkv, keys]
    off = size = 0.0
    for a in range(0, t, 256 * step):
        keys = range(a, min(a + 256, t))
        rows = slice(a, t if cu is None else min(x for x in cu if x >= keys.stop))
        rows = slice(a, min(rows.stop, -(-keys.stop // s) * s))   # no later sequence sees them
        want = _want(q.view(t, hq, 128)[rows], k.view(t, hkv, 128), lse.view(t, hq)[rows], start[rows], i[rows] + 1, keys)
        have = flat[:, a:keys.stop].double()
        assert ((have - want).abs() <= bound * want).all(), (a, ((have - want).abs() / want).max().item())
        off += float((have - want).square().sum())
        size += float(want.square().sum())
    assert math.sqrt(off / size) <= eps + 2.0 ** -19, math.sqrt(off / size)
