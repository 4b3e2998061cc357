"""The decode over an 8-bit cache where its workgroups plan for themselves and shares of
the line of keys go on from one (sequence, KV head) pair into the next, evaluated in 64
bits on the device."""

import math

import pytest
import torch

from switchattentionkernels_amd import (build_switch_kv_cache, switch_gqa_decode_quantized_forward,
                                        switch_kv_cache_append)

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
D, LOG2E = 128, math.log2(math.e)


def _line(keys, hkv):
    """(shared, halved): how the line of these sequences' keys is cut for three
    workgroups per CU: 192 positions beside each pair's keys, unless whole shares for each
    pair are at most 160 keys longer; halved from 4096 on."""
    target = 3 * torch.cuda.get_device_properties(0).multi_processor_count
    total, pairs = sum(keys) * hkv, sum(n > 0 for n in keys) * hkv
    share = -(-(total + 192 * pairs) // target)
    shared = pairs >= target or -(-total // (target - pairs)) > max(share, 128) + 160
    return shared, shared and share >= 4096


def _values(codes, scales, block, n):
    s = scales.double().repeat_interleave(block, dim=-1)[:, :n]
    return codes[:n].float().double().transpose(0, 1) * s[..., None]            # [Hkv, n, 128]


@pytest.mark.parametrize("dtype,b,n_lo,n_hi,hq,hkv,w,p,block,weights,halved", [
    (E4M3, 64, 500, 1500, 32, 8, 200, 0.5, 64, False, False),
    (INT8, 64, 500, 1500, 64, 8, 200, 0.5, 16, True, False),
    (INT8, 130, 1, 900, 24, 8, 700, 0.3, 32, True, False),
    (E4M3, 256, 300, 700, 4, 4, 90, 0.4, 16, True, False),
    (INT8, 1000, 1, 300, 3, 1, 50, 0.5, 32, True, False),       # 4 sequences planned by a thread
    (E4M3, 70, 1000, 2100, 40, 8, 333, 0.5, 128, True, False),  # codes of more than 256 MiB
    (E4M3, 16, 24800, 25600, 16, 8, 1024, 1.0, 64, True, True),
    (INT8, 17, 24000, 25600, 64, 8, 20000, 0.7, 64, False, True),
])
def test_shares_that_go_on_into_the_next_pair(dtype, b, n_lo, n_hi, hq, hkv, w, p, block, weights, halved):
    gen = torch.Generator().manual_seed(b + hq)
    lens = torch.randint(n_lo, n_hi + 1, (b,), generator=gen)
    lens[b // 2] = n_hi
    if b > 20:
        lens[torch.rand(b, generator=gen) < 0.1] = 0            # empty sequences between the others
    full = torch.rand(b, generator=gen) < p
    keys = [n if f else min(n, w) for n, f in zip(lens.tolist(), full.tolist())]
    assert _line(keys, hkv) == (True, halved)
    dev = torch.Generator(device=DEV).manual_seed(b)
    cache = build_switch_kv_cache(b, n_hi, hkv, device=DEV, dtype=dtype, block_size=block)
    cache.k_scales.fill_(math.nan)                              # blocks without a row stay so
    cache.v_scales.fill_(math.nan)
    counts, zero = lens.to(torch.int32).to(DEV), torch.zeros(b, dtype=torch.int32, device=DEV)
    for at in range(0, n_hi, 6400):                             # whole blocks of every size
        m = min(6400, n_hi - at)
        k, v = (torch.randn(b, m, hkv, D, generator=dev, device=DEV).to(torch.bfloat16) for _ in range(2))
        left = (counts - at).clamp(0, m)
        switch_kv_cache_append(cache, k, v, torch.minimum(counts, zero + at), row_counts=left)
    del k, v
    q = torch.randn(b, 1, hq, D, generator=dev, device=DEV).to(torch.bfloat16)
    sums = torch.rand(b, hkv, n_hi, generator=dev, device=DEV) if weights else None
    was = sums.double() if weights else None
    args = (q, cache, counts, full.to(DEV))
    out, lse = switch_gqa_decode_quantized_forward(*args, window_size=w, key_weights=sums)
    again = switch_gqa_decode_quantized_forward(*args, window_size=w)
    assert torch.equal(out.view(torch.int16), again[0].view(torch.int16)) and torch.equal(lse, again[1])
    g = hq // hkv
    for i in range(b):
        n = int(lens[i])
        lo = 0 if full[i] else max(n - w, 0)
        if n == 0:
            assert torch.isnan(out[i]).all() and torch.isneginf(lse[i]).all()
            assert not weights or torch.equal(sums[i].double(), was[i])
            continue
        kk, vv = (_values(c[i], s[i], block, n)[:, lo:] for c, s in ((cache.k, cache.k_scales),
                                                                    (cache.v, cache.v_scales)))
        x = q[i, 0].double().view(hkv, g, D)
        s = torch.matmul(kk, x.transpose(1, 2).contiguous()) * (D ** -0.5 * LOG2E)     # [Hkv, keys, g]
        m = s.amax(1, keepdim=True)
        e = torch.exp2(s - m)
        total = e.sum(1, keepdim=True)
        pr = e / total
        want = torch.matmul(pr.transpose(1, 2).contiguous(), vv.contiguous()).view(hq, D)
        want_lse = (m + torch.log2(total)).view(hq)
        # A score: 128 exact products summed in fp32, scaled twice, 130 * 2^-24 of sum |q_i k_i|
        # (log2 units).  A weight: that of its score and of the LSE, and 2^-20 for the
        # exponentials, sums and merges; 2^-23 for its three parts.  O: one rounding more.
        dots = D ** -0.5 * LOG2E * float(kk.norm(dim=-1).max() * x.norm(dim=-1).max())
        ds = 130 * 2.0 ** -24 * dots
        eps = 2 * math.log(2) * ds + 2.0 ** -20
        off = (out[i, 0].double() - want).abs()
        assert (off <= 2.0 ** -8 * want.abs() + (eps + 2.0 ** -23) * float(vv.abs().max())).all(), (i, off.max().item())
        assert ((lse[i, 0].double() - want_lse).abs() <= ds + 2.0 ** -20 + 2.0 ** -22 * want_lse.abs()).all(), i
        if weights:
            expect = was[i].clone()
            expect[:, lo:n] += pr.sum(2)
            bound = 2.0 ** -23 * expect
            bound[:, lo:n] += eps * pr.sum(2)
            assert ((sums[i].double() - expect).abs() <= bound).all(), i
            assert torch.equal(sums[i, :, :lo].double(), was[i, :, :lo]) and torch.equal(sums[i, :, n:].double(), was[i, :, n:])
