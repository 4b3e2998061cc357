"""Plain evaluation in 64 bits of a routed decode step behind shared prefixes."""

import math

import numpy as np

U = 2.0 ** -24


def decode(q, k_prefix, v_prefix, prefix_lens, prefix_ids, k_cache, v_cache, lens, full, window, sm_scale=None):
    """float64 arrays: q [B, Hq, 128], prefixes [P, Lp, Hkv, 128], caches [B, L, Hkv, 128].
    Returns (O, LSE in log2, bound on O, bound on LSE); a row without keys has O = NaN and
    LSE = -inf.

    Bounds.  A score is a sum of 128 exact products in fp32, scaled: off by at most 134 U
    times the sum of their magnitudes, in log2 units; its weight by that times ln 2, the
    sums over n keys by n + 64 U (exp2, merges).  P enters the product with V as two bf16
    numbers, 2^-16.  O is rounded once to bf16, 2^-8."""
    batch, hq, _ = q.shape
    hkv = k_cache.shape[2]
    g = hq // hkv
    c = (128 ** -0.5 if sm_scale is None else sm_scale) * math.log2(math.e)
    out, size = np.full((batch, hq, 128), np.nan), np.zeros((batch, hq, 128))
    lse, d_lse = np.full((batch, hq), -np.inf), np.zeros((batch, hq))
    for b in range(batch):
        i = prefix_ids[b]
        before = min(max(prefix_lens[i], 0), k_prefix.shape[1]) if 0 <= i < len(prefix_lens) else 0
        own = min(max(lens[b], 0), k_cache.shape[1])
        k = np.concatenate([k_prefix[i, :before] if before else k_cache[b, :0], k_cache[b, :own]])
        v = np.concatenate([v_prefix[i, :before] if before else v_cache[b, :0], v_cache[b, :own]])
        first = 0 if full[b] else max(before + own - window, 0)
        k, v = k[first:], v[first:]
        if len(k) == 0:
            continue
        for h in range(hq):
            with np.errstate(all="ignore"):
                kh, vh = k[:, h // g], v[:, h // g]
                x = kh @ q[b, h] * c
                dots = np.abs(c) * (np.abs(kh) @ np.abs(q[b, h]))
                top = x.max()
                p = np.exp2(x - (top if np.isfinite(top) else 0.0))
                total = p.sum()
                out[b, h] = (p @ vh) / total
                lse[b, h] = top + np.log2(total) if np.isfinite(top) else np.nan
                ds = 134 * U * np.nanmax(np.where(p > 0, dots, 0.0)) if np.isfinite(top) else np.nan
                eps = 2 * math.log(2) * ds + (len(k) + 64) * U + 2.0 ** -16
                size[b, h] = 2.0 ** -8 * np.abs(out[b, h]) + 1.01 * eps * (p @ np.abs(vh)) / total
                d_lse[b, h] = ds + (len(k) + 64) * U / math.log(2) + 2.0 ** -22 * abs(lse[b, h])
    return out, lse, size + 1e-30, d_lse
