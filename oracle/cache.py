"""Plain evaluation of the 8-bit KV cache's operators, on the CPU.

Codes and scales in numpy, attention in 64 bits.  No code is shared with the
package: scales are found by search, e4m3 codes by an explicit table of the
format's values.
"""

from __future__ import annotations

import math

import numpy as np
import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
MIN_EXP = -100
BF16_MAX = 255 * 2.0 ** 120


def _e4m3_table() -> np.ndarray:
    """Values of codes 0 .. 126: 4 exponent bits (bias 7), 3 mantissa bits."""
    out = []
    for c in range(127):
        e, m = c >> 3, c & 7
        out.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return np.array(out)


_TABLE = _e4m3_table()


def scale_for(amax: float, dtype) -> float:
    """The smallest power of two from 2^-100 on that holds amax; NaN for NaN or inf."""
    if not math.isfinite(amax):
        return math.nan
    e = MIN_EXP
    while amax > QMAX[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def round_code(x: np.ndarray, dtype) -> np.ndarray:
    """fp32 values in the codes' range to the values of the nearest codes, ties to
    even; NaN to NaN, or 0 where no code stands for it."""
    nan = np.isnan(x)
    x = np.where(nan, 0.0, x).astype(np.float64)
    if dtype == torch.int8:
        return np.rint(x)
    a = np.abs(x)
    hi = np.searchsorted(_TABLE, a, side="left").clip(0, 126)     # first code >= a
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = _TABLE[hi] - a, a - _TABLE[lo]
    pick = np.where(d_hi < d_lo, hi, np.where(d_lo < d_hi, lo, np.where(hi % 2 == 0, hi, lo)))
    pick = np.where(_TABLE[hi] == a, hi, pick)
    return np.where(nan, math.nan, np.copysign(_TABLE[pick], x))


def keep_finite(x: np.ndarray, scale: float, dtype) -> np.ndarray:
    """Codes' values of a block with this scale; for those whose product lies above
    bf16's largest number the largest whose product does not."""
    known = np.arange(128.0) if dtype == torch.int8 else _TABLE
    if math.isnan(scale) or known[-1] * float(scale) <= BF16_MAX:
        return x
    top = known[known * float(scale) <= BF16_MAX].max()
    return np.clip(x, -top, top)


def code_values(codes: torch.Tensor) -> np.ndarray:
    """What codes stand for, without their scales."""
    if codes.dtype == torch.int8:
        return codes.cpu().numpy().astype(np.float64)
    u = codes.view(torch.uint8).cpu().numpy()
    mag = np.append(_TABLE, math.nan)[u & 127]
    return np.where(u & 128, -mag, mag)


def cache_values(codes: torch.Tensor, scales: torch.Tensor, block: int) -> np.ndarray:
    """[B, L, Hkv, 128] in 64 bits."""
    n = codes.shape[1]
    s = np.repeat(scales.double().cpu().numpy(), block, axis=2)[:, :, :n]
    with np.errstate(invalid="ignore"):
        return code_values(codes) * s.transpose(0, 2, 1)[..., None]


def append(codes: torch.Tensor, scales: torch.Tensor, block: int, new, lens):
    """Append ``new[b]`` (fp32 numpy [n_b, Hkv, 128]) behind ``lens[b]`` rows.
    Returns (values of all rows, scales, new lengths) in numpy."""
    dtype = codes.dtype
    cap, heads = codes.shape[1], codes.shape[2]
    raw = code_values(codes).astype(np.float32)
    sc = scales.float().cpu().numpy().copy()
    after = []
    for b, rows in enumerate(new):
        n = min(max(int(lens[b]), 0), cap)
        end = min(n + len(rows), cap)
        after.append(end)
        for j in range(n // block, -(-end // block)):
            lo, hi = max(n, j * block), min(end, (j + 1) * block)
            if lo >= hi:
                continue
            for h in range(heads):
                x = rows[lo - n:hi - n, h].astype(np.float32)
                a = np.abs(x)
                s = scale_for(float(a.max()) if np.isfinite(a).all() else math.inf, dtype)
                if lo > j * block:                     # the block holds rows already
                    old = float(sc[b, h, j])
                    s = math.nan if math.isnan(old) or math.isnan(s) else max(old, s)
                    if not math.isnan(old) and s != old:
                        ratio = np.float32(old) / np.float32(s)
                        raw[b, j * block:lo, h] = keep_finite(
                            round_code(raw[b, j * block:lo, h] * ratio, dtype), s, dtype)
                sc[b, h, j] = s
                with np.errstate(invalid="ignore"):
                    raw[b, lo:hi, h] = keep_finite(round_code(x / np.float32(s), dtype), s, dtype)
    with np.errstate(invalid="ignore"):
        values = raw.astype(np.float64) * np.repeat(sc.astype(np.float64), block, axis=2)[:, :, :cap] \
            .transpose(0, 2, 1)[..., None]
    return values, sc, after


def read(codes: torch.Tensor, scales: torch.Tensor, block: int, starts, rows: int, lens=None):
    """[B, rows, Hkv, 128]; 0 outside the valid rows."""
    x = cache_values(codes, scales, block)
    out = np.zeros((x.shape[0], rows) + x.shape[2:])
    for b in range(x.shape[0]):
        end = x.shape[1] if lens is None else min(int(lens[b]), x.shape[1])
        for i in range(rows):
            r = int(starts[b]) + i
            if 0 <= r < end:
                out[b, i] = x[b, r]
    return out


def decode(q: torch.Tensor, k: np.ndarray, v: np.ndarray, lens, full, window: int, scale=None):
    """(O, LSE, weights, dots) in 64 bits from a cache's values: weights [B, Hkv, L],
    dots the largest sum of |q_i k_i| a score was made of."""
    b, hq, d = q.shape
    cap, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    c = (d ** -0.5 if scale is None else scale) * math.log2(math.e)
    qd = q.double().cpu().numpy()
    out = np.full((b, hq, d), math.nan)
    lse = np.full((b, hq), -math.inf)
    weights = np.zeros((b, hkv, cap))
    dots = 0.0
    for i in range(b):
        n = min(max(int(lens[i]), 0), cap)
        lo = 0 if full[i] else max(n - window, 0)
        if n == 0:
            continue
        for h in range(hq):
            kk, vv = k[i, lo:n, h // g], v[i, lo:n, h // g]
            s = c * (kk @ qd[i, h])
            dots = max(dots, float(np.nanmax(np.abs(kk) @ np.abs(qd[i, h]))) * c)
            m = s.max()
            p = np.exp2(s - m)
            lse[i, h] = m + math.log2(p.sum())
            p /= p.sum()
            out[i, h] = p @ vv
            weights[i, h // g, lo:n] += p
    return out, lse, weights, dots


def key_weights(q, k, lse, start, end, scale=None):
    """Sums [B * Skv, Hkv] of every key's weight over the rows: q [rows, Hq, 128],
    k [keys, Hkv, 128] flattened, lse [rows, Hq], bounds [start, end) per row."""
    rows, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    c = (d ** -0.5 if scale is None else scale) * math.log2(math.e)
    out = torch.zeros(k.shape[0], hkv, dtype=torch.float64)
    j = torch.arange(k.shape[0])
    see = (j >= start[:, None]) & (j < end[:, None])
    for h in range(hq):
        s = c * (q[:, h].double() @ k[:, h // g].double().t()) - lse[:, h].double()[:, None]
        out[:, h // g] += torch.where(see, torch.exp2(s), 0.0).sum(0)
    return out


def evict(k: np.ndarray, v: np.ndarray, weights: np.ndarray, lens, budget: int, recent: int, block: int,
          dtype):
    """What a cut to ``budget`` rows leaves: per sequence and head the kept rows,
    and the destination's values, scales and weights.  k, v: values [B, L, Hkv, 128]."""
    b, cap, heads, d = k.shape
    kept, after = {}, []
    nblk = -(-budget // block)
    ok, ov = np.zeros((b, budget, heads, d)), np.zeros((b, budget, heads, d))
    sk, sv = np.zeros((b, heads, nblk)), np.zeros((b, heads, nblk))
    ow = np.zeros((b, heads, budget))
    for i in range(b):
        n = min(max(int(lens[i]), 0), cap)
        after.append(min(n, budget))
        for h in range(heads):
            rows = list(range(n))
            if n > budget:
                def rank(r):
                    w = weights[i, h, r]
                    return (0, 0.0, r) if math.isnan(w) else (1, -w, r)
                best = sorted(range(n - recent), key=rank)[:budget - recent]
                rows = sorted(best) + rows[n - recent:]
            kept[i, h] = rows
            ow[i, h, :len(rows)] = weights[i, h, rows]
            for out, sc, x in ((ok, sk, k), (ov, sv, v)):
                for j in range(0, len(rows), block):
                    part = x[i, rows[j:j + block], h].astype(np.float32)
                    a = np.abs(part)
                    s = scale_for(float(a.max()) if np.isfinite(a).all() else math.inf, dtype)
                    sc[i, h, j // block] = s
                    with np.errstate(invalid="ignore"):
                        out[i, j:j + len(part), h] = keep_finite(
                            round_code(part / np.float32(s), dtype), s, dtype) * s
    return kept, after, ok, ov, sk, sv, ow
