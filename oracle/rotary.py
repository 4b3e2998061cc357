"""Plain evaluation in 64 bits of the norm and rotation of query and key rows.

Everything is numpy float64; angles are formed in 80-bit floats, where an fp32 or fp64
frequency of about 1 times a 31-bit position is off by less than 2^-32 radians.  Each
function also gives a bound on what fp32 sums and products of the same terms may be
off by, from the counts of roundings on the way (``U`` is half a unit of fp32).
"""

import numpy as np

U = 2.0 ** -24
BF16_HALF_STEP = 2.0 ** -8


def np64(t):
    return t.detach().double().cpu().numpy()


def unit(positions, inv_freq, sections):
    """cos and sin [B, S, 1, n] of positions [axes, B, S] (int arrays)."""
    axis = np.repeat(np.arange(len(sections)), sections)
    at = np.asarray(positions)[axis].transpose(1, 2, 0).astype(np.longdouble)
    angle = at * np.asarray(inv_freq).astype(np.longdouble)
    return (np.cos(angle).astype(np.float64)[:, :, None], np.sin(angle).astype(np.float64)[:, :, None])


def _pairs(rotary, interleaved):
    i = np.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def turn(x, cos, sin, interleaved):
    """(x rotated, sum of the magnitudes of each result's terms)."""
    a, b = _pairs(2 * cos.shape[-1], interleaved)
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


def forward(x, weight, eps, cos, sin, interleaved):
    """(rotated rows, their bound).  The norm: 16 products of squares in a lane's chain, 3
    sums over lanes, mean and eps (22 roundings, half of them in the root), root, quotient
    and two products: 16 U.  The angle: 2^-34 turns at most, its conversion and scaling, the series
    and its end: 5 U of sine and cosine.  Two products and a sum: 3 U."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * weight
    y, size = turn(x, cos, sin, interleaved)
    return y, 24 * U * size


def backward(dy, x, weight, eps, cos, sin, interleaved):
    """(dx, its bound, dw, its bound); dw None without a weight."""
    g, size = turn(dy, cos, -sin, interleaved)
    off = 8 * U * size                                   # of g, as above without the norm
    if weight is None:
        return g, off, None, None
    r = 1.0 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps)
    u = x * r
    gw = g * weight
    mean = (gw * u).mean(axis=-1, keepdims=True)
    dx = r * (gw - u * mean)
    # r 16 U, u 17 U, the mean's sum 20 U beside both, products and the difference.
    dx_off = r * (np.abs(weight) * off + 20 * U * np.abs(gw) + np.abs(u) * (
        (np.abs(weight * u) * off).mean(axis=-1, keepdims=True)
        + 80 * U * np.abs(gw * u).mean(axis=-1, keepdims=True)))
    axes = tuple(range(x.ndim - 1))
    rows = x.size // 128
    # A chain of at most rows / 8 terms in a lane, then 5 + 4 + 64 partial sums.
    chain = min(rows, rows / 8 + 80) + 20
    dw_off = (np.abs(u) * off).sum(axis=axes) + chain * U * np.abs(g * u).sum(axis=axes)
    return dx, dx_off, (g * u).sum(axis=axes), dw_off


def near(got, want, off, half_step):
    """Whether ``got`` is ``want`` rounded once, by at most ``half_step`` of the value, after
    an error of at most ``off``; values that are not finite agree."""
    fine = np.isfinite(want)
    same = np.array_equal(np.isnan(got[~fine]), np.isnan(want[~fine])) and np.array_equal(
        got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    room = off + half_step * (np.abs(want) + off) + 1e-40
    return same and bool((np.abs(got - want)[fine] <= room[fine]).all())
