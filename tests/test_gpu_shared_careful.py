"""Prefix pieces of several tiles that run again for values that are not finite, copies past
the memory-side cache, and both at once for more than 256 sequences, against 64 bits
(``oracle/shared.py``)."""

import math

import numpy as np
import pytest
import torch

from oracle import shared as S
from switchattentionkernels_amd import switch_gqa_decode_shared_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
INF, NAN = math.inf, math.nan


def _np(t):
    return t.double().cpu().numpy()


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check(args, window, picked):
    q, kp, vp, plens, ids, kc, vc, lens, full = args
    o, lse = switch_gqa_decode_shared_forward(*args, window_size=window)
    ro, rl, d_o, d_lse = S.decode(_np(q[picked, 0]), _np(kp), _np(vp), plens.tolist(), ids[picked].tolist(),
                                  _np(kc[picked]), _np(vc[picked]), lens[picked].tolist(), full[picked].tolist(), window)
    go, gl = _np(o[picked, 0]), _np(lse[picked, 0])
    assert np.array_equal(np.isnan(go), np.isnan(ro)) and np.array_equal(np.isinf(go), np.isinf(ro))
    assert (go[np.isinf(ro)] == ro[np.isinf(ro)]).all()
    ok = np.isfinite(ro)
    assert ok.any() and (np.abs(go[ok] - ro[ok]) <= d_o[ok]).all()
    assert np.array_equal(np.isnan(gl), np.isnan(rl))
    ok = np.isfinite(rl)
    assert (np.abs(gl[ok] - rl[ok]) <= d_lse[ok]).all()
    return go


N, ENDS, WINDOW = 24700, 24697, 20000   # 101 MB of rows; the last tile ends inside


def _long(batch, hkv=8, group=2):
    """Sequences of both routes behind one prefix, whose local rows begin behind some of its
    tiles and inside one (at ENDS - WINDOW + len)."""
    gen = torch.Generator(device=DEV).manual_seed(batch)
    rows = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(BF16)  # noqa: E731
    lens = [(7 * i) % 41 for i in range(batch)]
    return [rows(batch, 1, hkv * group, 128), rows(1, N, hkv, 128), rows(1, N, hkv, 128), _int32([ENDS]), _int32([0] * batch),
            rows(batch, 40, hkv, 128), rows(batch, 40, hkv, 128), _int32(lens),
            torch.tensor([i % 2 == 0 for i in range(batch)], device=DEV)]


# One tile takes 64 sequences of two query heads per KV head: 5 are streamed, 70 are not.
@pytest.mark.parametrize("batch", [5, 70])
def test_a_large_prefix_to_its_ragged_end(batch):
    args = _long(batch)
    assert N * 8 * 512 >= 96 << 20
    for t in args[1:3]:
        t[:, ENDS:] = NAN                    # behind the prefix
    _check(args, WINDOW, [0, 1, 2, batch - 1])


@pytest.mark.parametrize("batch", [5, 70])
def test_values_that_are_not_finite_in_pieces_of_several_tiles(batch):
    """Pieces of 700 to 800 keys: in their first, middle and last tiles, in the prefix's ragged end,
    around the first keys of the local rows, and behind the prefix."""
    args = _long(batch)
    kp, vp, full = args[1], args[2], args[8]
    first = ENDS - WINDOW                    # of a local sequence with no own row
    for t in (kp, vp):
        t[:, ENDS:] = NAN
    for i, (at, value) in enumerate([(0, INF), (63, NAN), (64, -INF), (129, INF), (700, NAN), (767, INF), (768, -INF), (1500, NAN),
                                     (first - 1, NAN), (first, INF), (first + 7, NAN), (first + 13, -INF), (first + 14, INF),
                                     (first + 40, NAN), (12345, INF), (12346, INF), (20000, -INF), (ENDS - 64, NAN),
                                     (ENDS - 2, INF), (ENDS - 1, -INF)]):
        vp[0, at, i % 7, (37 * i) % 128] = value
    vp[0, 9000, 2] = INF                     # a whole head row
    kp[0, 3000, 7, 5] = NAN                  # ahead of every local row: those of full routes only
    kp[0, 15000, 6, 9] = INF                 # a score of +inf or -inf
    picked = [0, 1, 2, 3, batch - 1]
    go = _check(args, WINDOW, picked)
    nan_rows = np.isnan(go).all(axis=-1)     # heads 14 and 15 attend key 3000 where routed full
    assert (nan_rows[:, 14:] == full[picked].cpu().numpy()[:, None]).all()
    assert not nan_rows[:, :12].any()


@pytest.mark.parametrize("odd", [False, True])
def test_more_than_256_sequences_with_caches_past_the_memory_side_cache(odd):
    b, cap, hkv, group = 300, 260, 8, 2
    gen = torch.Generator(device=DEV).manual_seed(7)
    rows = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(BF16)  # noqa: E731
    assert b * cap * hkv * 512 >= 256 << 20
    lens = [(17 * i) % (cap + 1) for i in range(b)]
    args = [rows(b, 1, hkv * group, 128), rows(3, 500, hkv, 128), rows(3, 500, hkv, 128), _int32([500, 70, 333]),
            _int32([i % 4 - 1 for i in range(b)]), rows(b, cap, hkv, 128), rows(b, cap, hkv, 128), _int32(lens),
            torch.tensor([i % 3 == 0 for i in range(b)], device=DEV)]
    for i, n in enumerate(lens):
        args[5][i, n:], args[6][i, n:] = NAN, NAN
    picked = [0, 1, 2, 3, 4, 5, 6, 7, 63, 64, 151, 255, 256, 257, 298, 299]
    if odd:
        for j, i in enumerate(picked):
            if lens[i] > 0:
                args[6][i, (31 * j) % lens[i], j % hkv, (19 * j) % 128] = (NAN, INF, -INF)[j % 3]
        args[2][0, 450, 3, 50], args[2][2, 5, 4, 51] = INF, NAN
    _check(args, 150, picked)
