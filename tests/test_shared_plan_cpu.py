"""The plan of a decode step behind prefixes as the library works it out: every key of every tile
in one piece, partials that do not share a place, and all of them within the workspace and
the grid (``swattn_shared_plan``: the functions that the device runs)."""

import ctypes

import numpy as np
import pytest

from switchattentionkernels_amd import _lib


def _plan(plens, ids, lens, full, cap, prefix_cap, hq, hkv, window):
    L = _lib.lib()
    batch, prefixes = len(ids), len(plens)
    arrays = [np.ascontiguousarray(x, dtype=t) for x, t in ((plens, np.int32), (ids, np.int32), (lens, np.int32), (full, np.uint8))]
    most = 512 + batch * hkv
    totals, pieces = np.zeros(8, np.int64), np.zeros((most, 8), np.int32)
    own = np.zeros((batch, hkv, 4), np.int64)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    assert L.swattn_shared_plan(*map(ptr, arrays), batch, cap, prefixes, prefix_cap, hq, hkv, window, ptr(totals), ptr(pieces),
                                most, ptr(own)) == 0
    return totals, pieces[:totals[0]], own


def _check(plens, ids, lens, full, cap, prefix_cap, hq, hkv, window):
    n_pieces, held, shares, slots, slots_held, grid, share, line = (
        plan := _plan(plens, ids, lens, full, cap, prefix_cap, hq, hkv, window))[0].tolist()
    pieces, own = plan[1], plan[2]
    # What is attended, from the definition.
    seqs = 128 // (hq // hkv)
    rows = np.clip(plens, 0, prefix_cap)
    mine = np.clip(lens, 0, cap)
    groups = {}
    for b, i in enumerate(ids):
        if 0 <= i < len(plens):
            start = 0 if full[b] else max(rows[i] + mine[b] - window, 0)
            if start < rows[i]:
                groups.setdefault((i, int(not full[b])), []).append(start)
    keys = np.where(np.asarray(full) != 0, mine, np.minimum(mine, window))
    # Every (prefix, route, tile, KV head): its keys in order, in up to 255 pieces.
    want = {(i, r, t, h): (min(s), rows[i]) for (i, r), s in groups.items() for t in range(-(-len(s) // seqs)) for h in range(hkv)}
    got = {}
    for i, r, t, h, first, end, place, parts in pieces.tolist():
        got.setdefault((i, r, t, h), []).append((first, end, place, parts))
    assert set(got) == set(want)
    for x, parts in got.items():
        parts.sort()
        assert len(parts) <= 255 and all(p[3] == len(parts) for p in parts)
        assert parts[0][0] == want[x][0] and parts[-1][1] == want[x][1]
        assert all(a[1] == b[0] and b[2] == a[2] + 1 for a, b in zip(parts, parts[1:])) and all(a < b for a, b, _, _ in parts)
        assert all((b - a) % 64 == 0 for a, b, _, _ in parts[:-1])
    assert sorted(pieces[:, 6].tolist()) == list(range(n_pieces)) and n_pieces <= held
    # The line: pairs behind one another, cut into shares; a slot for each (share, pair) that meet at a key.
    assert n_pieces + shares <= grid and (own[:, :, 1] == keys[:, None]).all()
    behind, taken = 0, 0
    for first, n, slot, parts in own.reshape(-1, 4).tolist():
        if n == 0:
            assert parts == 0
            continue
        assert first >= behind and parts == (first + n - 1) // share - first // share + 1 <= 256
        assert slot >= taken
        behind, taken = first + n, slot + parts
    assert behind <= line <= shares * share and taken == slots <= slots_held


def test_random_plans():
    rng = np.random.default_rng(0)
    for i in range(400):
        g, hkv = int(rng.integers(1, 9)), int(rng.integers(1, 17))
        prefixes, batch = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 10))
        prefix_cap, cap = int(2 ** rng.uniform(0, 17)), int(2 ** rng.uniform(0, 15))
        many = rng.random() < 0.3      # few of the prefixes are continued
        ids = rng.integers(-1, 2 if many else prefixes + 1, batch)
        _check(rng.integers(-1, prefix_cap + 2, prefixes), ids, rng.integers(-1, cap + 2, batch) * (rng.random(batch) < 0.9),
               rng.random(batch) < rng.choice([0.0, 0.25, 1.0]), cap, prefix_cap, g * hkv, hkv, int(2 ** rng.uniform(0, 17)))


@pytest.mark.parametrize("batch,prefixes,hkv,g", [(1, 1, 1, 1), (1024, 1024, 8, 8), (1024, 1024, 8, 1), (1024, 512, 8, 1),
                                                  (1023, 1, 16, 7), (256, 256, 64, 2), (257, 256, 16, 5)])
@pytest.mark.parametrize("own", [0, 1, 130])
def test_as_many_tiles_as_there_can_be(batch, prefixes, hkv, g, own):
    """A tile for every sequence where there are prefixes enough, both routes of each; every piece as
    short as pieces are; no own rows, one each, more than a share's least."""
    ids, full = [(i // 2) % prefixes for i in range(batch)], [i % 2 for i in range(batch)]
    for rows in (1, 64, 65, 1000):
        _check([rows] * prefixes, ids, [own] * batch, full, max(own, 1), rows, g * hkv, hkv, 10 ** 6)


def test_shares_of_far_positions():
    """Lines and tiles that end just below 2^31 positions."""
    cap = 2 ** 31 // (1000 * 8) - 193
    _check([5], [0] * 1000, [cap - i for i in range(1000)], [1] * 1000, cap, 5, 8, 8, 7)
    rows = 2 ** 31 // (2 * 8) - 65     # two tiles of 8 KV heads
    _check([rows], [0] * 8, [1] * 8, [1] * 8, 1, rows, 8, 8, 7)
    _check([2 ** 31 - 66], [0], [0], [1], 1, 2 ** 31 - 66, 1, 1, 7)


def test_shapes_that_the_decode_refuses():
    ints = (ctypes.c_int64 * 64)()
    for shape, window in (((1025, 1, 1, 1, 8, 8), 1), ((1, 1, 1025, 1, 8, 8), 1), ((1, 1, 1, 1, 8, 8), 0), ((1, 2 ** 31, 1, 1, 8, 8), 1)):
        assert _lib.lib().swattn_shared_plan(ints, ints, ints, ints, *shape, window, ints, ints, 0, ints) == -1
