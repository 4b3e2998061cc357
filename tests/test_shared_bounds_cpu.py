"""The shapes that a decode step behind prefixes takes end where the header says."""

import pytest

from switchattentionkernels_amd import _lib

MOST = 2 ** 31 - 1


def _tiles(batch, prefixes, group):
    return min(batch, 2 * prefixes + batch // (128 // group))


def _taken(*shape):
    return _lib.lib().swattn_shared_decode_workspace_bytes(*shape) > 0


@pytest.mark.parametrize("batch,prefixes,heads_kv,group", [(1, 1, 1, 1), (1, 1, 8, 8), (64, 1, 8, 4), (1024, 1, 64, 1),
                                                           (1024, 1024, 8, 8), (777, 3, 5, 5), (200, 2, 16, 3)])
def test_last_lengths(batch, prefixes, heads_kv, group):
    heads = (heads_kv * group, heads_kv)
    own = min(MOST // (batch * heads_kv) - 192, MOST)
    tiles = _tiles(batch, prefixes, group)
    prefix = min(MOST // (tiles * heads_kv) - 64, MOST)
    assert _taken(batch, own, prefixes, 1, *heads) and not _taken(batch, own + 1, prefixes, 1, *heads)
    assert _taken(batch, 1, prefixes, prefix, *heads) and not _taken(batch, 1, prefixes, prefix + 1, *heads)
    assert _taken(batch, own, prefixes, prefix, *heads)
