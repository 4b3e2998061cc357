"""The C ABI's gradients of a rotation without norms take no rows (no GPU: what is refused)."""

import ctypes

from switchattentionkernels_amd import _lib

P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def _bwd(q, k, q_weight, k_weight, seq=0):
    strides = (ctypes.c_int64 * 3)(128, 128, 128)
    rows = [x for t in (q, k) for x in (t, None if t is None else strides)]
    return _lib.lib().swattn_rotary_bwd(P, P, *rows, P, P, 1, (ctypes.c_int32 * 1)(64), 1, 0, q_weight, k_weight, 0,
                                        ctypes.c_float(1e-6), P, P, None, None, 2, seq, 4, 2, 128, None, 0, None)


def test_rows_are_asked_for_where_there_is_a_norm():
    assert _bwd(None, None, None, None) == 0          # no tokens: nothing launched
    assert _bwd(ODD, None, None, None) == 0           # not looked at
    assert _bwd(P, None, P, None) == 0 and _bwd(None, P, None, P) == 0
    for rows in ((None, P, P, None), (P, None, None, P), (ODD, P, P, P), (P, ODD, P, P)):
        assert _bwd(*rows) == -1, rows
        assert b"strides" in _lib.lib().swattn_last_error()
