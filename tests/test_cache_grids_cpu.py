"""Launches of 2^32 threads and more are refused before anything is launched."""

import ctypes

from switchattentionkernels_amd import _lib


def test_an_eviction_of_too_many_pairs_is_refused():
    """Its search takes 1024 threads a (sequence, KV head) pair, its copy 256 a block."""
    L = _lib.lib()
    src = [ctypes.c_void_p(4096 * (i + 1)) for i in range(6)]
    dst = [ctypes.c_void_p(4096 * (i + 1) + 256) for i in range(6)]
    for heads, out_len in ((65, 1), (200, 16), (65, 50)):           # 2^22 pairs and more
        assert 65535 * heads >= 2 ** 22
        size = L.swattn_cache_evict_workspace_bytes(65535, heads, 1)
        st = L.swattn_cache_evict(*src, *dst, 65535, 10, out_len, heads, 128, 16, 0, 1, 0, ctypes.c_void_p(256),
                                  size, None)
        assert st == -1 and b"grid too large" in L.swattn_last_error(), (heads, out_len, st, L.swattn_last_error())
