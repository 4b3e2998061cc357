"""An append behind more than 2^30 rows, whose blocks counted on from there pass row 2^31
(``rows`` of the C ABI is a limit, here the largest)."""

import pytest
import torch

from switchattentionkernels_amd import _lib, build_switch_kv_cache, switch_kv_cache_append

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("new", [1, 24])
def test_append_behind_2_to_30_rows(new):
    """Of the cache only the last rows' memory is there, as a caller that maps it by need
    can have: the call touches no other, and does what it does to a small cache."""
    block, cap, n = 128, 2 ** 30 + 1024, 2 ** 30 + 1000
    first = n // block * block                                # the row that the buffers start with
    gen = torch.Generator().manual_seed(new)
    held = torch.randn(1, n - first, 1, 128, generator=gen).to(torch.bfloat16).to(DEV)
    x = (4 * torch.randn(1, new, 1, 128, generator=gen)).to(torch.bfloat16).to(DEV)
    zero, lens = (torch.tensor([v], dtype=torch.int32, device=DEV) for v in (0, n))
    caches = []
    for _ in range(2):
        cache = build_switch_kv_cache(1, cap - first, 1, device=DEV, block_size=block)
        for t in (cache.k, cache.v):
            t.view(torch.uint8).fill_(0x55)
        cache.k_scales.fill_(7.0)
        cache.v_scales.fill_(7.0)
        assert switch_kv_cache_append(cache, held, -held, zero).tolist() == [n - first]
        caches.append(cache)
    far, near = caches
    want = switch_kv_cache_append(near, x, -x, torch.tensor([n - first], dtype=torch.int32, device=DEV))
    cu = torch.tensor([0, new], dtype=torch.int32, device=DEV)
    out, minus = torch.zeros_like(zero), -x
    torch.cuda.synchronize()
    print(f"append of {new} rows behind row {n}, blocks of the limit from {n // block} on", flush=True)
    st = _lib.lib().swattn_cache_append(
        x.data_ptr(), minus.data_ptr(), cu.data_ptr(), None, lens.data_ptr(),
        far.k.data_ptr() - first * 128, far.v.data_ptr() - first * 128,
        far.k_scales.data_ptr() - first // block * 4, far.v_scales.data_ptr() - first // block * 4,
        out.data_ptr(), 1, 2 ** 31 - 1, new, cap, 1, 128, block, 0, _lib.stream_handle(DEV))
    assert st == 0, _lib.lib().swattn_last_error()
    torch.cuda.synchronize()
    assert out.item() - first == want.item()
    for a, b in ((far.k, near.k), (far.v, near.v), (far.k_scales, near.k_scales), (far.v_scales, near.v_scales)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
