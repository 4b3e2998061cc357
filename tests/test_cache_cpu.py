"""The 8-bit KV cache without a GPU: its C ABI, its refusals, its oracle."""

import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (SwitchKVCache, _lib, build_switch_kv_cache, decode,
                                        switch_gqa_decode_quantized_forward,
                                        switch_kv_cache_append, switch_kv_cache_evict,
                                        switch_kv_cache_read)
from switchattentionkernels_amd import cache as cache_module

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(256)
F = ctypes.c_float(0.1)


def test_library_exports_what_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "swattn_cache.h")).read(), flags=re.S)
    found = {m.group(1): len([a for a in m.group(2).split(",") if a.strip()])
             for m in re.finditer(r"\b(swattn_\w+)\s*\(([^)]*)\)\s*;", text)}
    assert set(found) == set(_lib.CACHE_SIGNATURES)
    for name, n in found.items():
        assert hasattr(_lib.lib(), name) and len(_lib.CACHE_SIGNATURES[name][1]) == n, name


def _refused(status, words, code=-1):
    assert status == code, (status, _lib.lib().swattn_last_error())
    assert words.encode() in _lib.lib().swattn_last_error(), _lib.lib().swattn_last_error()


def test_c_abi_refusals():
    L = _lib.lib()

    def append(batch=2, rows=3, cap=10, heads=2, dim=128, block=16, code=0, new=P, k=P, out=ctypes.c_void_p(512),
               cu=None, counts=None):
        return L.swattn_cache_append(new, P, cu, counts, P, k, P, P, P, out, batch, rows, rows, cap, heads,
                                     dim, block, code, None)

    _refused(append(dim=64), "head_dim")
    _refused(append(batch=0), "bad shape")
    _refused(append(cap=2 ** 31), "too large")
    _refused(append(block=48), "block must be")
    _refused(append(block=0), "block must be")
    _refused(append(code=2), "unknown code")
    _refused(append(rows=-1), "number of rows")
    _refused(append(cu=P, counts=P), "exclude")
    _refused(append(k=None), "null")
    _refused(append(new=None), "null")
    _refused(append(out=P), "lens_out")
    _refused(append(new=ctypes.c_void_p(264)), "16-byte")

    def read(rows=3, start=0, k=P, out=P, block=16, code=1):
        return L.swattn_cache_read(k, P, P, P, None, start, None, out, P, 2, rows, 10, 2, 128, block, code, None)

    _refused(read(rows=-1), "range of rows")
    _refused(read(start=-1), "range of rows")
    _refused(read(rows=2 ** 27), "too many rows")
    _refused(read(k=None), "null")
    _refused(read(out=ctypes.c_void_p(264)), "16-byte")
    _refused(read(block=8), "block must be")
    assert read(rows=0) == 0

    def dec(hq=4, hkv=2, window=5, block=16, code=0, ws=P, size=1 << 30, q=P, dim=128, weights=None):
        return L.swattn_cache_decode_fwd(q, P, P, P, P, P, P, P, P, weights, 2, 100, hq, hkv, dim, window, block,
                                         code, F, ws, size, None)

    need = L.swattn_cache_decode_workspace_bytes(2, 100, 4, 2, 0)
    more = L.swattn_cache_decode_workspace_bytes(2, 100, 4, 2, 1)
    assert more - need == 2 * 4 * 128 * 4          # scores, fp32, 100 keys rounded up to 128
    assert L.swattn_cache_decode_workspace_bytes(2, 100, 5, 2, 1) == 0
    _refused(dec(dim=64), "head_dim")
    _refused(dec(hq=5), "multiple")
    _refused(dec(hq=18), "at most 8")
    _refused(dec(window=0), "window")
    _refused(dec(block=17), "block must be")
    _refused(dec(code=-1), "unknown code")
    _refused(dec(q=None), "null")
    _refused(dec(q=ctypes.c_void_p(264)), "16-byte")
    _refused(dec(ws=ctypes.c_void_p(272)), "256-byte")
    _refused(dec(size=need - 1), "workspace", -2)
    _refused(dec(size=more - 1, weights=P), "workspace", -2)

    def evict(budget=5, recent=2, out_len=10, ws=P, size=1 << 20, shift=256):
        a = [ctypes.c_void_p(4096 * (i + 1)) for i in range(6)]
        b = [ctypes.c_void_p(4096 * (i + 1) + shift) for i in range(6)]
        return L.swattn_cache_evict(*a, *b, 2, 10, out_len, 2, 128, 16, 0, budget, recent, ws, size, None)

    _refused(evict(budget=0), "budget")
    _refused(evict(budget=11), "budget")
    _refused(evict(recent=6), "recent")
    _refused(evict(recent=-1), "recent")
    _refused(evict(shift=0), "destination")
    _refused(evict(shift=8), "16-byte")
    _refused(evict(size=L.swattn_cache_evict_workspace_bytes(2, 2, 5) - 1), "workspace", -2)
    _refused(evict(ws=ctypes.c_void_p(272)), "256-byte")
    assert L.swattn_cache_evict_workspace_bytes(0, 2, 5) == 0


def test_c_abi_refusals_of_the_key_weights():
    L = _lib.lib()

    def call(batch=1, sq=8, skv=8, hq=4, hkv=2, dim=128, window=4, nf=3, nl=5, q=P, k=P, starts=None,
             ws=P, size=1 << 30, scale=F):
        return L.swattn_prefill_key_weights(q, k, P, P, nf, P, nl, starts, None, None, P, batch, sq, skv, hq, hkv,
                                            dim, window, scale, ws, size, None)

    need = L.swattn_prefill_key_weights_workspace_bytes(1, 8, 4, 2, 128, 3, 5)
    assert need > 0 and L.swattn_prefill_key_weights_workspace_bytes(1, 8, 5, 2, 128, 3, 5) == 0
    _refused(call(dim=64), "head_dim")
    _refused(call(skv=0), "bad shape")
    _refused(call(hq=5), "multiple")
    _refused(call(window=0), "window")
    _refused(call(scale=ctypes.c_float(math.nan)), "finite")
    _refused(call(nf=4), "index counts")
    _refused(call(nf=-1), "index counts")
    _refused(call(sq=2 ** 40, nf=2 ** 40), "2^31")
    _refused(call(sq=2 ** 29, nf=2, nl=2, size=1 << 60), "rows of Q")
    _refused(call(starts=P), "metadata")
    _refused(call(q=None), "null")
    _refused(call(k=ctypes.c_void_p(264)), "16-byte")
    _refused(call(size=need - 1), "workspace", -2)
    _refused(call(ws=ctypes.c_void_p(272)), "256-byte")


def _cache(b=2, n=40, h=2, dtype=torch.int8, block=16):
    s = (b, h, -(-n // block))
    return SwitchKVCache(torch.zeros(b, n, h, 128, dtype=dtype), torch.zeros(b, n, h, 128, dtype=dtype),
                         torch.ones(s), torch.ones(s), block)


class _OnDevice(torch.Tensor):
    """A CPU tensor that passes for a device tensor, so that the refusals that
    need one can be seen without a GPU (nothing is launched)."""

    @property
    def is_cuda(self):
        return True


def _dev(t):
    return t.as_subclass(_OnDevice)


def _dev_cache(**kw):
    c = _cache(**kw)
    return SwitchKVCache(*(_dev(t) for t in (c.k, c.v, c.k_scales, c.v_scales)), c.block_size)


def _swap(c, **kw):
    return SwitchKVCache(**{**{f: getattr(c, f) for f in ("k", "v", "k_scales", "v_scales", "block_size")}, **kw})


@pytest.mark.parametrize("change,error,words", [
    (dict(k=torch.zeros(2, 40, 2, 128)), TypeError, "float8_e4m3fn or int8"),
    (dict(v=torch.zeros(2, 40, 2, 128, dtype=torch.float8_e4m3fn)), TypeError, "alike"),
    (dict(k_scales=torch.ones(2, 2, 3, dtype=torch.float64)), TypeError, "FP32"),
    (dict(block_size=24), ValueError, "block_size"),
    (dict(v=torch.zeros(2, 41, 2, 128, dtype=torch.int8)), ValueError, "alike"),
    (dict(v_scales=torch.ones(2, 2, 2)), ValueError, "ceil"),
    (dict(block_size=32), ValueError, "ceil"),
    (dict(v=torch.zeros(2, 40, 128, 2, dtype=torch.int8).transpose(2, 3)), ValueError, "contiguous"),
])
def test_a_broken_cache_is_refused_everywhere(change, error, words):
    cache = _swap(_dev_cache(), **change)
    lens = torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16)
    for call in (lambda: switch_kv_cache_append(cache, rows, rows, lens),
                 lambda: switch_kv_cache_read(cache, 0, 3),
                 lambda: switch_gqa_decode_quantized_forward(rows, cache, lens, lens > 0),
                 lambda: switch_kv_cache_evict(cache, lens, torch.zeros(2, 2, 40), budget=3, recent=1)):
        with pytest.raises(error, match=words):
            call()


def test_arguments_that_are_no_tensors_are_refused():
    a = np.zeros((2, 40, 2, 128), np.int8)
    with pytest.raises((TypeError, AttributeError)):
        switch_kv_cache_read(SwitchKVCache(a, a, a, a, 16), 0, 3)


def test_host_caches_are_refused():
    with pytest.raises(ValueError, match="accelerator"):
        switch_kv_cache_read(_cache(), 0, 3)
    with pytest.raises(ValueError, match="accelerator"):
        build_switch_kv_cache(1, 4, 1, device="cpu")
    with pytest.raises(TypeError, match="codes"):
        build_switch_kv_cache(1, 4, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="block_size"):
        build_switch_kv_cache(1, 4, 1, device="cuda", block_size=8)
    with pytest.raises(ValueError, match="at least one"):
        build_switch_kv_cache(1, 0, 1, device="cuda")


def test_append_refusals():
    c = _dev_cache()
    lens = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 3, 2, 128, dtype=torch.bfloat16)
    for args, kw, error, words in (
            ((x.float(), x, lens), {}, TypeError, "BF16"),
            ((x[:, :2], x, lens), {}, ValueError, "one shape"),
            ((x[:1], x[:1], lens), {}, ValueError, "batch sizes"),
            ((x[..., :64], x[..., :64], lens), {}, ValueError, "KV heads"),
            ((x.transpose(0, 1).contiguous().transpose(0, 1),) * 2 + (lens,), {}, ValueError, "contiguous"),
            ((x, x, lens.long()), {}, ValueError, "cache_lens"),
            ((x, x, lens[:1]), {}, ValueError, "cache_lens"),
            ((x, x, lens), dict(row_counts=lens.long()), ValueError, "row_counts"),
            ((x, x, lens), dict(row_counts=lens, cu_seqlens=[0, 1, 3]), ValueError, "exclude"),
            ((x, x, lens), dict(cu_seqlens=[0, 1, 3]), ValueError, "batch size 1"),
            ((x[:1], x[:1], lens), dict(cu_seqlens=[0, 3]), ValueError, "one sequence for each"),
            ((x[:1], x[:1], lens), dict(cu_seqlens=[0, 2, 1]), ValueError, "non-decreasing"),
            ((x[:1], x[:1], lens), dict(cu_seqlens=[0, 2, 4]), ValueError, "end at"),
            ((torch.zeros(2, 41, 2, 128, dtype=torch.bfloat16),) * 2 + (lens,), {}, ValueError, "more rows")):
        with pytest.raises(error, match=words):
            switch_kv_cache_append(c, *args, **kw)
    with pytest.raises(ValueError, match="overlap"):
        switch_kv_cache_append(_swap(c, v=c.k), x, x, lens)
    with pytest.raises(ValueError, match="negative"):
        switch_kv_cache_read(c, 0, -1)
    with pytest.raises(ValueError, match="negative"):
        switch_kv_cache_read(c, -1, 1)
    with pytest.raises(ValueError, match="starts"):
        switch_kv_cache_read(c, lens.long(), 1)


def test_decode_and_evict_refusals():
    c = _dev_cache()
    lens, full = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.bool)
    q, w = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 40)
    call = switch_gqa_decode_quantized_forward
    for args, kw, error, words in (
            ((q.float(), c, lens, full), {}, TypeError, "BF16"),
            ((q[..., :64], c, lens, full), {}, ValueError, "contiguous"),
            ((q.repeat(1, 2, 1, 1), c, lens, full), {}, ValueError, "Hq"),
            ((q[:1], c, lens, full), {}, ValueError, "batch sizes"),
            ((q[:, :, :3].contiguous(), c, lens, full), {}, ValueError, "multiple"),
            ((q.repeat(1, 1, 5, 1), c, lens, full), {}, ValueError, "multiple"),
            ((q, c, lens, full), dict(window_size=0), ValueError, "window_size"),
            ((q, c, lens.long(), full), {}, ValueError, "cache_lens"),
            ((q, c, lens, lens), {}, ValueError, "full_mask"),
            ((q, c, lens, full), dict(key_weights=w.double()), TypeError, "FP32"),
            ((q, c, lens, full), dict(key_weights=w[:, :, :39]), ValueError, "Hkv,L"),
            ((q, c, lens, full), dict(key_weights=w.transpose(0, 1).contiguous().transpose(0, 1)), ValueError,
             "contiguous")):
        with pytest.raises(error, match=words):
            call(*args, **kw)
    ok = dict(budget=10, recent=3)
    other = _dev_cache()
    for args, kw, error, words in (
            ((c, lens, w), dict(ok, budget=0), ValueError, "budget"),
            ((c, lens, w), dict(ok, recent=11), ValueError, "recent"),
            ((c, lens, w), dict(ok, recent=-1), ValueError, "recent"),
            ((c, lens, w), dict(ok, capacity=9), ValueError, "at least budget"),
            ((c, lens, w[:1]), ok, ValueError, "Hkv,L"),
            ((c, lens, w), dict(ok, out=other), ValueError, "go together"),
            ((c, lens, w), dict(ok, out=other, out_weights=w.clone(), capacity=40), ValueError, "exclude"),
            ((c, lens, w), dict(ok, out=_dev_cache(block=32), out_weights=w.clone()), ValueError, "block_size"),
            ((c, lens, w), dict(ok, out=_dev_cache(h=1), out_weights=w.clone()), ValueError, "KV heads"),
            ((c, lens, w), dict(ok, out=_dev_cache(n=9), out_weights=w[:, :, :9].clone()), ValueError, "budget"),
            ((c, lens, w), dict(ok, out=other, out_weights=w[:, :, :9].clone()), ValueError, "Hkv,L"),
            ((c, lens, w), dict(ok, out=c, out_weights=w.clone()), ValueError, "share memory"),
            ((c, lens, w), dict(ok, out=other, out_weights=w), ValueError, "share memory"),
            ((c, lens, w), dict(ok, out=_swap(other, v=other.k), out_weights=w.clone()), ValueError,
             "share memory")):
        with pytest.raises(error, match=words):
            switch_kv_cache_evict(*args, **kw)


def test_oracle_e4m3_equals_torchs_cast():
    """Every value of the format, the midpoints between them and their neighbours."""
    t = C._TABLE
    assert np.array_equal(torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy(), t)
    mid = (t[1:] + t[:-1]) / 2
    x = np.concatenate([t, mid, np.nextafter(np.float32(mid), np.float32(0)), np.nextafter(np.float32(mid), np.float32(1e9))])
    x = np.concatenate([x, -x]).astype(np.float32)
    assert np.array_equal(C.round_code(x, torch.float8_e4m3fn),
                          torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


def test_oracle_scales_are_the_smallest_that_hold():
    for dtype, qmax in C.QMAX.items():
        for a in (qmax, qmax * 1.001, qmax * 0.999, 1e-35, 3.3e38, 1.0, 0.75):
            s = C.scale_for(a, dtype)
            assert a <= qmax * s and math.log2(s) == int(math.log2(s))
            assert s == 2.0 ** C.MIN_EXP or a > qmax * s / 2
        assert C.scale_for(0.0, dtype) == 2.0 ** C.MIN_EXP and math.isnan(C.scale_for(math.inf, dtype))


def test_oracle_decode_against_a_loop():
    gen = torch.Generator().manual_seed(0)
    q = torch.randn(1, 2, 128, generator=gen).to(torch.bfloat16)
    k, v = (torch.randn(1, 5, 1, 128, generator=gen).double().numpy() for _ in range(2))
    o, lse, w, _ = C.decode(q, k, v, [5], [False], 3)
    for h in range(2):
        e = [math.exp(sum(float(q[0, h, i]) * k[0, j, 0, i] for i in range(128)) / math.sqrt(128)) for j in (2, 3, 4)]
        assert abs(lse[0, h] - math.log2(sum(e))) < 1e-12
        assert np.allclose(o[0, h], sum(x * v[0, j, 0] for x, j in zip(e, (2, 3, 4))) / sum(e))
    assert np.allclose(w.sum(), 2.0) and not w[0, 0, :2].any()


def test_public_names():
    import switchattentionkernels_amd as swa
    for name in ("SwitchKVCache", "build_switch_kv_cache", "switch_kv_cache_append", "switch_kv_cache_read",
                 "switch_gqa_decode_quantized_forward", "switch_kv_cache_evict",
                 "switch_gqa_prefill_key_weights"):
        assert name in swa.__all__ and hasattr(swa, name)
    assert cache_module.BLOCK_SIZES == (16, 32, 64, 128) and decode.LOG2E == math.log2(math.e)
