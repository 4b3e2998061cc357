"""Norm and rotation of queries and keys without a GPU: the C ABI, its refusals, and the
oracle against another way to write it."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

from oracle import rotary as R
import switchattentionkernels_amd as sw
from switchattentionkernels_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, P2, ODD = ctypes.c_void_p(256), ctypes.c_void_p(512), ctypes.c_void_p(264)


def test_library_exports_what_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "swattn_rotary.h")).read(), flags=re.S)
    found = {m.group(1): len([a for a in m.group(2).split(",") if a.strip()])
             for m in re.finditer(r"\b(swattn_\w+)\s*\(([^)]*)\)\s*;", text)}
    assert set(found) == set(_lib.ROTARY_SIGNATURES)
    for name, n in found.items():
        assert hasattr(_lib.lib(), name) and len(_lib.ROTARY_SIGNATURES[name][1]) == n, name


def _ints(kind, *x):
    return (kind * len(x))(*x)


GOOD = dict(q=P, qs=(128, 128, 128), k=P, ks=(128, 128, 128), pos=P, freq=P, sections=(64,), axes=1, eps=1e-6, out=P,
            batch=2, seq=3, hq=4, hkv=2, dim=128)


def _how(a):
    sections = _ints(ctypes.c_int32, *a["sections"]) if a["sections"] is not None else None
    return a["pos"], a["freq"], 1, sections, a["axes"], 0, P, P, 0, ctypes.c_float(a["eps"])


def _strides(s):
    return None if s is None else _ints(ctypes.c_int64, *s)


def _fwd(**change):
    a = dict(GOOD, **change)
    return _lib.lib().swattn_rotary_fwd(a["q"], _strides(a["qs"]), a["k"], _strides(a["ks"]), *_how(a), a["out"], a["out"],
                                        a["batch"], a["seq"], a["hq"], a["hkv"], a["dim"], None)


def _append(**change):
    a = dict(dict(GOOD, v=P, vs=(0, 128, 128), kc=P, vc=P, lens=P, lens_out=P2, cap=10), **change)
    return _lib.lib().swattn_rotary_append(
        a["q"], _strides(a["qs"]), a["k"], _strides(a["ks"]), a["v"], _strides(a["vs"]), *_how(a), a["out"], a["kc"],
        a["vc"], a["lens"], None, a["lens_out"], a["batch"], a["seq"], a["cap"], a["hq"], a["hkv"], a["dim"], None)


def _bwd(**change):
    a = dict(dict(GOOD, g=P, dwq=P, ws=P, ws_bytes=1 << 30, qw=P), **change)
    how = list(_how(a))
    how[6] = a["qw"]
    return _lib.lib().swattn_rotary_bwd(a["g"], P, a["q"], _strides(a["qs"]), a["k"], _strides(a["ks"]), *how, a["out"],
                                        a["out"], a["dwq"], None, a["batch"], a["seq"], a["hq"], a["hkv"], a["dim"],
                                        a["ws"], a["ws_bytes"], None)


def _refused(status, words, code=-1):
    assert status == code, (status, _lib.lib().swattn_last_error())
    assert words.encode() in _lib.lib().swattn_last_error(), _lib.lib().swattn_last_error()


@pytest.mark.parametrize("call", [_fwd, _append, _bwd])
def test_c_abi_refusals(call):
    _refused(call(dim=64), "head_dim")
    _refused(call(batch=0), "bad shape")
    _refused(call(seq=-1), "bad shape")
    _refused(call(hq=0), "bad shape")
    _refused(call(batch=1 << 16, seq=1 << 15), "too large")
    _refused(call(hq=65536), "too large")
    _refused(call(pos=None), "null")
    _refused(call(freq=None), "null")
    _refused(call(sections=None), "null")
    _refused(call(axes=5, sections=(8,) * 5), "axes")
    _refused(call(axes=0), "axes")
    _refused(call(sections=(0,)), "positive")
    _refused(call(axes=2, sections=(72, -8)), "positive")
    _refused(call(sections=(60,)), "frequencies")
    _refused(call(sections=(72,)), "frequencies")
    for change in (dict(q=None), dict(k=ODD), dict(qs=None), dict(qs=(128, 4, 128)), dict(ks=(-128, 128, 128))):
        _refused(call(**change), "strides")
    _refused(call(out=ODD), "16-byte")


def test_c_abi_refusals_of_one_call():
    _refused(_append(cap=0), "cache_len")
    _refused(_append(cap=2 ** 31), "cache_len")
    _refused(_append(v=None), "strides")
    _refused(_append(kc=None), "null")
    _refused(_append(vc=ODD), "16-byte")
    _refused(_append(lens=None), "null")
    _refused(_append(lens_out=P), "alias")
    _refused(_bwd(g=ODD), "16-byte")
    _refused(_bwd(qw=None), "needs the weight")
    _refused(_bwd(ws=None), "workspace", -2)
    _refused(_bwd(ws_bytes=255), "workspace", -2)
    _refused(_bwd(ws=ODD), "256-byte")
    assert _fwd(seq=0) == 0                       # nothing to do, nothing launched
    L = _lib.lib()
    assert L.swattn_rotary_bwd_workspace_bytes(0, 3, 4, 2) == 0
    # One partial of 512 bytes for each of a tensor's workgroups of four tokens.
    assert L.swattn_rotary_bwd_workspace_bytes(2, 3, 4, 2) == 512 * (2 + 2)


def test_python_refuses_what_is_not_on_a_gpu():
    q, k = (torch.zeros(1, 2, h, 128, dtype=torch.bfloat16) for h in (4, 2))
    pos, freq = torch.zeros(1, 1, 2, dtype=torch.int32), torch.ones(64)
    with pytest.raises(ValueError, match="accelerator"):
        sw.switch_qk_rotary_forward(q, k, pos, freq)
    with pytest.raises(TypeError, match="BF16"):
        sw.switch_qk_rotary_forward(q.float(), k, pos, freq)
    with pytest.raises(TypeError, match="BF16"):
        sw.switch_qk_rotary_forward(np.zeros((1, 2, 4, 128)), k, pos, freq)
    with pytest.raises(ValueError, match="accelerator"):
        sw.switch_qk_rotary_append(q, k, k, k, k, pos[0, 0], pos, freq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_is_a_product_of_complex_numbers(interleaved):
    rng = np.random.default_rng(0)
    x, n = rng.standard_normal((2, 3, 2, 128)), 24
    pos, freq = rng.integers(-99, 99, (3, 2, 3)), 10.0 ** -rng.random(n)
    cos, sin = R.unit(pos, freq, [4, 12, 8])
    got, _ = R.forward(x, None, 0.0, cos, sin, interleaved)
    axis = [0] * 4 + [1] * 12 + [2] * 8
    for b, s, i in np.ndindex(2, 3, n):
        a, c = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        z = (x[b, s, :, a] + 1j * x[b, s, :, c]) * np.exp(1j * pos[axis[i], b, s] * freq[i])
        assert np.allclose(got[b, s, :, a], z.real, atol=1e-12) and np.allclose(got[b, s, :, c], z.imag, atol=1e-12)
    assert np.array_equal(got[..., 2 * n:], x[..., 2 * n:])


def test_oracle_gradients_are_those_of_autograd():
    torch.manual_seed(0)
    x = torch.randn(2, 3, 2, 128, dtype=torch.float64, requires_grad=True)
    w = torch.randn(128, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(2, 3, 2, 128, dtype=torch.float64)
    pos, freq = np.arange(6).reshape(1, 2, 3), np.linspace(0.1, 1, 64)
    cos, sin = R.unit(pos, freq, [64])
    u = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-3) * w
    c, s = torch.from_numpy(cos), torch.from_numpy(sin)
    y = torch.cat([u[..., :64] * c - u[..., 64:] * s, u[..., 64:] * c + u[..., :64] * s], dim=-1)
    want = torch.autograd.grad(y, (x, w), dy)
    dx, _, dw, _ = R.backward(R.np64(dy), R.np64(x), R.np64(w), 1e-3, cos, sin, False)
    assert np.allclose(dx, want[0].numpy(), atol=1e-10) and np.allclose(dw, want[1].numpy(), atol=1e-10)
