"""Decode behind shared prefixes without a GPU: the C ABI, its refusals, the bounds that the
workspace relies on, and the oracle."""

import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

import oracle
from oracle import shared as S
import switchattentionkernels_amd as sw
from switchattentionkernels_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def test_library_exports_what_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "swattn_shared.h")).read(), flags=re.S)
    found = {m.group(1): len([a for a in m.group(2).split(",") if a.strip()])
             for m in re.finditer(r"\b(swattn_\w+)\s*\(([^)]*)\)\s*;", text)}
    assert set(found) == set(_lib.SHARED_SIGNATURES)
    for name, n in found.items():
        assert hasattr(_lib.lib(), name) and len(_lib.SHARED_SIGNATURES[name][1]) == n, name


def _call(**change):
    a = dict(dict(q=P, kp=P, kc=P, full=P, out=P, batch=2, cap=10, prefixes=1, plen=20, hq=8, hkv=2, dim=128, window=4, scale=0.1,
                  ws=P, ws_bytes=1 << 40), **change)
    return _lib.lib().swattn_shared_decode_fwd(
        a["q"], a["kp"], P, P, P, a["kc"], P, P, a["full"], a["out"], P, a["batch"], a["cap"], a["prefixes"], a["plen"],
        a["hq"], a["hkv"], a["dim"], a["window"], ctypes.c_float(a["scale"]), a["ws"], a["ws_bytes"], None)


def _refused(status, words, code=-1):
    assert status == code, (status, _lib.lib().swattn_last_error())
    assert words.encode() in _lib.lib().swattn_last_error(), _lib.lib().swattn_last_error()


def test_c_abi_refusals():
    _refused(_call(dim=64), "head_dim")
    for name in ("batch", "cap", "prefixes", "plen", "hq", "hkv"):
        _refused(_call(**{name: 0}), "bad shape")
    _refused(_call(hq=9), "multiple")
    _refused(_call(hq=18), "at most 8")
    _refused(_call(window=0), "window")
    _refused(_call(batch=1025), "too large")
    _refused(_call(prefixes=1025), "too large")
    _refused(_call(cap=2 ** 31), "too large")
    _refused(_call(cap=2 ** 29), "too large")       # 2 x 2 pairs of them, with their starts
    _refused(_call(plen=2 ** 30), "too large")      # two tiles x 2 KV heads
    _refused(_call(q=None), "null")
    _refused(_call(full=None), "null")
    _refused(_call(kp=ODD), "16-byte")
    _refused(_call(out=ODD), "16-byte")
    _refused(_call(ws=None), "workspace", -2)
    _refused(_call(ws_bytes=_lib.lib().swattn_shared_decode_workspace_bytes(2, 10, 1, 20, 8, 2) - 1), "workspace", -2)
    _refused(_call(ws=ODD), "256-byte")


def test_workspace_holds_every_part():
    """512 shares of the line and 64 more where pieces leave it few, one per pair beside;
    as many prefix pieces and one per (tile, KV head), with a tile's rows each."""
    L = _lib.lib()

    def al(x):
        return -(-x // 256) * 256

    cus = 256   # also what the library assumes where it finds no device
    for batch, prefixes, hq, hkv in ((1, 1, 8, 8), (64, 1, 32, 8), (40, 3, 40, 8), (1024, 1024, 8, 1), (1000, 2, 64, 8)):
        g = hq // hkv
        seqs = 128 // g
        tiles = min(batch, 2 * prefixes + batch // seqs)
        slots, pieces = 2 * cus + 2 * cus // 8 + batch * hkv, 2 * cus + tiles * hkv
        rows = min(batch, seqs) * g
        want = (al(slots * g * 512) + al(slots * g * 8) + al(16 * (1 + batch)) + al(16 * batch) + al(pieces * rows * 512)
                + al(pieces * rows * 8))
        assert L.swattn_shared_decode_workspace_bytes(batch, 100, prefixes, 100, hq, hkv) == want
    assert L.swattn_shared_decode_workspace_bytes(1025, 100, 1, 100, 8, 8) == 0


def test_launches_of_2_32_threads_are_refused():
    """256 threads per output row (prefix pieces are fewer: positions below 2^31 leave 2^24 / 1.5)."""
    size = _lib.lib().swattn_shared_decode_workspace_bytes
    rows = 2 ** 24
    assert size(1024, 1, 1, 1, rows // 1024, rows // 1024 // 8) == 0
    assert size(1023, 1, 1, 1, rows // 1024, rows // 1024 // 8) > 0
    for scale in (math.nan, math.inf, -math.inf):
        _refused(_call(scale=scale), "scale_log2")


def test_planned_pieces_stay_within_the_workspace():
    """The device's arithmetic for random lengths: no more pieces than the workspace and the
    grid hold, none empty, every key in one of them, shares of the line within theirs."""
    rng = np.random.default_rng(0)
    target, cost16, least = 512, 24, 64
    for _ in range(3000):
        g, hkv = int(rng.integers(1, 9)), int(rng.integers(1, 17))
        seqs = 128 // g
        prefixes, batch = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 10))
        plen, cap = int(2 ** rng.uniform(0, 17)), int(2 ** rng.uniform(0, 15))
        ids, local = rng.integers(-1, prefixes, batch), rng.integers(0, 2, batch)
        keys = rng.integers(0, cap + 1, batch)
        line = int((keys.sum() + 192 * (keys > 0).sum()) * hkv)
        groups = []
        for i in range(2 * prefixes):
            cnt = int(((ids == i // 2) & (local == i % 2)).sum())
            n = int(rng.integers(0, plen + 1))
            if cnt and n:
                groups.append((-(-cnt // seqs), n))
        tiles = sum(t for t, _ in groups)
        bound = target + min(batch, 2 * prefixes + batch // seqs) * hkv
        positions = sum(t * n for t, n in groups)
        cost = line + -(-positions * hkv * cost16 // 16)
        share = (cost * -(-2 ** 32 // target) >> 32) + 1       # cost / target at least
        assert share * target >= cost and share <= cost // target + 2
        length = -(-max(-(-share * 16 // cost16), -(-plen // 255), 64) // 64) * 64
        pieces = 0
        for t, n in groups:
            parts = -(-n // length)
            each = -(-(-(-n // parts)) // 64) * 64
            parts = -(-n // each)
            assert 1 <= parts <= 255 and (parts - 1) * each < n <= parts * each
            pieces += t * hkv * parts
        assert pieces <= bound and tiles <= min(batch, 2 * prefixes + batch // seqs)
        left = max(target - pieces, least)
        assert left <= bound + least - pieces


def test_python_refuses_what_is_not_on_a_gpu():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="accelerator"):
        sw.switch_gqa_decode_shared_forward(z(1, 1, 4, 128), z(1, 5, 2, 128), z(1, 5, 2, 128), i, i, z(1, 3, 2, 128),
                                            z(1, 3, 2, 128), i, i == 0)
    with pytest.raises(TypeError, match="BF16"):
        sw.switch_gqa_decode_shared_forward(None, *[i] * 8)


def test_oracle_is_the_decode_over_one_cache():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, kp, vp, kc, vc = r(3, 4, 128), r(2, 20, 2, 128), r(2, 20, 2, 128), r(3, 9, 2, 128), r(3, 9, 2, 128)
    ids, plens, lens, full = [1, 0, -1], [13, 20], [4, 9, 2], [True, False, False]
    o, lse, _, _ = S.decode(*(x.double().numpy() for x in (q, kp, vp)), plens, ids, kc.double().numpy(),
                            vc.double().numpy(), lens, full, 12)
    for b, i in enumerate(ids):
        n = plens[i] if i >= 0 else 0
        k, v = (torch.cat([p[i, :n], c[b, :lens[b]]])[None] for p, c in ((kp, kc), (vp, vc)))
        ro, rl = oracle.decode_attention(q[b:b + 1], k, v, torch.tensor([n + lens[b]], dtype=torch.int32),
                                         torch.tensor([full[b]]), window_size=12)
        assert np.allclose(o[b], ro[0].numpy(), atol=1e-5) and np.allclose(lse[b], rl[0].numpy(), atol=1e-4)
