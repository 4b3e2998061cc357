"""Decode behind shared prefixes on the GPU against 64 bits (``oracle/shared.py``, where
the bounds are derived)."""

import math

import numpy as np
import pytest
import torch

from oracle import shared as S
from switchattentionkernels_amd import (switch_gqa_decode_forward, switch_gqa_decode_shared_forward,
                                        switch_qk_rotary_append, switch_qk_rotary_forward)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _np(t):
    return t.double().cpu().numpy()


def _rows(gen, *shape, spread=0.35):
    x = torch.randn(*shape, generator=gen) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=gen))
    return x.to(BF16)


def _case(seed, prefix_lens, prefix_cap, ids, lens, cap, hq, hkv, full, garbage=True):
    """CPU rows; rows behind the lengths hold NaN and infinities."""
    gen = torch.Generator().manual_seed(seed)
    b, p = len(ids), len(prefix_lens)
    c = dict(q=_rows(gen, b, 1, hq, 128, spread=0.0), plens=list(prefix_lens), ids=list(ids), lens=list(lens),
             full=list(full), gen=gen)
    for name in ("k", "v"):
        c[name + "p"], c[name + "c"] = _rows(gen, p, prefix_cap, hkv, 128), _rows(gen, b, cap, hkv, 128)
        if garbage:
            bad = torch.tensor([math.nan, math.inf, -math.inf], dtype=BF16)
            for x, ends in ((c[name + "p"], prefix_lens), (c[name + "c"], lens)):
                for i, n in enumerate(ends):
                    rest = x[i, min(max(n, 0), x.shape[1]):]
                    rest[:] = bad[torch.randint(0, 3, rest.shape, generator=gen)]
    return c


def _up(c):
    return [c["q"].to(DEV), c["kp"].to(DEV), c["vp"].to(DEV), _int32(c["plens"]), _int32(c["ids"]), c["kc"].to(DEV),
            c["vc"].to(DEV), _int32(c["lens"]), torch.tensor(c["full"], device=DEV)]


def _check(c, window, sm_scale=None, got=None):
    if got is None:
        got = switch_gqa_decode_shared_forward(*_up(c), window_size=window, sm_scale=sm_scale)
    o, lse = got
    assert o.dtype == BF16 and o.shape == c["q"].shape and lse.shape == c["q"].shape[:3]
    ro, rl, d_o, d_lse = S.decode(_np(c["q"][:, 0]), _np(c["kp"]), _np(c["vp"]), c["plens"], c["ids"], _np(c["kc"]),
                                  _np(c["vc"]), c["lens"], c["full"], window, sm_scale)
    go, gl = _np(o[:, 0]), _np(lse[:, 0])
    wrong = int((np.isnan(go) != np.isnan(ro)).sum()), int((np.isinf(go) != np.isinf(ro)).sum())
    assert wrong == (0, 0)
    ok = np.isfinite(ro)
    assert bool((go[np.isinf(ro)] == ro[np.isinf(ro)]).all())
    worst = (np.abs(go[ok] - ro[ok]) / d_o[ok]).max(initial=0.0)
    assert worst <= 1.0, worst
    assert np.array_equal(np.isnan(gl), np.isnan(rl)) and np.array_equal(np.isneginf(gl), np.isneginf(rl))
    ok = np.isfinite(rl)
    assert (np.abs(gl[ok] - rl[ok]) <= d_lse[ok]).all()
    return o, lse


EDGES = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 200, 257, 300]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (6, 2), (8, 2), (5, 1), (12, 2), (7, 1), (16, 2), (3, 3)])
@pytest.mark.parametrize("window", [1, 50, 100, 1000])
def test_lengths_and_windows(hq, hkv, window):
    """Every prefix length at the edges of a tile, own lengths from 0 on; windows inside the
    own rows, into the prefix and past its start; both routes."""
    n = len(EDGES)
    ids = list(range(n)) * 2
    lens = [(7 * i) % 41 for i in range(2 * n)]
    lens[0] = lens[n] = 0
    c = _case(window, EDGES, 320, ids, lens, 41, hq, hkv, [i < n for i in range(2 * n)])
    _check(c, window)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 2), (10, 2), (16, 2)])
@pytest.mark.parametrize("batch", [1, 15, 33, 130])
def test_many_rows_of_one_prefix(hq, hkv, batch):
    """Tiles that end inside a wave, and several tiles, of both routes."""
    lens = [(13 * i) % 70 for i in range(batch)]
    c = _case(batch, [333], 333, [0] * batch, lens, 70, hq, hkv, [i % 3 > 0 for i in range(batch)])
    _check(c, 90)


def test_no_prefix_and_ids_outside():
    ids = [-1, 0, 2, 2 ** 31 - 1, -2 ** 31, 1, 1, 0]
    c = _case(3, [40, 0], 64, ids, [9, 0, 0, 12, 5, 0, 3, 4], 12, 8, 2, [True, True, False, True, False, True, False, False])
    o, lse = _check(c, 6)
    assert torch.isnan(o[2]).all() and torch.isneginf(lse[2]).all() and torch.isnan(o[5]).all()


def test_lengths_outside_their_range_are_clamped():
    c = _case(4, [70, 30], 64, [0, 1, 0, 1], [20, -3, 11, 12], 12, 4, 2, [True, False, False, True], garbage=False)
    c["plens"][1] = -5
    _check(c, 40)


def test_as_over_one_cache():
    """The same rows in one cache: the other decode step gives the same to rounding."""
    b, lp, cap = 6, 500, 60
    c = _case(5, [lp], lp, [0] * b, [60, 1, 33, 17, 48, 5], cap, 32, 8, [True, False] * 3, garbage=False)
    o, lse = switch_gqa_decode_shared_forward(*_up(c), window_size=100)
    k, v = (torch.cat([c[x + "p"].expand(b, -1, -1, -1), c[x + "c"]], dim=1).to(DEV) for x in "kv")
    want, want_lse = switch_gqa_decode_forward(c["q"].to(DEV), k, v, _int32([lp + n for n in c["lens"]]),
                                               torch.tensor(c["full"], device=DEV), window_size=100)
    assert (o.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()
    assert (lse - want_lse).abs().max() <= 1e-4
    squeezed, _ = switch_gqa_decode_shared_forward(*[_up(c)[0][:, 0]] + _up(c)[1:], window_size=100)
    assert torch.equal(squeezed, o[:, 0])


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    gen = torch.Generator().manual_seed(100 + seed)
    rand = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))  # noqa: E731
    p, b, cap, lp = rand(1, 5), rand(1, 70), rand(1, 200), rand(1, 1500)
    hkv = rand(1, 4)
    c = _case(seed, [rand(0, lp) for _ in range(p)], lp, [rand(-1, p - 1) for _ in range(b)],
              [rand(0, cap) for _ in range(b)], cap, hkv * rand(1, 8), hkv, [rand(0, 1) == 1 for _ in range(b)])
    _check(c, rand(1, 700))


def test_largest_batch_and_number_of_prefixes():
    """1024 sequences over 1024 prefixes (each a tile of its own), and over one."""
    ids = [(7 * i) % 1024 for i in range(1024)]
    c = _case(7, [(i % 9) for i in range(1024)], 8, ids, [i % 4 for i in range(1024)], 3, 2, 1,
              [i % 2 == 0 for i in range(1024)])
    _check(c, 5)
    c = _case(8, [200], 200, [0] * 1024, [i % 4 for i in range(1024)], 3, 2, 1, [i % 2 == 0 for i in range(1024)])
    _check(c, 50)


@pytest.mark.parametrize("batch,prefixes", [(256, 256), (257, 3), (5, 257), (300, 700)])
def test_plans_of_one_and_of_four_per_thread(batch, prefixes):
    gen = torch.Generator().manual_seed(batch)
    ids = torch.randint(-1, prefixes, (batch,), generator=gen).tolist()
    ids[0], ids[-1] = 0, prefixes - 1
    c = _case(18, [(11 * i) % 70 for i in range(prefixes)], 70, ids, [(5 * i) % 12 for i in range(batch)], 11, 4, 2,
              [i % 3 != 1 for i in range(batch)])
    _check(c, 20)


def test_long_prefix_in_many_pieces():
    c = _case(9, [20000], 20011, [0, 0, 0], [7, 300, 2], 300, 4, 1, [True, True, False])
    _check(c, 5000)


def test_scales():
    """A negative one, 0, a large one."""
    c = _case(10, [90], 90, [0] * 5, [3, 9, 4, 0, 1], 9, 8, 2, [True, False, True, True, False])
    for scale in (-0.3, 0.0, 2.0):
        _check(c, 20, scale)


@pytest.mark.parametrize("where", ["prefix", "own"])
def test_values_that_are_not_finite(where):
    """NaN and infinities in valid rows reach the rows that attend them and no others: local
    rows of the same tile, whose windows begin behind them, among those."""
    b, lp, cap = 12, 150, 20
    full = [i % 3 == 0 for i in range(b)]
    for name, value in (("v", math.inf), ("v", math.nan), ("k", math.nan), ("v", -math.inf)):
        c = _case(11, [lp], lp, [0] * b, [1 + i for i in range(b)], cap, 8, 2, full)
        if where == "prefix":
            for at, head, dim in ((149, 0, 3), (130, 1, 77), (128, 0, 64), (101, 1, 127), (64, 0, 31)):
                c[name + "p"][0, at, head, dim] = value
        else:
            c[name + "c"][4, 2, 0, 5] = c[name + "c"][7, 7, 1, 100] = value
        o, _ = _check(c, 30)
        odd = ~torch.isfinite(o[:, 0].float()).all(dim=-1).cpu()
        assert odd.any() and not odd.all()


def test_scores_past_the_range_of_fp32():
    """Scores of -inf ahead of finite ones weigh nothing."""
    c = _case(12, [100], 100, [0, 0], [40, 5], 40, 4, 2, [True, False])
    c["q"].fill_(3e38)
    c["kp"].zero_(), c["kc"].zero_()
    c["kp"][0, :70], c["kc"][:, :3] = -3e38, -3e38
    c["vp"][0, :70], c["vc"][:, :3] = 1e4, 1e4
    o, lse = switch_gqa_decode_shared_forward(*_up(c), window_size=60)
    for i, (n, keys) in enumerate(((40, 30 + 37), (5, 30 + 2))):
        v = torch.cat([c["vp"][0, 70:], c["vc"][i, 3:n]]).float().mean(dim=0)      # [Hkv, 128]
        assert torch.allclose(o[i, 0].float().cpu(), v.repeat_interleave(2, dim=0), rtol=2 ** -8, atol=1e-5)
        assert torch.allclose(lse[i].cpu(), torch.full((1, 4), math.log2(keys)), rtol=1e-6)


def test_repeats_are_bit_identical_and_other_streams_agree():
    c = _case(13, [700, 90], 700, [0, 1] * 20, [(3 * i) % 50 for i in range(40)], 50, 32, 8, [i % 4 == 0 for i in range(40)])
    args = _up(c)
    o, lse = switch_gqa_decode_shared_forward(*args, window_size=80)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:                           # calls at once, each with a workspace of its own
        with torch.cuda.stream(s):
            got.append(switch_gqa_decode_shared_forward(*args, window_size=80))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a.view(torch.int16), o.view(torch.int16)) and torch.equal(b, lse)


def test_captured_and_replayed():
    """Lengths, routes and prefixes change between replays."""
    c = _case(14, [300, 40], 310, [0, 1, 0, -1, 0], [5, 9, 0, 3, 20], 24, 8, 2, [True, False, False, True, False], garbage=False)
    args = _up(c)
    switch_gqa_decode_shared_forward(*args, window_size=64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = switch_gqa_decode_shared_forward(*args, window_size=64)
    for plens, ids, lens, full in (([300, 40], [0, 1, 0, -1, 0], [5, 9, 0, 3, 20], [1, 0, 0, 1, 0]),
                                   ([310, 0], [1, 1, 1, 1, 1], [24, 1, 2, 3, 4], [1, 1, 1, 0, 0]),
                                   ([1, 300], [1, 0, 1, 0, 1], [0, 0, 0, 0, 0], [0, 1, 1, 0, 0]),
                                   ([300, 40], [0, 0, 0, 0, 0], [24, 24, 24, 24, 24], [0, 0, 0, 0, 0])):
        for i, x in ((3, plens), (4, ids), (7, lens)):
            args[i].copy_(_int32(x))
        args[8].copy_(torch.tensor(full, device=DEV) == 1)
        args[0].add_(0.25)
        c.update(q=args[0].cpu(), plens=plens, ids=ids, lens=lens, full=[x == 1 for x in full])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        _check(c, 64, got=got)
        want = switch_gqa_decode_shared_forward(*args, window_size=64)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, want))


def test_far_rows():
    """A prefix and own rows whose byte offsets pass 2^32."""
    rows = 1 << 23
    kp, vp = (torch.empty(3, rows, 1, 128, dtype=BF16, device=DEV) for _ in range(2))
    kc, vc = (torch.empty(3, rows, 1, 128, dtype=BF16, device=DEV) for _ in range(2))
    c = _case(15, [77, 150, 140], 150, [2, 1, 2], [6, 9, 30], 30, 4, 1, [True, False, True])
    for big, small in ((kp, "kp"), (vp, "vp"), (kc, "kc"), (vc, "vc")):
        big[:, :c[small].shape[1]] = c[small].to(DEV)
    args = _up(c)
    got = switch_gqa_decode_shared_forward(args[0], kp, vp, args[3], args[4], kc, vc, args[7], args[8], window_size=100)
    _check(c, 100, got=got)


@pytest.mark.parametrize("batch", [5, 70])
def test_a_large_prefix(batch):
    """Of more than 96 MB, with a ragged end: streamed where one tile takes all sequences."""
    n, hkv = 24011, 8
    gen = torch.Generator(device=DEV).manual_seed(batch)
    rows = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(BF16)  # noqa: E731
    q, kp, vp = rows(batch, 1, 16, 128), rows(1, n, hkv, 128), rows(1, n, hkv, 128)
    kc, vc = rows(batch, 40, hkv, 128), rows(batch, 40, hkv, 128)
    lens = _int32([(7 * i) % 41 for i in range(batch)])
    full = torch.tensor([i % 2 == 0 for i in range(batch)], device=DEV)
    plens, ids = _int32([n - 3]), _int32([0] * batch)
    o, lse = switch_gqa_decode_shared_forward(q, kp, vp, plens, ids, kc, vc, lens, full, window_size=700)
    picked = [0, 1, batch - 1]
    c = dict(q=q[picked].cpu(), kp=kp.cpu(), vp=vp.cpu(), kc=kc[picked].cpu(), vc=vc[picked].cpu(), plens=[n - 3],
             ids=[0] * 3, lens=lens[picked].tolist(), full=full[picked].tolist())
    _check(c, 700, got=(o[picked], lse[picked]))


def test_a_serving_loop():
    """Prompts behind a shared prefix, then steps: rotated queries and keys, appended, attended;
    each step against one cache that holds the prefix and the own rows together."""
    gen = torch.Generator().manual_seed(16)
    b, lp, cap, hq, hkv, w = 5, 130, 24, 8, 2, 60
    freq = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).to(DEV)
    weight = (1 + 0.2 * torch.randn(2, 128, generator=gen)).to(DEV)
    how = dict(q_weight=weight[0], k_weight=weight[1])
    rows = lambda n, h: _rows(gen, b, n, h, 128).to(DEV)  # noqa: E731
    # The prefix: position 0 on, kept once.
    pos = torch.arange(lp, dtype=torch.int32, device=DEV)[None]
    kp, vp = _rows(gen, 1, lp, hkv, 128).to(DEV), _rows(gen, 1, lp, hkv, 128).to(DEV)
    _, kp = switch_qk_rotary_forward(kp, kp, pos, freq, k_weight=weight[1])
    plens, ids = _int32([lp]), _int32([0, 0, -1, 0, 0])
    at = torch.where(ids >= 0, plens[0], 0)
    kc, vc = (torch.zeros(b, cap, hkv, 128, dtype=BF16, device=DEV) for _ in range(2))
    one_k, one_v = (torch.zeros(b, lp + cap, hkv, 128, dtype=BF16, device=DEV) for _ in range(2))
    for i in (0, 1, 3, 4):
        one_k[i, :lp], one_v[i, :lp] = kp[0], vp[0]
    lens, one_lens = _int32([0] * b), at.to(torch.int32)
    # Prompts of different lengths, then single tokens.
    counts = _int32([7, 1, 5, 3, 0])
    for n in (7, 1, 1, 1):
        q, k, v = rows(n, hq), rows(n, hkv), rows(n, hkv)
        pos = (at + lens).to(torch.int32)[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)
        cnt = counts if n > 1 else None
        qr, new = switch_qk_rotary_append(q, k, v, kc, vc, lens, pos, freq, row_counts=cnt, **how)
        qr2, one_new = switch_qk_rotary_append(q, k, v, one_k, one_v, one_lens, pos, freq, row_counts=cnt, **how)
        assert torch.equal(qr, qr2)
        lens, one_lens = new, one_new
        if n > 1:
            continue
        full = torch.rand(b, generator=gen).to(DEV) < 0.5
        o, lse = switch_gqa_decode_shared_forward(qr, kp, vp, plens, ids, kc, vc, lens, full, window_size=w)
        want, want_lse = switch_gqa_decode_forward(qr, one_k, one_v, one_lens, full, window_size=w)
        assert (o.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()
        assert (lse - want_lse).abs().max() <= 1e-4
    assert lens.tolist() == [10, 4, 8, 6, 3]


def test_refusals():
    c = _case(17, [9], 12, [0, 0], [3, 4], 6, 4, 2, [True, False])
    names = ("q", "k_prefix", "v_prefix", "prefix_lens", "prefix_ids", "k_cache", "v_cache", "cache_lens", "full_mask")
    ok = dict(zip(names, _up(c)))
    switch_gqa_decode_shared_forward(**ok)
    big = torch.zeros(1025, 1, 2, 128, dtype=BF16, device=DEV)
    bad = [
        (TypeError, "BF16", dict(q=ok["q"].float())),
        (TypeError, "BF16", dict(k_prefix=None)),
        (TypeError, "BF16", dict(v_cache=ok["v_cache"].half())),
        (ValueError, "accelerator", dict(q=ok["q"].cpu())),
        (ValueError, "accelerator", dict(v_prefix=ok["v_prefix"].cpu())),
        (ValueError, "contiguous", dict(k_cache=ok["k_cache"].transpose(1, 2).contiguous().transpose(1, 2))),
        (ValueError, "contiguous", dict(k_prefix=torch.zeros(1 * 12 * 256 + 1, dtype=BF16, device=DEV)[1:].view(1, 12, 2, 128))),
        (ValueError, "q must be", dict(q=ok["q"].expand(2, 2, 4, 128).contiguous())),
        (ValueError, "one shape", dict(v_cache=ok["v_cache"][:, :5].contiguous())),
        (ValueError, "prefixes must be", dict(v_prefix=ok["v_prefix"][:, :5].contiguous())),
        (ValueError, "head_dim", dict(q=ok["q"][..., :64].contiguous())),
        (ValueError, "batch sizes", dict(q=ok["q"][:1])),
        (ValueError, "multiple", dict(q=ok["q"][:, :, :3].contiguous())),
        (ValueError, "multiple", dict(q=torch.zeros(2, 1, 18, 128, dtype=BF16, device=DEV))),
        (ValueError, "prefixes must have", dict(k_prefix=ok["k_prefix"][:, :, :1].contiguous(),
                                               v_prefix=ok["v_prefix"][:, :, :1].contiguous())),
        (ValueError, "at least one", dict(k_prefix=ok["k_prefix"][:, :0], v_prefix=ok["v_prefix"][:, :0])),
        (ValueError, "1024", dict(q=big, k_cache=big, v_cache=big)),
        (ValueError, "1024", dict(k_prefix=big, v_prefix=big)),
        (ValueError, "cache_lens", dict(cache_lens=ok["cache_lens"].long())),
        (ValueError, "prefix_ids", dict(prefix_ids=ok["prefix_ids"][:1])),
        (ValueError, "prefix_lens", dict(prefix_lens=ok["cache_lens"])),
        (ValueError, "full_mask", dict(full_mask=ok["cache_lens"])),
        (ValueError, "window_size", dict(window_size=0)),
        (ValueError, "sm_scale", dict(sm_scale=math.nan)),
        (ValueError, "sm_scale", dict(sm_scale=-math.inf)),
    ]
    for kind, words, change in bad:
        with pytest.raises(kind, match=words):
            switch_gqa_decode_shared_forward(**dict(ok, **change))
    # Not contiguous where a copy does.
    wide = dict(ok, cache_lens=torch.stack([ok["cache_lens"]] * 2, dim=1)[:, 0], full_mask=torch.stack([ok["full_mask"]] * 2, dim=1)[:, 0])
    a, b = switch_gqa_decode_shared_forward(**wide), switch_gqa_decode_shared_forward(**ok)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
