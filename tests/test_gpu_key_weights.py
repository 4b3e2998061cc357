"""``switch_gqa_prefill_key_weights`` against a plain evaluation in 64 bits.

A weight is 2^(c q.k - LSE).  Its score is a sum of 128 exact products in fp32,
scaled once: off by at most 130 * 2^-24 * c * sum |q_i k_i|, and the subtraction
of the given LSE by 2^-24 of the larger operand, in log2 units; ln 2 of that
relative to the weight, and 2^-22 for the exponential.  A sum of n such positive
weights is off by at most n * 2^-24 more, relative; the kernel adds in parts of at
most 2^11 before it adds the parts, n <= 2^12 here: 2^-12 covers the additions
in the worst case and `rms` holds them to their usual size.
"""

import math

import pytest
import torch

from oracle import cache as C
from switchattentionkernels_amd import (build_switch_attention_metadata, build_switch_query_indices,
                                        shard_attention_metadata, switch_gqa_prefill_forward,
                                        switch_gqa_prefill_key_weights)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _qk(gen, b, sq, skv, hq, hkv):
    r = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16)  # noqa: E731
    return r(b, sq, hq, 128), r(b, skv, hkv, 128)


def _check(got, q, k, lse, start, end, scale=None):
    """got [B, Hkv, Skv] against the rows' bounds on flattened keys."""
    b, sq, hq, _ = q.shape
    skv, hkv = k.shape[1:3]
    want = C.key_weights(q.reshape(b * sq, hq, 128), k.reshape(b * skv, hkv, 128), lse.reshape(b * sq, hq),
                         start, end, scale).view(b, skv, hkv).transpose(1, 2)
    c = (128 ** -0.5 if scale is None else abs(scale)) * math.log2(math.e)
    dots = c * float((q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max()))   # >= sum |q_i k_i|
    live = lse[torch.isfinite(lse)]
    size = max(float(live.abs().max()) if live.numel() else 0.0, dots)
    eps = math.log(2) * (130 * 2.0 ** -24 * dots + 2.0 ** -24 * 2 * size) + 2.0 ** -22
    got = got.double().cpu()
    assert ((got - want).abs() <= (eps + 2.0 ** -12) * want).all()
    assert not got[want == 0].any()
    rms = ((got - want).norm() / want.norm().clamp(min=1e-300)).item()
    assert rms <= eps + 2.0 ** -19, rms


def _default_bounds(b, sq, skv, full, local, w):
    i = torch.arange(sq)
    start, end = torch.zeros(b * sq, dtype=torch.long), torch.zeros(b * sq, dtype=torch.long)
    for rows, lo in ((full, 0 * i), (local, (i - w + 1).clamp(min=0))):
        r = rows.long().cpu()
        base = r // sq * skv
        end[r] = base + (r % sq + 1).clamp(max=skv)
        start[r] = torch.minimum(base + lo[r % sq], end[r])
    return start, end


@pytest.mark.parametrize("b,s,hq,hkv,w,p", [
    (1, 1, 8, 2, 5, 1.0), (1, 1, 4, 1, 5, 0.0), (1, 257, 8, 2, 64, 0.25), (2, 300, 6, 2, 33, 0.5),
    (3, 128, 5, 5, 1, 0.3), (1, 1025, 16, 2, 256, 0.0), (1, 1024, 7, 1, 2000, 1.0),
    (2, 700, 40, 8, 100, 0.4), (1, 2047, 8, 4, 300, 0.1), (1, 640, 12, 1, 200, 0.5),
])
def test_against_the_formula(b, s, hq, hkv, w, p):
    gen = torch.Generator().manual_seed(s + hq)
    q, k = _qk(gen, b, s, s, hq, hkv)
    full, local = build_switch_query_indices((torch.rand(b, s, generator=gen) < p).to(DEV))
    _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, window_size=w)
    got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w)
    assert got.shape == (b, hkv, s) and got.dtype == torch.float32
    start, end = _default_bounds(b, s, s, full, local, w)
    _check(got, q, k, lse.cpu(), start, end)
    # Every query's weights sum to one.
    assert abs(got.double().sum().item() / (b * s * hq) - 1) < 1e-5
    again = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w)
    assert torch.equal(got, again)


@pytest.mark.parametrize("sq,skv", [(40, 500), (500, 40), (300, 1), (1, 777)])
def test_other_lengths_of_q_and_kv_and_scales(sq, skv):
    """Rows behind the keys (no legal key for late local rows), keys that no row sees."""
    gen = torch.Generator().manual_seed(sq)
    q, k = _qk(gen, 2, sq, skv, 8, 2)
    full, local = build_switch_query_indices((torch.rand(2, sq, generator=gen) < 0.4).to(DEV))
    for w, scale in ((30, None), (7, 0.02), (1000, 0.2)):
        _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, window_size=w,
                                            sm_scale=scale)
        got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w,
                                             sm_scale=scale)
        start, end = _default_bounds(2, sq, skv, full, local, w)
        _check(got, q, k, lse.cpu(), start, end, scale)


@pytest.mark.parametrize("b,sq,skv", [(2, 3000, 40), (3, 1000, 300), (5, 600, 257)])
def test_many_rows_behind_the_keys_of_a_batch(b, sq, skv):
    """Late local rows without a key lie between the sequences' rows that share a tile
    of keys; fresh workspaces hold NaN."""
    gen = torch.Generator().manual_seed(sq)
    q, k = _qk(gen, b, sq, skv, 8, 2)
    full, local = build_switch_query_indices((torch.rand(b, sq, generator=gen) < 0.1).to(DEV))
    for w in (7, 100, 2 ** 40):
        _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, window_size=min(w, sq))
        torch.cuda.synchronize()
        torch.full((2 ** 26,), math.nan, device=DEV)
        got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w)
        _check(got, q, k, lse.cpu(), *_default_bounds(b, sq, skv, full, local, w))


def test_packed_sequences_and_shards():
    gen = torch.Generator().manual_seed(5)
    lens = [1, 300, 0, 77, 512, 40]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    t = cu[-1]
    q, k = _qk(gen, 1, t, t, 10, 2)
    full, local = build_switch_query_indices((torch.rand(t, generator=gen) < 0.5).to(DEV))
    md = build_switch_attention_metadata(t, t, device=DEV, window_size=50, cu_seqlens=cu)
    _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, metadata=md, window_size=50)
    got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, metadata=md, window_size=50)
    start = torch.zeros(t, dtype=torch.long)
    start[full.long().cpu()] = md.full_starts.long().cpu()[full.long().cpu()]
    start[local.long().cpu()] = md.local_starts.long().cpu()[local.long().cpu()]
    _check(got, q, k, lse.cpu(), start, md.causal_ends.long().cpu())
    # A later chunk's queries against earlier keys: rows that see none among them.
    pos = torch.arange(400, 400 + t, dtype=torch.int32, device=DEV)
    md = shard_attention_metadata(pos, kv_start=0, kv_end=t, window_size=500)
    _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, metadata=md)
    got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, metadata=md)
    start[full.long().cpu()] = md.full_starts.long().cpu()[full.long().cpu()]
    start[local.long().cpu()] = md.local_starts.long().cpu()[local.long().cpu()]
    _check(got, q, k, lse.cpu(), start, md.causal_ends.long().cpu())


def test_non_finite_keys_and_queries_stay_where_they_are_seen():
    gen = torch.Generator().manual_seed(2)
    s, w = 600, 40
    q, k = _qk(gen, 1, s, s, 4, 2)
    full, local = build_switch_query_indices((torch.rand(s, generator=gen) < 0.2).to(DEV))
    _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, window_size=w)
    clean = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w)
    k2 = k.clone()
    k2[0, 333, 1] = math.nan
    got = switch_gqa_prefill_key_weights(q.to(DEV), k2.to(DEV), lse, full, local, window_size=w)
    nan = torch.isnan(got[0])
    assert nan[1, 333] and nan.sum() == 1
    got[0, 1, 333] = clean[0, 1, 333]
    assert torch.equal(got, clean)
    row = int(local[len(local) // 2])
    q2 = q.clone()
    q2[0, row, 0] = math.inf
    got = switch_gqa_prefill_key_weights(q2.to(DEV), k.to(DEV), lse, full, local, window_size=w)
    seen = torch.zeros(s, dtype=torch.bool)
    seen[max(row - w + 1, 0):row + 1] = True
    assert torch.equal(got[0, 1], clean[0, 1])
    assert torch.equal(got[0, 0][~seen.to(DEV)], clean[0, 0][~seen.to(DEV)])


def test_no_rows_no_keys():
    q, k = torch.zeros(2, 0, 4, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 9, 2, 128, dtype=torch.bfloat16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    lse = torch.zeros(2, 0, 4, device=DEV)
    got = switch_gqa_prefill_key_weights(q, k, lse, none, none)
    assert got.shape == (2, 2, 9) and not got.any()
    assert switch_gqa_prefill_key_weights(q, k[:, :0], lse, none, none).shape == (2, 2, 0)


def test_captured_calls_equal_eager_ones():
    gen = torch.Generator().manual_seed(3)
    s = 900
    q, k = (x.to(DEV) for x in _qk(gen, 1, s, s, 8, 2))
    full, local = build_switch_query_indices((torch.rand(s, generator=gen) < 0.3).to(DEV))

    def step():
        _, lse = switch_gqa_prefill_forward(q, k, k, full, local, window_size=100)
        return switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=100)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(torch.bfloat16))
        k.copy_(torch.randn(k.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_refusals_on_the_device():
    gen = torch.Generator().manual_seed(1)
    q, k = (x.to(DEV) for x in _qk(gen, 1, 20, 20, 4, 2))
    full, local = build_switch_query_indices(torch.ones(20, dtype=torch.bool, device=DEV))
    lse = torch.zeros(1, 20, 4, device=DEV)
    call = switch_gqa_prefill_key_weights
    for args, kw, words in (((q, k, lse[:, :19], full, local), {}, "lse"),
                            ((q, k, lse.double(), full, local), {}, "lse"),
                            ((q, k, lse, full, local), dict(window_size=0), "window_size"),
                            ((q, k, lse, full, local), dict(sm_scale=math.inf), "sm_scale"),
                            ((q, k, lse, full[:19], local), {}, "cover"),
                            ((q, k[:, :0], lse, full, local), {}, "at least one"),
                            ((q, k, lse, full.flip(0), local), {}, "increasing")):
        with pytest.raises(ValueError, match=words):
            call(*args, **kw)
    md = build_switch_attention_metadata(20, 20, device=DEV, window_size=5)
    md.causal_ends.copy_(md.causal_ends.flip(0))
    with pytest.raises(ValueError, match="non-decreasing"):
        call(q, k, lse, full, local, metadata=md)


def test_lists_of_any_origin_are_checked():
    """Lists that the compaction did not make: checked by the call, whatever their
    length, with the errors of the forward and no result."""
    gen = torch.Generator().manual_seed(7)
    for s in (30, 3000, 300000):
        hq = 1 if s > 10000 else 4
        q, k = torch.randn(1, s, hq, 128, generator=gen).to(torch.bfloat16).to(DEV), None
        k = q[:, :, :1].contiguous()
        full, local = build_switch_query_indices((torch.rand(s, generator=gen) < 0.3).to(DEV))
        _, lse = switch_gqa_prefill_forward(q, k, k, full, local, window_size=50)
        want = switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=50)
        for f, l in ((full.clone(), local.clone()), (full.long(), local.long()), (full[None], local[None])):
            assert torch.equal(switch_gqa_prefill_key_weights(q, k, lse, f, l, window_size=50), want)
        for change, words in (((full, -1, s), "outside"), ((full, 0, -1), "outside"), ((local, -1, s + 5), "outside"),
                              ((full, 1, full[0]), "increasing"), ((local, 2, local[1]), "increasing"),
                              ((full, 0, local[0]), "disjoint" if local[0] < full[1] else "increasing")):
            src, at, value = change
            bad = src.clone()
            bad[at] = value
            pair = (bad, local.clone()) if src is full else (full.clone(), bad)
            with pytest.raises(ValueError, match=words):
                switch_gqa_prefill_key_weights(q, k, lse, *pair, window_size=50)
        assert torch.equal(switch_gqa_prefill_key_weights(q, k, lse, full, local, window_size=50), want)


def test_unchecked_lists_cannot_be_captured():
    gen = torch.Generator().manual_seed(8)
    q, k = (x.to(DEV) for x in _qk(gen, 1, 64, 64, 4, 2))
    full, local = build_switch_query_indices((torch.rand(64, generator=gen) < 0.5).to(DEV))
    lse = torch.zeros(1, 64, 4, device=DEV)
    f, l = full.clone(), local.clone()
    switch_gqa_prefill_key_weights(q, k, lse, f, l)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            switch_gqa_prefill_key_weights(q, k, lse, f, l)
        held = switch_gqa_prefill_key_weights(q, k, lse, full, local)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, switch_gqa_prefill_key_weights(q, k, lse, full, local))


@pytest.mark.parametrize("seed", range(40))
def test_random_cases(seed):
    """Random batches, lengths of Q and of K, groups, windows and routes, in memory that
    held NaN before.  A sum has n <= 5 * 700 * 8 terms, but a lane adds one of a block of
    32, at most 128 blocks a part, and there are fewer than 900 blocks in 250 parts:
    (128 + 5 + 250) * 2^-24 stays below 2^-15."""
    gen = torch.Generator().manual_seed(500 + seed)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=gen))]  # noqa: E731
    size = lambda hi: int(2 ** (torch.rand(1, generator=gen).item() * math.log2(hi)))  # noqa: E731
    b, sq, skv, hkv, group = pick(1, 1, 2, 3, 5), size(700), size(700), pick(1, 2, 3), pick(1, 2, 4, 5, 8)
    skv = pick(skv, sq)
    w, p = size(2000), pick(0.0, 0.1, 0.25, 0.5, 0.9, 1.0)
    print(f"seed {seed}: B{b} Sq{sq} Skv{skv} Hq{hkv * group}/{hkv} W{w} p {p}", flush=True)
    q, k = _qk(gen, b, sq, skv, hkv * group, hkv)
    full, local = build_switch_query_indices((torch.rand(b, sq, generator=gen) < p).to(DEV))
    _, lse = switch_gqa_prefill_forward(q.to(DEV), k.to(DEV), k.to(DEV), full, local, window_size=w)
    torch.cuda.synchronize()
    torch.full((2 ** 25,), math.nan, device=DEV)
    got = switch_gqa_prefill_key_weights(q.to(DEV), k.to(DEV), lse, full, local, window_size=w)
    _check(got, q, k, lse.cpu(), *_default_bounds(b, sq, skv, full, local, w))
