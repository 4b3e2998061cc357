"""Norm and rotation of queries and keys on the GPU, forward, backward and with an
append, against 64 bits (``oracle/rotary.py``, where the bounds are derived)."""

import itertools
import math

import numpy as np
import pytest
import torch

from oracle import rotary as R
from switchattentionkernels_amd import (build_switch_query_indices, switch_gqa_prefill, switch_gqa_prefill_backward,
                                        switch_gqa_prefill_forward, switch_qk_rotary, switch_qk_rotary_append,
                                        switch_qk_rotary_backward, switch_qk_rotary_forward)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rows(gen, *shape, spread=1.0):
    x = torch.randn(*shape, generator=gen) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=gen))
    return x.to(BF16)


def _freq(n, base=1e4, dtype=F64):
    return (base ** (-torch.arange(n, dtype=F64) / n)).to(dtype)


def _case(seed, b, s, hq, hkv, n=64, sections=None, weights=F32, far=8191, dtype=F64, base=1e4):
    """CPU tensors: q, k, positions, inv_freq, sections, weights."""
    gen = torch.Generator().manual_seed(seed)
    sections = [n] if sections is None else sections
    pos = torch.randint(-far, far + 1, (len(sections), b, s), generator=gen, dtype=torch.int32)
    w = [None if weights is None else (1 + 0.3 * torch.randn(128, generator=gen)).to(weights) for _ in range(2)]
    return dict(q=_rows(gen, b, s, hq, 128), k=_rows(gen, b, s, hkv, 128), pos=pos, freq=_freq(n, base, dtype),
                sections=sections, qw=w[0], kw=w[1], gen=gen)


def _up(t):
    return None if t is None else t.to(DEV)


def _how(c, interleaved, eps):
    return dict(sections=c["sections"], interleaved=interleaved, q_weight=_up(c["qw"]), k_weight=_up(c["kw"]), eps=eps)


def _unit(c):
    return R.unit(c["pos"].numpy(), c["freq"].numpy(), c["sections"])


def _check_rows(c, name, got, interleaved, eps):
    w = c[name + "w"]
    want, off = R.forward(R.np64(c[name]), None if w is None else R.np64(w), eps, *_unit(c), interleaved)
    assert got.dtype == BF16 and got.is_contiguous() and got.shape == c[name].shape
    assert R.near(R.np64(got), want, off, R.BF16_HALF_STEP), name


SHAPES = [(1, 1, 1, 1), (2, 3, 8, 2), (1, 7, 4, 1), (3, 5, 40, 8), (1, 33, 9, 7), (2, 2, 64, 8), (1, 300, 16, 3)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_shapes(shape, interleaved):
    c = _case(1, *shape)
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, interleaved, 1e-6))
    for name, x in zip("qk", got):
        _check_rows(c, name, x, interleaved, 1e-6)


@pytest.mark.parametrize("n,sections", [(8, None), (16, [5, 11]), (24, [8, 8, 8]), (32, None), (40, [1, 38, 1]),
                                        (48, [12, 12, 12, 12]), (56, [50, 6]), (64, [16, 24, 24]), (64, [61, 1, 1, 1])])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [None, F32, BF16])
def test_forward_frequencies_axes_weights(n, sections, interleaved, weights):
    c = _case(n, 2, 9, 10, 3, n=n, sections=sections, weights=weights, dtype=F32 if n % 16 else F64)
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, interleaved, 1e-5))
    for name, x in zip("qk", got):
        _check_rows(c, name, x, interleaved, 1e-5)
        if 2 * n < 128 and weights is None:      # dims behind the rotated ones: untouched
            assert torch.equal(x[..., 2 * n:].cpu(), c[name][..., 2 * n:])


@pytest.mark.parametrize("dtype", [F32, F64])
def test_far_positions(dtype):
    """The ends of int32 and powers of two on the way, with frequencies of 1 and above."""
    edge = sorted({s * (2 ** e + d) for e in range(31) for d in (-1, 0, 1) for s in (-1, 1)} | {2 ** 31 - 1, -2 ** 31})
    edge = [p for p in edge if -2 ** 31 <= p < 2 ** 31]
    c = _case(5, 1, len(edge), 2, 1, weights=None, dtype=dtype, base=5e5)
    c["freq"] = (c["freq"].double() * 3.7).to(dtype)
    c["pos"] = torch.tensor(edge, dtype=torch.int32).view(1, 1, -1)
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]))
    # 2^31 times 3.7 in 80-bit floats: off by 2^-31 radians, beside the bound's 24 U.
    for name, x in zip("qk", got):
        _check_rows(c, name, x, False, 1e-6)


@pytest.mark.parametrize("tokens,heads", [(5119, (1, 1)), (5120, (9, 1)), (5121, (1, 9)), (6000, (3, 2)), (10241, (17, 1))])
def test_tokens_shared_out_over_the_waves(tokens, heads):
    """Whole rounds of tokens, and what is left of them, to every token's last row; calls large
    enough to go past the memory-side cache are tested by the sizes below."""
    c = _case(12, 1, tokens, *heads, n=8)
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    for name, x in zip("qk", got):
        _check_rows(c, name, x, False, 1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,weights", [(6001, F32), (6001, None), (17001, F32)])
def test_large_calls_as_small_ones(tokens, weights, interleaved):
    """Calls of 100 MB and more, streamed, against the same rows in small calls."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    q, k, gq, gk = (torch.randn(1, tokens, h, 128, generator=gen, device=DEV).to(BF16) for h in (32, 8, 32, 8))
    c = _case(13, 1, tokens, 1, 1, weights=weights)
    how, pos, freq = _how(c, interleaved, 1e-6), _up(c["pos"]), _up(c["freq"])
    got = switch_qk_rotary_forward(q, k, pos, freq, **how)
    grads = switch_qk_rotary_backward(gq, gk, q, k, pos, freq, **how)
    kc, vc = (torch.zeros(1, tokens, 8, 128, dtype=BF16, device=DEV) for _ in range(2))
    switch_qk_rotary_append(q, k, k, kc, vc, _int32([0]), pos, freq, **how)
    assert torch.equal(kc, got[1]) and torch.equal(vc, k)
    for i in range(0, tokens, 2500):
        s = slice(i, i + 2500)
        part = switch_qk_rotary_forward(q[:, s], k[:, s], pos[..., s].contiguous(), freq, **how)
        dx = switch_qk_rotary_backward(gq[:, s], gk[:, s], q[:, s], k[:, s], pos[..., s].contiguous(), freq, **how)
        assert all(torch.equal(a[:, s], b) for a, b in zip(got + grads[:2], part + dx[:2]))


def test_one_weight_only():
    c = _case(6, 2, 5, 4, 2)
    for drop in ("qw", "kw"):
        d = dict(c, **{drop: None})
        got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(d, False, 1e-6))
        for name, x in zip("qk", got):
            _check_rows(d, name, x, False, 1e-6)


def test_strided_rows_are_taken_as_they_are():
    """Slices of a projection, heads before tokens, an expanded batch, a single head's row."""
    c = _case(7, 2, 6, 8, 2)
    want = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    qkv = torch.full((2, 6, 14, 128), math.nan, dtype=BF16, device=DEV)
    qkv[:, :, 2:10], qkv[:, :, 10:12] = _up(c["q"]), _up(c["k"])
    turned = [_up(c[x]).transpose(1, 2).contiguous().transpose(1, 2) for x in "qk"]
    assert not turned[0].is_contiguous()
    for q, k in ((qkv[:, :, 2:10], qkv[:, :, 10:12]), turned):
        got = switch_qk_rotary_forward(q, k, _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
        assert all(torch.equal(a, b) and a.is_contiguous() for a, b in zip(got, want))
    one = dict(c, q=c["q"][:1], k=c["k"][:1])
    wide = switch_qk_rotary_forward(_up(one["q"]).expand(2, -1, -1, -1), _up(one["k"]).expand(2, -1, -1, -1),
                                    _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    full = dict(c, q=c["q"][:1].expand(2, -1, -1, -1).contiguous(), k=c["k"][:1].expand(2, -1, -1, -1).contiguous())
    for name, x in zip("qk", wide):
        _check_rows(full, name, x, False, 1e-6)


def test_values_that_are_not_finite_stay_in_their_row():
    c = _case(8, 1, 4, 3, 1, n=16)
    c["q"][0, 1, 1, 5], c["q"][0, 2, 0, 100], c["k"][0, 3, 0, 40] = math.inf, math.nan, -math.inf
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    bad = torch.isnan(got[0]).any(dim=-1)[0].cpu()
    assert bad[1, 1] and bad[2, 0] and int(bad.sum()) == 2
    c["qw"] = c["kw"] = None                     # without a norm: only the pairs that hold them
    got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    odd = ~torch.isfinite(got[0][0].cpu())
    assert odd[1, 1].nonzero().flatten().tolist() == [5, 21] and odd[2, 0].nonzero().flatten().tolist() == [100]
    assert int(odd.sum()) == 3
    assert torch.equal(got[1][0, 3, 0, 40].cpu(), torch.tensor(-math.inf, dtype=BF16))


def test_frequencies_that_are_not_numbers_show():
    c = _case(9, 1, 3, 2, 1, n=16, weights=None)
    for bad in (math.nan, math.inf, 2.0 ** 41):
        f = c["freq"].clone()
        f[3] = bad
        got = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(f))[0]
        assert torch.isnan(got).any(dim=0).any(dim=0).any(dim=0).nonzero().flatten().tolist() == [3, 19]


def test_rows_of_zeros():
    c = _case(10, 1, 2, 2, 1)
    c["q"].zero_()
    q, _ = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 1e-6))
    assert not q.any()
    q, _ = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]), **_how(c, False, 0.0))
    assert torch.isnan(q).all()                  # 0 / 0, as the formula has it


def test_no_tokens():
    c = _case(11, 2, 0, 4, 2)
    q, k = (_up(c[x]).requires_grad_() for x in "qk")
    w = [_up(c[x]).requires_grad_() for x in ("qw", "kw")]
    oq, ok = switch_qk_rotary(q, k, _up(c["pos"]), _up(c["freq"]), q_weight=w[0], k_weight=w[1])
    assert oq.shape == q.shape and ok.shape == k.shape
    g = torch.autograd.grad((oq, ok), (q, k, *w), (torch.empty_like(oq), torch.empty_like(ok)))
    assert g[0].shape == q.shape and not g[2].any() and not g[3].any()
    kc, vc = (torch.ones(2, 3, 2, 128, dtype=BF16, device=DEV) for _ in range(2))
    out, lens = switch_qk_rotary_append(q.detach(), k.detach(), k.detach(), kc, vc, _int32([1, 5]), _up(c["pos"]),
                                        _up(c["freq"]))
    assert lens.tolist() == [1, 3] and out.shape == q.shape and bool((kc == 1).all() and (vc == 1).all())


# ---------------------------------------------------------------------------
# Gradients
# ---------------------------------------------------------------------------
def _check_backward(c, interleaved, eps, got, grads):
    for i, name in enumerate("qk"):
        w = c[name + "w"]
        dx, off, dw, dw_off = R.backward(R.np64(grads[i]), R.np64(c[name]), None if w is None else R.np64(w), eps,
                                         *_unit(c), interleaved)
        assert got[i].dtype == BF16 and got[i].is_contiguous()
        assert R.near(R.np64(got[i]), dx, off, R.BF16_HALF_STEP), "d" + name
        if w is None:
            assert got[2 + i] is None
        else:
            assert got[2 + i].dtype == w.dtype
            assert R.near(R.np64(got[2 + i]), dw, dw_off, R.BF16_HALF_STEP if w.dtype == BF16 else R.U), "dw " + name


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [None, F32, BF16])
def test_backward_shapes(shape, interleaved, weights):
    c = _case(20, *shape, n=48, sections=[16, 16, 16], weights=weights)
    grads = [_rows(c["gen"], *c[x].shape) for x in "qk"]
    got = switch_qk_rotary_backward(*(_up(g) for g in grads), _up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]),
                                    **_how(c, interleaved, 1e-6))
    _check_backward(c, interleaved, 1e-6, got, grads)


def test_backward_many_rows_is_reproducible():
    c = _case(21, 2, 4099, 16, 2, base=1e6)
    grads = [_rows(c["gen"], *c[x].shape) for x in "qk"]
    args = [_up(g) for g in grads] + [_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"])]
    got = switch_qk_rotary_backward(*args, **_how(c, False, 1e-6))
    _check_backward(c, False, 1e-6, got, grads)
    again = switch_qk_rotary_backward(*args, **_how(c, False, 1e-6))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradients_against_differences():
    """Central differences of the 64-bit formula along random directions."""
    c = _case(22, 1, 3, 2, 2, n=32, sections=[20, 12])
    grads = [_rows(c["gen"], *c[x].shape) for x in "qk"]
    got = switch_qk_rotary_backward(*(_up(g) for g in grads), _up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]),
                                    **_how(c, True, 1e-6))
    for i, name in enumerate("qk"):
        x, w, dy = R.np64(c[name]), R.np64(c[name + "w"]), R.np64(grads[i])
        loss = lambda x, w: (R.forward(x, w, 1e-6, *_unit(c), True)[0] * dy).sum()  # noqa: E731
        rng, h = np.random.default_rng(i), 2.0 ** -17
        for _ in range(5):
            d = rng.standard_normal(x.shape) * np.abs(x)
            slope = (loss(x + h * d, w) - loss(x - h * d, w)) / (2 * h)
            # One rounding of each of dx's values; differences: h^2 of the third derivative.
            room = 2 ** -8 * np.abs(R.np64(got[i]) * d).sum() + 1e-4 * np.abs(slope) + 1e-6
            assert abs((R.np64(got[i]) * d).sum() - slope) <= room
            e = rng.standard_normal(128)
            slope = (loss(x, w + h * e) - loss(x, w - h * e)) / (2 * h)
            assert abs((R.np64(got[2 + i]) * e).sum() - slope) <= 1e-5 * np.abs(R.np64(got[2 + i]) * e).sum() + 1e-6


def test_autograd():
    """Leaves in a fused projection, expanded keys, weights; one of them without need."""
    c = _case(23, 2, 5, 4, 2)
    qkv = torch.cat([c["q"], c["k"], c["k"]], dim=2).to(DEV).requires_grad_()
    w = [_up(c["qw"]).requires_grad_(), _up(c["kw"])]
    how = dict(_how(c, False, 1e-6), q_weight=w[0], k_weight=w[1])
    q, k = switch_qk_rotary(qkv[:, :, :4], qkv[:, :, 4:6], _up(c["pos"]), _up(c["freq"]), **how)
    grads = [_rows(c["gen"], *x.shape) for x in (q, k)]
    torch.autograd.backward((q, k), [_up(g) for g in grads])
    _check_backward(c, False, 1e-6, (qkv.grad[:, :, :4].contiguous(), qkv.grad[:, :, 4:6].contiguous(), w[0].grad,
                                     switch_qk_rotary_backward(*(_up(g) for g in grads), _up(c["q"]), _up(c["k"]),
                                                               _up(c["pos"]), _up(c["freq"]), **how)[3]), grads)
    assert not qkv.grad[:, :, 6:].any() and w[1].grad is None
    # Only one output used: the other's gradient is zero.
    x = _up(c["q"]).requires_grad_()
    q, k = switch_qk_rotary(x, _up(c["k"]), _up(c["pos"]), _up(c["freq"]))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(q.float().square().sum(), x, create_graph=True)[0].sum().backward()


def test_gradients_that_start_anywhere():
    """Gradients that come as views: not contiguous, and not at a multiple of 16 bytes."""
    c = _case(25, 2, 5, 4, 2)
    leaves = [_up(c[x]).requires_grad_() for x in ("q", "k", "qw", "kw")]
    outs = switch_qk_rotary(leaves[0], leaves[1], _up(c["pos"]), _up(c["freq"]), sections=c["sections"],
                            q_weight=leaves[2], k_weight=leaves[3])
    grads = [_rows(c["gen"], *x.shape) for x in outs]
    odd = torch.empty(grads[0].numel() + 1, dtype=BF16, device=DEV)[1:].view(grads[0].shape)
    odd.copy_(grads[0])
    turned = _up(grads[1]).transpose(1, 2).contiguous().transpose(1, 2)
    got = torch.autograd.grad(outs, leaves, (odd, turned))
    _check_backward(c, False, 1e-6, got, grads)


def test_one_gradient_only():
    """What is not asked for is not given; an output that nothing uses has a gradient of 0."""
    c = _case(26, 2, 5, 4, 2)
    names = ("q", "k", "qw", "kw")
    for want in names:
        leaf = {x: _up(c[x]).requires_grad_(x == want) for x in names}
        q, k = switch_qk_rotary(leaf["q"], leaf["k"], _up(c["pos"]), _up(c["freq"]), q_weight=leaf["qw"],
                                k_weight=leaf["kw"])
        out, other = (q, k) if want[0] == "q" else (k, q)
        out.backward(torch.ones_like(out))
        ones = [torch.ones_like(x) if x is out else torch.zeros_like(x) for x in (q, k)]
        full = switch_qk_rotary_backward(*ones, leaf["q"], leaf["k"], _up(c["pos"]), _up(c["freq"]),
                                         q_weight=leaf["qw"], k_weight=leaf["kw"])
        assert torch.equal(leaf[want].grad, full[names.index(want)])
        assert all(leaf[x].grad is None for x in names if x != want)


def test_training_step_captured_and_replayed():
    c = _case(27, 1, 40, 8, 2)
    leaves = [_up(c[x]).requires_grad_() for x in ("q", "k", "qw", "kw")]
    pos, freq = _up(c["pos"]), _up(c["freq"])
    grads = [_up(_rows(c["gen"], *c[x].shape)) for x in "qk"]

    def step():
        outs = switch_qk_rotary(leaves[0], leaves[1], pos, freq, q_weight=leaves[2], k_weight=leaves[3])
        return outs + torch.autograd.grad(outs, leaves, grads)

    def eager():
        return [x.detach().clone() for x in step()]

    eager()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [x.detach() for x in step()]
    for i in range(4):
        with torch.no_grad():
            for x in leaves + grads:
                x.copy_(x * (1.0 + 0.25 * i))
        pos.add_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, eager())), i


def test_two_layers_of_the_same_weights_captured():
    """The second call meets what the first one's leaves hold on the capturing stream: allowed."""
    c = _case(32, 2, 21, 4, 2)
    leaves = [_up(c[x]).requires_grad_() for x in ("q", "k", "qw", "kw")]
    pos, freq = _up(c["pos"]), _up(c["freq"])
    grads = [_up(_rows(c["gen"], *c[x].shape)) for x in "qk"]

    def step():
        how = dict(q_weight=leaves[2], k_weight=leaves[3])
        q, k = switch_qk_rotary(leaves[0], leaves[1], pos, freq, **how)
        return torch.autograd.grad(switch_qk_rotary(q, k, pos, freq, **how), leaves, grads)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_capture_is_refused_while_an_eager_graph_of_the_leaves_lives():
    c = _case(28, 1, 9, 4, 2)
    q, w = _up(c["q"]).requires_grad_(), _up(c["qw"]).requires_grad_()
    k, pos, freq = _up(c["k"]), _up(c["pos"]), _up(c["freq"])
    run = lambda: switch_qk_rotary(q, k, pos, freq, q_weight=w)  # noqa: E731
    kept = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = k + 1
        with pytest.raises(RuntimeError, match="eager graph"):
            run()
        with torch.no_grad():                    # without a graph of its own it stays allowed
            out = run()
    two.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(two, k + 1) and all(torch.equal(a, b) for a, b in zip(out, kept))


def test_arguments_that_are_copied_keep_their_gradients():
    """Weights that are strided views, positions of one axis without its dimension."""
    c = _case(29, 2, 5, 4, 2)
    wide = torch.stack([c["qw"], c["kw"]], dim=-1).to(DEV).requires_grad_()
    q, k = (_up(c[x]).requires_grad_() for x in "qk")
    pos = torch.stack([c["pos"][0]] * 2, dim=-1).to(DEV)[..., 0]
    outs = switch_qk_rotary(q, k, pos, _up(c["freq"]), q_weight=wide[:, 0], k_weight=wide[:, 1])
    grads = [_rows(c["gen"], *x.shape) for x in outs]
    got = torch.autograd.grad(outs, (q, k, wide), [_up(g) for g in grads])
    _check_backward(c, False, 1e-6, (*got[:2], got[2][:, 0], got[2][:, 1]), grads)


def test_training_step_with_the_prefill():
    """Projection slices, norm and rotation, routed attention, and back: as the calls by themselves."""
    b, s, hq, hkv = 1, 300, 8, 2
    c = _case(31, b, s, hq, hkv)
    qkv = torch.cat([c["q"], c["k"], _rows(c["gen"], b, s, hkv, 128)], dim=2).to(DEV).requires_grad_()
    w = [_up(c[x]).requires_grad_() for x in ("qw", "kw")]
    pos, freq = torch.arange(s, dtype=torch.int32, device=DEV)[None], _up(c["freq"])
    how = dict(q_weight=w[0], k_weight=w[1])
    q, k, v = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:].contiguous()
    lists = build_switch_query_indices(torch.rand(s, generator=c["gen"]).to(DEV) < 0.4)
    qr, kr = switch_qk_rotary(q, k, pos, freq, **how)
    out, lse = switch_gqa_prefill(qr, kr, v, *lists, window_size=64)
    dout = _up(_rows(c["gen"], *out.shape))
    out.backward(dout)
    with torch.no_grad():
        q1, k1 = switch_qk_rotary_forward(q, k, pos, freq, **how)
        o1, lse1 = switch_gqa_prefill_forward(q1, k1, v, *lists, window_size=64)
        dq, dk, dv = switch_gqa_prefill_backward(q1, k1, v, o1, lse1, dout, *lists, window_size=64)
        want = switch_qk_rotary_backward(dq, dk, q, k, pos, freq, **how)
    assert torch.equal(out, o1) and torch.equal(lse, lse1)
    assert torch.equal(qkv.grad, torch.cat([want[0], want[1], dv], dim=2))
    assert torch.equal(w[0].grad, want[2]) and torch.equal(w[1].grad, want[3])


def test_changed_inputs_are_noticed_by_autograd():
    c = _case(24, 1, 4, 2, 1)
    x, pos = _up(c["q"]).requires_grad_(), _up(c["pos"])
    q, _ = switch_qk_rotary(x, _up(c["k"]), pos, _up(c["freq"]))
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        q.float().sum().backward()


# ---------------------------------------------------------------------------
# Appends
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t", [1, 2, 19])
@pytest.mark.parametrize("heads", [(8, 2), (40, 8), (3, 3)])
@pytest.mark.parametrize("counts", [False, True])
def test_append(t, heads, counts):
    b, cap = 6, 23
    c = _case(30 + t, b, t, *heads)
    v = _rows(c["gen"], b, t, heads[1], 128)
    lens = [0, 5, cap - t, cap - 1, cap, 40 - 57 * (t % 2)]     # full, and outside [0, L]
    n = [t, t - 1, t, t, 1, t] if counts else [t] * b
    if counts:
        n[3], n[5] = t + 3, -2 if t == 2 else t
    kc, vc = (_rows(c["gen"], b, cap, heads[1], 128).to(DEV) for _ in range(2))
    was = kc.clone(), vc.clone()
    lens_t = _int32(lens)
    q, after = switch_qk_rotary_append(_up(c["q"]), _up(c["k"]), _up(v), kc, vc, lens_t, _up(c["pos"]), _up(c["freq"]),
                                       row_counts=_int32(n) if counts else None, **_how(c, False, 1e-6))
    want_q, want_k = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]),
                                              **_how(c, False, 1e-6))
    assert torch.equal(q, want_q) and lens_t.tolist() == lens
    for i in range(b):
        old = min(max(lens[i], 0), cap)
        new = min(max(n[i], 0), t)
        assert int(after[i]) == min(old + new, cap)
        new = min(new, cap - old)
        for cache, before, rows in ((kc, was[0], want_k), (vc, was[1], _up(v))):
            want = before[i].clone()
            want[old:old + new] = rows[i, :new]
            assert torch.equal(cache[i].view(torch.int16), want.view(torch.int16))


def test_append_strided_and_far_rows():
    """K and V as slices of a projection; rows whose byte offset passes 2^32."""
    b, cap, t = 2, 1 << 23, 3
    c = _case(40, b, t, 4, 1)
    qkv = torch.cat([c["q"], c["k"], c["k"] * 2], dim=2).to(DEV)
    kc, vc = (torch.zeros(b, cap, 1, 128, dtype=BF16, device=DEV) for _ in range(2))
    _, after = switch_qk_rotary_append(qkv[:, :, :4], qkv[:, :, 4:5], qkv[:, :, 5:], kc, vc, _int32([7, cap - 4]),
                                       _up(c["pos"]), _up(c["freq"]))
    assert after.tolist() == [10, cap - 1]
    _, k = switch_qk_rotary_forward(_up(c["q"]), _up(c["k"]), _up(c["pos"]), _up(c["freq"]))
    for i, at in enumerate((7, cap - 4)):
        assert torch.equal(kc[i, at:at + 3], k[i]) and torch.equal(vc[i, at:at + 3], (c["k"][i] * 2).to(DEV))
    assert int((kc != 0).any(dim=-1).sum()) == 6


def test_captured_and_replayed():
    """Forward, backward and append in a graph, replayed with new inputs beside eager work."""
    c = _case(50, 4, 1, 8, 2)
    q, k, pos, lens = _up(c["q"]), _up(c["k"]), _up(c["pos"]), _int32([0, 3, 6, 9])
    kc, vc = (torch.zeros(4, 16, 2, 128, dtype=BF16, device=DEV) for _ in range(2))
    how = _how(c, False, 1e-6)
    freq = _up(c["freq"])
    run = lambda: (switch_qk_rotary_append(q, k, k, kc, vc, lens, pos, freq, **how),  # noqa: E731
                   switch_qk_rotary_backward(q, k, q, k, pos, freq, **how))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (out, after), grads = run()
    for i in range(4):
        q.copy_(_rows(c["gen"], *q.shape)), k.copy_(_rows(c["gen"], *k.shape))
        pos.add_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone(), after.clone(), kc.clone(), *(g.clone() for g in grads)]
        (want, want_after), want_grads = run()
        for a, b in zip(got, [want, want_after, kc, *want_grads]):
            assert torch.equal(a, b), i


def test_other_stream():
    c = _case(51, 2, 2000, 8, 2)
    args = [_up(c[x]) for x in ("q", "k", "pos", "freq")]
    how = _how(c, False, 1e-6)
    want = switch_qk_rotary_forward(*args, **how)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = args[0] * 1
        got = switch_qk_rotary_forward(q, *args[1:], **how)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_refusals():
    c = _case(60, 2, 3, 4, 2)
    ok = dict(q=_up(c["q"]), k=_up(c["k"]), positions=_up(c["pos"]), inv_freq=_up(c["freq"]), sections=[64],
              q_weight=_up(c["qw"]), k_weight=_up(c["kw"]), eps=1e-6)
    switch_qk_rotary_forward(**ok)
    switch_qk_rotary_forward(**dict(ok, positions=ok["positions"][0], sections=None))
    wide = torch.zeros(2, 3, 4, 132, dtype=BF16, device=DEV)
    bad = [
        (TypeError, "BF16", dict(q=ok["q"].float())),
        (TypeError, "BF16", dict(k=None)),
        (ValueError, "accelerator", dict(q=c["q"])),
        (ValueError, "accelerator", dict(k=c["k"])),
        (ValueError, "must be \\[B,S,H,128\\]", dict(q=ok["q"][0])),
        (ValueError, "must be \\[B,S,H,128\\]", dict(q=ok["q"][..., :64])),
        (ValueError, "must be \\[B,S,H,128\\]", dict(k=ok["k"][:, :, :0])),
        (ValueError, "contiguous and start", dict(q=wide[..., 4:])),
        (ValueError, "contiguous and start", dict(q=wide[..., :128])),
        (ValueError, "contiguous and start", dict(q=ok["q"].transpose(2, 3).contiguous().transpose(2, 3))),
        (ValueError, "same batch", dict(k=ok["k"][:1])),
        (ValueError, "same batch", dict(k=ok["k"][:, :2])),
        (TypeError, "inv_freq", dict(inv_freq=ok["inv_freq"].bfloat16())),
        (ValueError, "inv_freq", dict(inv_freq=ok["inv_freq"][:60], sections=[60])),
        (ValueError, "inv_freq", dict(inv_freq=c["freq"])),
        (ValueError, "inv_freq", dict(inv_freq=torch.ones(72, device=DEV), sections=[72])),
        (ValueError, "inv_freq", dict(inv_freq=ok["inv_freq"][:0], sections=None)),
        (ValueError, "sections", dict(sections=[63])),
        (ValueError, "sections", dict(sections=[64, 0])),
        (ValueError, "sections", dict(sections=[])),
        (ValueError, "sections", dict(sections=[60, 1, 1, 1, 1])),
        (ValueError, "positions must be", dict(sections=[32, 32])),
        (TypeError, "int32", dict(positions=ok["positions"].long())),
        (TypeError, "int32", dict(positions=None)),
        (ValueError, "positions must be", dict(positions=ok["positions"][:, :, :2])),
        (ValueError, "positions must be", dict(positions=c["pos"])),
        (TypeError, "q_weight", dict(q_weight=ok["q_weight"].double())),
        (ValueError, "k_weight", dict(k_weight=ok["k_weight"][:64])),
        (ValueError, "k_weight", dict(k_weight=c["kw"])),
        (TypeError, "same type", dict(k_weight=ok["k_weight"].bfloat16())),
        (ValueError, "eps", dict(eps=-1e-6)),
        (ValueError, "eps", dict(eps=math.nan)),
    ]
    for kind, words, change in bad:
        with pytest.raises(kind, match=words):
            switch_qk_rotary_forward(**dict(ok, **change))
    # Not contiguous where a copy does: as the contiguous ones.
    every = torch.stack([ok["positions"], ok["positions"] + 1], dim=-1)[..., 0]
    freq = torch.stack([ok["inv_freq"], ok["inv_freq"]], dim=-1)[..., 0]
    weight = torch.stack([ok["q_weight"], ok["q_weight"]], dim=-1)[..., 0]
    assert not (every.is_contiguous() or freq.is_contiguous() or weight.is_contiguous())
    got = switch_qk_rotary_forward(**dict(ok, positions=every, inv_freq=freq, q_weight=weight))
    assert all(torch.equal(a, b) for a, b in zip(got, switch_qk_rotary_forward(**ok)))
    g = torch.zeros_like(ok["q"]), torch.zeros_like(ok["k"])
    for i, wrong in itertools.product((0, 1), (g[0].float(), g[0][:1], g[0].cpu(), None)):
        with pytest.raises(ValueError, match="grad_"):
            switch_qk_rotary_backward(*[wrong if j == i else g[j] for j in (0, 1)], **ok)


def test_append_refusals():
    c = _case(61, 2, 3, 4, 2)
    kc, vc = (torch.zeros(2, 9, 2, 128, dtype=BF16, device=DEV) for _ in range(2))
    ok = dict(q=_up(c["q"]), k=_up(c["k"]), v=_up(c["k"]), k_cache=kc, v_cache=vc, cache_lens=_int32([0, 1]),
              positions=_up(c["pos"]), inv_freq=_up(c["freq"]))
    bad = [
        (ValueError, "identical", dict(v=ok["v"][:, :2])),
        (TypeError, "BF16", dict(v=ok["v"].float())),
        (TypeError, "BF16", dict(v=None)),
        (TypeError, "caches must be BF16", dict(k_cache=kc.float())),
        (TypeError, "caches must be BF16", dict(k_cache=None)),
        (ValueError, "device", dict(v_cache=vc.cpu())),
        (ValueError, "contiguous", dict(k_cache=torch.zeros(2, 2, 9, 128, dtype=BF16, device=DEV).transpose(1, 2))),
        (ValueError, "one shape", dict(k_cache=kc[:, :8].contiguous())),
        (ValueError, "one shape", dict(k_cache=kc[:1], v_cache=vc[:1])),
        (ValueError, "one shape", dict(k_cache=kc[:, :0], v_cache=vc[:, :0])),
        (ValueError, "cache_lens", dict(cache_lens=ok["cache_lens"].long())),
        (ValueError, "cache_lens", dict(cache_lens=ok["cache_lens"][:1])),
        (ValueError, "row_counts", dict(row_counts=ok["cache_lens"].cpu())),
        (ValueError, "share memory", dict(v_cache=kc)),
        (ValueError, "share memory", dict(k=kc[:, :3], v=vc[:, :3])),
    ]
    for kind, words, change in bad:
        with pytest.raises(kind, match=words):
            switch_qk_rotary_append(**dict(ok, **change))
    assert not kc.any() and not vc.any()
