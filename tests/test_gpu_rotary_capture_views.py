"""Captures of the differentiable rotation where an eager graph holds the leaf that an argument
is a view of: slices of a projection that is a leaf, a weight that is a strided view of one."""

import pytest
import torch

from switchattentionkernels_amd import switch_qk_rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _args(seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(2, 9, 8, 128, generator=gen, device=DEV).to(BF16)
    wide = 1 + 0.2 * torch.randn(128, 2, generator=gen, device=DEV)
    pos = torch.arange(9, dtype=torch.int32, device=DEV).expand(2, 9).contiguous()
    return qkv, wide, pos, 1e4 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)


@pytest.mark.parametrize("leaf", ["projection", "weights", "column"])
def test_refused_while_an_eager_graph_of_the_base_lives(leaf):
    qkv, wide, pos, freq = _args(1)
    (qkv if leaf == "projection" else wide).requires_grad_()

    def run():
        weights = {"q_weight": wide[:, 0], "k_weight": wide[:, 1]}
        if leaf == "projection":
            weights = {k: w.contiguous() for k, w in weights.items()}
        if leaf == "column":                     # one strided, one that is no view of a leaf
            weights["k_weight"] = wide.detach()[:, 1].contiguous()
        return switch_qk_rotary(qkv[:, :, :4], qkv[:, :, 4:6], pos, freq, **weights)

    kept = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = qkv.detach() + 1
        with pytest.raises(RuntimeError, match="eager graph"):
            run()
        with torch.no_grad():                    # without a graph of its own it stays allowed
            out = run()
    for _ in range(2):
        two.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(two, qkv.detach() + 1) and all(torch.equal(a, b) for a, b in zip(out, kept))


def test_captured_with_its_backward_when_none_lives():
    qkv, wide, pos, freq = _args(2)
    qkv.requires_grad_(), wide.requires_grad_()
    grads = [torch.ones(2, 9, h, 128, dtype=BF16, device=DEV) for h in (4, 2)]

    def step():
        outs = switch_qk_rotary(qkv[:, :, :4], qkv[:, :, 4:6], pos, freq, q_weight=wide[:, 0], k_weight=wide[:, 1])
        return [x.detach() for x in outs] + list(torch.autograd.grad(outs, (qkv, wide), grads))

    want = [x.clone() for x in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
