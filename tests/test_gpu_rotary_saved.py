"""What the rotation keeps for its gradients: rows only of a tensor that is normalised."""

import pytest
import torch

from switchattentionkernels_amd import switch_qk_rotary, switch_qk_rotary_backward

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
WEIGHTED = [(), ("q",), ("k",), ("q", "k")]


def _case(s=40, hq=8, hkv=2):
    gen = torch.Generator(device=DEV).manual_seed(s)
    rows = lambda h: torch.randn(2, s, h, 128, generator=gen, device=DEV).to(BF16)  # noqa: E731
    pos = torch.arange(s, dtype=torch.int32, device=DEV).expand(2, s).contiguous()
    freq = 1e4 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)
    weights = {x: 1 + 0.2 * torch.randn(128, generator=gen, device=DEV) for x in "qk"}
    return rows(hq), rows(hkv), pos, freq, weights, (rows(hq), rows(hkv))


@pytest.mark.parametrize("weighted", WEIGHTED)
def test_rows_without_a_norm_may_change_before_the_backward(weighted):
    q, k, pos, freq, w, grads = _case()
    how = {x + "_weight": w[x] for x in weighted}
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    want = switch_qk_rotary_backward(*grads, q, k, pos, freq, **how)
    for name, changed in (("q", 0), ("k", 1)):
        rows = [x * 1 for x in leaves]
        outs = switch_qk_rotary(*rows, pos, freq, **how)
        rows[changed].mul_(2.0)     # (its own gradient lets it: twice that of the leaf's is not asked for)
        if name in weighted:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(outs, leaves, grads)
        else:
            got = torch.autograd.grad(outs, leaves, grads)
            assert all(torch.equal(a, b) for a, b in zip(got, want[:2]))


@pytest.mark.parametrize("weighted", WEIGHTED)
def test_memory_between_forward_and_backward(weighted):
    """Slices of a projection of 96 MiB: alive behind the call only where a norm needs rows."""
    q, k, pos, freq, w, _ = _case(s=8192, hq=16, hkv=4)
    how = {x + "_weight": w[x] for x in weighted}
    leaf = torch.cat([q, k, k], dim=2).requires_grad_()
    del q, k
    before = torch.cuda.memory_allocated()
    qkv = leaf * 1
    outs = switch_qk_rotary(qkv[:, :, :16], qkv[:, :, 16:20], pos, freq, **how)
    kept = torch.cuda.memory_allocated() - before - sum(x.numel() * 2 for x in outs)
    del qkv
    kept_without = torch.cuda.memory_allocated() - before - sum(x.numel() * 2 for x in outs)
    assert kept >= 96 << 20
    assert (kept_without >= 96 << 20) if weighted else (kept_without < 1 << 20), kept_without
