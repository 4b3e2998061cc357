"""The plain evaluation's codes of the largest bf16 numbers, against an enumeration of all
codes."""

import numpy as np
import pytest
import torch

from oracle import cache as C

BF16_MAX = float(torch.finfo(torch.bfloat16).max)


def _known(dtype):
    if dtype == torch.int8:
        return np.arange(-127.0, 128.0)
    x = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    return np.unique(x[np.isfinite(x)])


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_the_nearest_code_that_stands_for_a_bf16_number(dtype):
    assert C.BF16_MAX == BF16_MAX
    known = _known(dtype)
    x = np.arange(128, 256) * 2.0 ** 120
    for amax in (x[-1], x[64], x[0], x[20]):
        scale = C.scale_for(amax, dtype)
        part = np.concatenate([x[x <= amax], -x[x <= amax]])
        got = C.keep_finite(C.round_code((part / scale).astype(np.float32), dtype), scale, dtype)
        allowed = known[np.abs(known) * scale <= BF16_MAX]
        off = np.abs(got - part / scale)
        assert np.isin(got, allowed).all()
        assert (off == np.abs(allowed[None] - (part / scale)[:, None]).min(1)).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_smaller_scales_change_nothing(dtype):
    known = _known(dtype)
    assert np.array_equal(C.keep_finite(known, 2.0 ** (119 if dtype != torch.int8 else 121), dtype), known)
    assert np.array_equal(C.keep_finite(known, float("nan"), dtype), known)
