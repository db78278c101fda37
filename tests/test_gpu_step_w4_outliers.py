"""Products with 4-bit weights of inputs next to far larger ones whose weights
are 0: what the others keep of their bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu

D = 1024


def outliers(group, n=120, seed=1):
    """Weights whose column 37 of every 128 has the zero's code."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 16, (n, D), dtype=torch.uint8, generator=g)
    z = torch.randint(0, 16, (n, D // group), dtype=torch.uint8, generator=g)
    c[:, 37::128] = z.repeat_interleave(group, 1)[:, 37::128]
    return c[:, 0::2] | c[:, 1::2] << 4, (torch.randn((n, D // group), generator=g) * 0.01).half(), z


@pytest.mark.parametrize("bits", [12, 20, 24, 28])
@pytest.mark.parametrize("batch", [1, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 128])
def test_inputs_next_to_an_outlier(hip, group, batch, bits):
    """The root mean square of the errors, each over the root of its products'
    squares. An input is off by 2^-23 of itself, and by 2^-51 of the largest of its
    128 columns, at most: 2^-23 of an input of 1 next to one of 2^28. With 8 steps'
    sums of 4 products of 32 and their scales, each rounded to 2^-24 of a partial
    sum that is about that root, and random (7 2^-24), 2^-20 in all is twice that."""
    w = outliers(group)
    dense = ref.w4_dense(*w)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((batch, D), generator=g)
    x[:, 37::128] *= 2.0 ** bits
    out = torch.empty((batch, dense.shape[0]), device="cuda")
    hip.w4_matmul_rows(out, hip.W4Weights(*(t.cuda() for t in w)), x.cuda())
    v = ref.f64(x)
    error = (ref.f64(out) - v @ dense.T) / torch.sqrt((v * v) @ (dense * dense).T)
    rms = float(error.square().mean().sqrt())
    assert rms < 2.0 ** -20, np.log2(rms)


@pytest.mark.parametrize("batch,bits", [(1, 30), (16, 30), (17, 60), (40, 60)])
def test_bf16_inputs_next_to_an_outlier(hip, batch, bits):
    """Up to 16 inputs are off by 2^-39 of the largest at most, 2^-9 next to one of
    2^30, and 2^-10 on average; more inputs are exact. A result is rounded to 2^-8 of
    itself at most, 2^-9 on average."""
    w = outliers(64)
    dense = ref.w4_dense(*w)
    x = torch.randn((batch, D), generator=torch.Generator().manual_seed(3))
    x[:, 37::128] *= 2.0 ** bits
    x = x.bfloat16()
    out = torch.empty((batch, dense.shape[0]), dtype=torch.bfloat16, device="cuda")
    hip.w4_matmul_rows(out, hip.W4Weights(*(t.cuda() for t in w)), x.cuda())
    v = ref.f64(x)
    error = (ref.f64(out) - v @ dense.T) / torch.sqrt((v * v) @ (dense * dense).T)
    assert float(error.square().mean().sqrt()) < 2.0 ** -8
