"""Products with 4-bit weights of 8-bit inputs whose scales are next to the ends
of f32."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_group", [0, 32, 128])
@pytest.mark.parametrize("batch", [1, 16, 17, 40])
def test_small_scales(hip, batch, x_group):
    """Sums of 3 2^17 and more by two scales whose product is no normal number:
    out is one. (Weights 15, inputs 101 to 127: nothing cancels.)"""
    d, n = 512, 50
    g = torch.Generator().manual_seed(batch)
    x = torch.randint(101, 128, (batch, d), dtype=torch.int8, generator=g)
    s = (torch.rand((batch, d // (x_group or d)), generator=g) + 1) * 1e-37
    w = (torch.full((n, d // 2), 255, dtype=torch.uint8), ((torch.rand((n, d // 128), generator=g) + 1) * 1e-4).half(),
         torch.zeros((n, d // 128), dtype=torch.uint8))
    out = torch.empty((batch, n), device="cuda")
    hip.w4_matmul_rows(out, hip.W4Weights(*(t.cuda() for t in w)), x.cuda(), s.cuda())
    wide = ref.f64(x) * ref.f64(s).repeat_interleave(x_group or d, 1)
    assert bool((ref.f64(out) > 1.2e-38).all()) and ref.w4_close(out, wide, w)


@pytest.mark.parametrize("x_group", [0, 32, 128])
@pytest.mark.parametrize("batch", [1, 16, 17, 40])
def test_large_scales_of_nothing(hip, batch, x_group):
    """Groups of codes 0 add 0, whatever the product of their scales."""
    d, n = 512, 50
    x = torch.zeros((batch, d), dtype=torch.int8)
    s = torch.full((batch, d // (x_group or d)), 1e36)
    x[:, -128:] = 1
    s[:, -1] = 1.0
    w = (torch.full((n, d // 2), 0x99, dtype=torch.uint8), torch.full((n, 4), 1024.0).half(), torch.zeros((n, 4), dtype=torch.uint8))
    if x_group == 32:
        s[:, -4:] = 1.0
    out = torch.empty((batch, n), device="cuda")
    hip.w4_matmul_rows(out, hip.W4Weights(*(t.cuda() for t in w)), x.cuda(), s.cuda())
    assert bool((out == 128 * 9 * 1024.0).all())
