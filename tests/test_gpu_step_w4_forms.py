"""Sizes that reach every layout of the products with 4-bit weights: few inputs
on 8 and 16 waves; one to eight tiles of columns on 8 and 16 waves."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref
from step_refs import TYPES

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (1, 15, 16), (1, 34, 14), (1, 1, 17), (9221, 3, 17), (1, 9, 19), (4206, 3, 23), (4213, 5, 34),
          (4549, 3, 52), (8662, 3, 57), (10882, 1, 58), (11000, 2, 67), (22560, 1, 68), (8320, 3, 77), (22025, 1, 100),
          (35, 5, 1310), (136, 3, 1700), (265, 1, 1800), (134, 3, 1650), (18169, 1, 32)]


@pytest.mark.parametrize("n,steps,batch", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32", "i8"])
def test_form(hip, kind, group, n, steps, batch):
    d = steps * 128 - (32 if group == 32 else 64 if group == 64 and steps > 1 else 0)
    g = torch.Generator().manual_seed(n + batch)
    w = (torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g),
         (torch.randn((n, d // group), generator=g) * 0.01).half(),
         torch.randint(0, 16, (n, d // group), dtype=torch.uint8, generator=g))
    packed = hip.W4Weights(*(t.cuda() for t in w))
    if kind == "i8":
        x, xg = torch.randint(-127, 128, (batch, d), dtype=torch.int8, generator=g), 32 if d % 128 else 128
        s = torch.rand((batch, d // xg), generator=g) + 0.1
        wide, dt = ref.f64(x) * ref.f64(s).repeat_interleave(xg, 1), torch.float32
        out = torch.full((batch, n), 9.0, device="cuda")
        hip.w4_matmul_rows(out, packed, x.cuda(), s.cuda())
    else:
        x = (torch.randn((batch, d), generator=g) * torch.exp(torch.randn(d, generator=g))).to(TYPES[kind])
        wide = ref.f64(x)
        out = torch.full((batch, n), 9.0, dtype=x.dtype, device="cuda")
        hip.w4_matmul_rows(out, packed, x.cuda())
    assert ref.w4_close(out, wide, w)
