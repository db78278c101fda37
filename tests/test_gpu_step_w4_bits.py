"""Products with 4-bit weights keep the bits of f32, whatever the groups and the
layout."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu

D = 2048


@pytest.mark.parametrize("batch", [1, 2, 8, 9, 17, 33, 80, 130])
@pytest.mark.parametrize("group", [32, 64, 256, D])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["f32", "i8", "i8 rows", "i8 32"])
def test_bits(hip, kind, zeros, group, batch):
    """The root mean square of the errors, each over the root of its products'
    squares, which partial sums are about. A value's sums: in an instruction 32
    products deep, 4 instructions and 16 steps in turn, 8 waves: some 60 roundings to
    2^-24 (random: 5 2^-24); of 8-bit inputs whole numbers instead, then up to 64
    groups' two products and sum (8 2^-24); f32 inputs 2^-23 each at most (1.2 2^-24).
    2^-20 in all is twice that."""
    g = torch.Generator().manual_seed(batch + group)
    w = (torch.randint(0, 256, (200, D // 2), dtype=torch.uint8, generator=g),
         (torch.rand((200, D // group), generator=g) * 0.01 + 0.005).half(),
         torch.randint(0, 16, (200, D // group), dtype=torch.uint8, generator=g) if zeros else None)
    packed = hip.W4Weights(*(None if t is None else t.cuda() for t in w))
    out = torch.empty((batch, 200), device="cuda")
    if kind == "f32":
        x = torch.randn((batch, D), generator=g)
        hip.w4_matmul_rows(out, packed, x.cuda())
        v = ref.f64(x)
    else:
        x_group = {"i8": 128, "i8 rows": D, "i8 32": 32}[kind]
        x = torch.randint(-127, 128, (batch, D), dtype=torch.int8, generator=g)
        s = torch.rand((batch, D // x_group), generator=g) + 0.1
        hip.w4_matmul_rows(out, packed, x.cuda(), s.cuda())
        v = ref.f64(x) * ref.f64(s).repeat_interleave(x_group, 1)
    dense = ref.w4_dense(*w)
    error = (ref.f64(out) - v @ dense.T) / torch.sqrt((v * v) @ (dense * dense).T)
    assert float(error.square().mean().sqrt()) < 2.0 ** -20
