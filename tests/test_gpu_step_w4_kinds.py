"""Products with 4-bit weights: every kind of input with and without zeros, f16 and
bf16 scales, in every kind of layout (few inputs; more, on 8 and on 16 waves; whole
rows and steps that end inside)."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref
from step_refs import TYPES

pytestmark = pytest.mark.gpu

# rows, columns, inputs
SIZES = [(37, 320, 1), (2100, 2048, 8), (45, 1024, 33), (200, 1280, 16), (4549, 384, 52), (300, 896, 70), (8320, 384, 77)]


def check(hip, kind, zeros, scales, group, n, d, batch, x_group=128):
    g = torch.Generator().manual_seed(n + batch)
    s = (torch.randn((n, d // group), generator=g) * 0.01).to(scales)
    w = (torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g), s,
         torch.randint(0, 16, (n, d // group), dtype=torch.uint8, generator=g) if zeros else None)
    packed = hip.W4Weights(*(None if t is None else t.cuda() for t in w))
    if kind == "i8":
        x = torch.randint(-127, 128, (batch, d), dtype=torch.int8, generator=g)
        xs = torch.rand((batch, d // (x_group or d)), generator=g) + 0.1
        wide = ref.f64(x) * ref.f64(xs).repeat_interleave(x_group or d, 1)
        for dt in TYPES.values():
            out = torch.full((batch, n), 9.0, dtype=dt, device="cuda")
            hip.w4_matmul_rows(out, packed, x.cuda(), xs.cuda())
            assert ref.w4_close(out, wide, w), dt
    else:
        x = (torch.randn((batch, d), generator=g) * torch.exp(torch.randn(d, generator=g))).to(TYPES[kind])
        out = torch.full((batch, n), 9.0, dtype=x.dtype, device="cuda")
        hip.w4_matmul_rows(out, packed, x.cuda())
        assert ref.w4_close(out, ref.f64(x), w)


@pytest.mark.parametrize("n,d,batch", SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("scales", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32", "i8"])
def test_kinds(hip, kind, zeros, scales, group, n, d, batch):
    if d % group:
        group = 64
    check(hip, kind, zeros, scales, group, n, d, batch, 32 if d % 128 else 128)


@pytest.mark.parametrize("x_group", [0, 32, 64, 256, 512])
@pytest.mark.parametrize("group", [32, 64, 128, 1024])
@pytest.mark.parametrize("batch", [1, 8, 33, 65])
def test_8_bit_inputs_without_zeros(hip, x_group, group, batch):
    check(hip, "i8", False, torch.bfloat16, group, 45, 1024, batch, x_group)


@pytest.mark.parametrize("batch", [1, 5, 40])
def test_8_bit_sums_are_exact_without_zeros(hip, batch):
    """With scales of one the products are whole numbers below 2^24."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-128, 128, (batch, 2048), dtype=torch.int8, generator=g)
    w = (torch.randint(0, 256, (70, 1024), dtype=torch.uint8, generator=g), torch.ones((70, 16), dtype=torch.bfloat16), None)
    out = torch.empty((batch, 70), device="cuda")
    hip.w4_matmul_rows(out, hip.W4Weights(w[0].cuda(), w[1].cuda()), x.cuda(), torch.ones(batch, device="cuda"))
    assert torch.equal(ref.f64(out), ref.f64(x) @ ref.w4_dense(*w).T)
