"""Products with 4-bit weights: more inputs than a launch has blocks for the
narrowest tiles."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,batch", [("f16", 65535 * 16 + 50), ("f32", 65535 * 8 + 50), ("i8", 65535 * 16 + 50)])
def test_many_inputs_of_few_rows(hip, kind, batch):
    """All are written; those next to the ends of blocks and launches are right."""
    n, d = 9, 768
    g = torch.Generator().manual_seed(1)
    w = (torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g),
         (torch.randn((n, d // 128), generator=g) * 0.01).half(),
         torch.randint(0, 16, (n, d // 128), dtype=torch.uint8, generator=g))
    packed = hip.W4Weights(*(t.cuda() for t in w))
    g = torch.Generator("cuda").manual_seed(2)
    at = torch.cat([torch.arange(a, min(a + 80, batch)) for a in (0, 1 << 17, (1 << 18) - 40, (1 << 19) - 40, batch - 80)])
    if kind == "i8":
        x = torch.randint(-127, 128, (batch, d), dtype=torch.int8, device="cuda", generator=g)
        s = torch.rand((batch, d // 128), device="cuda", generator=g) + 0.1
        out = torch.full((batch, n), 9e9, device="cuda")
        hip.w4_matmul_rows(out, packed, x, s)
        wide = ref.f64(x[at.cuda()]) * ref.f64(s[at.cuda()]).repeat_interleave(128, 1)
    else:
        x = torch.randn((batch, d), device="cuda", generator=g).to(ref.TYPES[kind])
        out = torch.full((batch, n), 9e4 if kind == "f32" else 6e4, dtype=x.dtype, device="cuda")
        hip.w4_matmul_rows(out, packed, x)
        wide = ref.f64(x[at.cuda()])
    assert bool((out < (9e8 if kind == "i8" else 5e4)).all())
    assert ref.w4_close(out[at.cuda()], wide, w)
