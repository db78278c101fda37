"""4-bit weights laid out on a stream that is behind the current one."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
def test_inputs_that_are_dropped(hip, handle, zeros):
    """The constructor's inputs are not kept: their memory goes to other tensors of
    the current stream, but only behind the layout's work."""
    n, d = 1024, 4096
    g = torch.Generator().manual_seed(1)
    host = [torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g), torch.rand((n, d // 64), generator=g).half(),
            torch.randint(0, 16, (n, d // 64), dtype=torch.uint8, generator=g) if zeros else None]
    want = hip.W4Weights(*(None if t is None else t.cuda() for t in host)).data.clone()
    busy = torch.zeros(1 << 29, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    tensors = [None if t is None else t.cuda() for t in host]
    shapes = [(t.shape, t.dtype) for t in tensors if t is not None]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):  # some 8 ms
            busy.add_(1)
    packed = hip.W4Weights(*tensors, stream=side.cuda_stream if handle else side)
    del tensors
    later = [torch.ones(shape, dtype=dt, device="cuda") for shape, dt in shapes for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(packed.data, want) and all(bool((t == 1).all()) for t in later)
