"""The step's operators on rows and weights whose offsets pass 32 bits."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu

FAR = 2_300_000_003  # elements between rows: odd, past 31 bits; twice it past 32


@pytest.fixture(scope="module")
def room():
    """Three rows of up to 1024 bf16 values that far apart."""
    x = torch.empty(2 * FAR + 1024, dtype=torch.bfloat16, device="cuda")
    yield x
    del x
    torch.cuda.empty_cache()


def rows(room, n, dim, seed):
    v = room.as_strided((n, dim), (FAR, 1))
    v.copy_(torch.randn((n, dim), generator=torch.Generator().manual_seed(seed)))
    return v


@pytest.mark.parametrize("dim", [96, 1000])
def test_norm(hip, room, dim):
    x, w = rows(room, 3, dim, 1), torch.rand(dim, generator=torch.Generator().manual_seed(2)).cuda() + 0.5
    out = torch.empty((3, dim), dtype=torch.bfloat16, device="cuda")
    hip.rms_norm(out, x, w)
    want = ref.norm(x, w, 1e-5)[1]
    assert ref.norm_close(out, want)
    codes, scales = torch.empty((3, dim), dtype=torch.int8, device="cuda"), torch.empty((3, 1), device="cuda")
    hip.rms_norm_q8(codes, scales, x, w)
    assert torch.equal(codes.cpu().double(), ref.norm_q8(x, w, 1e-5, 0)[0])
    hip.rms_norm(x, x, w)
    assert torch.equal(x, out)


def test_rope(hip, room):
    x = rows(room, 3, 512, 3).unflatten(1, (4, 128))
    pos, freqs = torch.tensor([7, 100000, 3], dtype=torch.int32), hip.rope_frequencies(128)
    want, err = ref.rope(x, pos, freqs.cpu(), True)
    hip.rope(x, None, freqs, positions=pos.cuda(), half=True)
    assert ref.rope_close(x, want, err)


@pytest.mark.parametrize("batch", [3])
def test_w4_inputs_and_outputs(hip, room, batch):
    g = torch.Generator().manual_seed(4)
    w = (torch.randint(0, 256, (200, 256), dtype=torch.uint8, generator=g), torch.rand((200, 4), generator=g).half(), None)
    packed = hip.W4Weights(w[0].cuda(), w[1].cuda())
    x = torch.randn((batch, 512), generator=g).to(torch.bfloat16).cuda()
    out = room.as_strided((batch, 200), (FAR, 1))
    hip.w4_matmul_rows(out, packed, x)
    assert ref.w4_close(out, ref.f64(x), w)
    near = out.clone()
    hip.w4_matmul_rows(near, packed, rows(room, batch, 512, 5))
    assert ref.w4_close(near, ref.f64(room.as_strided((batch, 512), (FAR, 1))), w)


def test_verify(hip, room):
    """Rows of probabilities 2.3 G values apart (f32: every second of the room's)."""
    far = FAR // 2
    p = room.view(torch.float32)[:2 * far + 400].as_strided((3, 400), (far, 1))
    g = torch.Generator().manual_seed(6)
    p.copy_(torch.softmax(torch.randn((3, 400), generator=g), -1))
    q = torch.softmax(torch.randn((3, 400), generator=g), -1)
    b = dict(drafted=torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32), accept=torch.tensor([0.0, 0.9, 0.5]),
             pick=torch.tensor([0.4]), starts=torch.tensor([0, 3], dtype=torch.int32))
    tokens, counts = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    hip.verify_rows(tokens, counts, p, b["drafted"].cuda(), b["accept"].cuda(), b["pick"].cuda(), b["starts"].cuda(),
                    draft=q.cuda())
    want_t, want_c = ref.verify(target=p, draft=q, **b)
    assert tokens.tolist() == want_t.tolist() and counts.tolist() == want_c.tolist()


@pytest.mark.parametrize("batch", [1, 20])
def test_w4_weights(hip, batch):
    """5.7 GB of codes; the last rows against 64 bits."""
    n, d, group = 700_000, 16384, 512
    g = torch.Generator("cuda").manual_seed(7)
    codes = torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.rand((n, d // group), device="cuda", generator=g).half()
    packed = hip.W4Weights(codes, scales)
    x = torch.randn((batch, d), device="cuda", generator=g).half()
    out = torch.empty((batch, n), dtype=torch.float16, device="cuda")
    hip.w4_matmul_rows(out, packed, x * 0.01)
    for at in (slice(0, 40), slice(524280, 524320), slice(n - 40, n)):
        assert ref.w4_close(out[:, at], ref.f64(x * 0.01), (codes[at], scales[at], None))
