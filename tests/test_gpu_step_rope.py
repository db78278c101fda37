"""Rotary positions against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_refs as ref
from step_refs import TYPES

pytestmark = pytest.mark.gpu


def heads(rows, n, hd, dt, seed, wide=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((rows, n + wide, hd), generator=g).to(dt).cuda()[:, :n]


def check(hip, q, k, freqs, half, pos, scale=1.0, **where):
    outs = hip.rope(q, k, freqs, half=half, scale=scale, q_out=None if q is None else torch.empty_like(q),
                    k_out=None if k is None else torch.empty_like(k), **where)
    for x, o in ((q, outs[0]), (k, outs[1])):
        if x is not None:
            assert ref.rope_close(o, *ref.rope(x, pos, freqs.cpu(), half, scale))
    return outs


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,rot", [(2, 2), (8, 4), (32, 32), (64, 64), (64, 20), (80, 80), (80, 32), (96, 96), (128, 128),
                                    (128, 96), (128, 34), (192, 64), (256, 256), (100, 50), (512, 512), (512, 498)])
@pytest.mark.parametrize("name", TYPES)
def test_shapes(hip, name, hd, rot, half):
    rows, dt = 6, TYPES[name]
    q, k = heads(rows, 5, hd, dt, 1, 3), heads(rows, 2, hd, dt, 2)
    pos = torch.tensor([0, 1, 77, 4095, 1000003, -9], dtype=torch.int32)
    check(hip, q, k, hip.rope_frequencies(rot, 1e6), half, pos, positions=pos.cuda())


@pytest.mark.parametrize("nq,nk", [(1, 0), (0, 1), (1, 1), (7, 1), (32, 8), (64, 64), (130, 3)])
def test_head_counts(hip, nq, nk):
    q = heads(3, nq, 64, torch.bfloat16, 3) if nq else None
    k = heads(3, nk, 64, torch.bfloat16, 4) if nk else None
    pos = torch.tensor([5, 123456, 2], dtype=torch.int32)
    check(hip, q, k, hip.rope_frequencies(64), True, pos, positions=pos.cuda())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("name", TYPES)
def test_in_place_in_a_fused_projection(hip, name, half):
    """q and k of one buffer, part of the head; everything else stays."""
    g = torch.Generator().manual_seed(5)
    fused = torch.randn((9, 8, 72), generator=g).to(TYPES[name]).cuda()
    before = fused.clone()
    q, k = fused[:, :4], fused[:, 4:6]
    pos = torch.arange(9, dtype=torch.int32) * 1001
    freqs = hip.rope_frequencies(40, 5e5)
    want = [check(hip, x, None, freqs, half, pos, positions=pos.cuda())[0] for x in (q, k)]
    hip.rope(q, k, freqs, positions=pos.cuda(), half=half)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(fused[:, 6:], before[:, 6:]) and torch.equal(fused[:, :, 40:], before[:, :, 40:])


@pytest.mark.parametrize("n_seq", [1, 2, 63, 64, 65, 200, 4097, 5000])
def test_positions_of_a_ragged_batch(hip, n_seq):
    """Sequences without rows among them; rows outside the batch are left alone."""
    r = np.random.RandomState(n_seq)
    rows = r.randint(0, 3, n_seq)
    rows[0], rows[-1] = 2, 1
    starts = np.concatenate([[3], 3 + np.cumsum(rows)]).astype(np.int32)
    lens = (rows + r.randint(0, 100000, n_seq)).astype(np.int32)
    n = int(starts[-1]) + 4
    pos = np.zeros(n, np.int64)
    for s in range(n_seq):
        for i in range(rows[s]):
            pos[starts[s] + i] = lens[s] - rows[s] + i
    x = heads(n, 2, 32, torch.float32, 6)
    freqs = hip.rope_frequencies(32)
    out = torch.full_like(x, 7.0)
    hip.rope(x, None, freqs, starts=torch.from_numpy(starts).cuda(), lens=torch.from_numpy(lens).cuda(), q_out=out)
    inside = slice(3, n - 4)
    want, err = ref.rope(x[inside], torch.from_numpy(pos[inside]), freqs.cpu(), False)
    assert ref.rope_close(out[inside], want, err)
    assert bool((out[:3] == 7).all()) and bool((out[n - 4:] == 7).all())


def test_far_positions_and_scale(hip):
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 10 ** 9 + 7], dtype=torch.int32)
    x = heads(4, 3, 64, torch.float32, 7)
    for kind in ("plain", "linear", "base", "yarn", "model"):
        freqs = hip.rope_frequencies(64, 1e6, kind, 16.0, 4096)
        check(hip, x, None, freqs, False, pos, scale=1.2772588, positions=pos.cuda())


def test_turning_back(hip):
    """A negative position undoes a turn up to the roundings of both."""
    x = heads(5, 2, 64, torch.float32, 8)
    pos = torch.tensor([1, 17, 999, 65536, 10 ** 6], dtype=torch.int32).cuda()
    freqs = hip.rope_frequencies(64)
    there = hip.rope(x, None, freqs, positions=pos, q_out=torch.empty_like(x))[0]
    hip.rope(there, None, freqs, positions=-pos)
    a, b = x[..., 0::2].abs(), x[..., 1::2].abs()
    room = ((a + b) * 2 * 12 * ref.U + 1e-30).repeat_interleave(2, -1)  # |a'| + |b'| <= sqrt 2 (|a| + |b|)
    assert bool(((there - x).abs() <= room).all())


def test_values_that_are_no_numbers_stay_in_their_pair(hip):
    x = heads(2, 2, 64, torch.float32, 9)
    x[0, 1, 6] = float("inf")
    pos = torch.tensor([3, 3], dtype=torch.int32).cuda()
    out = hip.rope(x, None, hip.rope_frequencies(64), positions=pos, q_out=torch.empty_like(x))[0]
    bad = ~out.isfinite()
    assert bool(bad[0, 1, 6:8].all()) and int(bad.sum()) == 2


def test_frequencies(hip):
    f = hip.rope_frequencies(8, 10000.0, device="cpu")
    assert torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    lin = hip.rope_frequencies(8, 10000.0, "linear", 4.0, device="cpu")
    assert torch.allclose(lin * 4, f, rtol=1e-14, atol=0)


def test_no_rows(hip):
    x, freqs = heads(0, 2, 64, torch.float32, 1), hip.rope_frequencies(64)
    none, start = torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    hip.rope(x, None, freqs, positions=none)
    hip.rope(x, x, freqs, starts=start, lens=none)
