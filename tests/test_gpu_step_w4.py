"""Products with 4-bit weights against 64 bits: every form of the inputs, group
sizes, zeros, sizes that end inside a tile and a step."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_refs as ref
from step_refs import TYPES

pytestmark = pytest.mark.gpu


def weights(n, d, group, zeros, seed=1, dt=torch.float16):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g)
    scales = (torch.randn((n, d // group), generator=g) * 0.01).to(dt)
    z = torch.randint(0, 16, (n, d // group), dtype=torch.uint8, generator=g) if zeros else None
    return codes, scales, z


def on_gpu(hip, w):
    return hip.W4Weights(*(None if t is None else t.cuda() for t in w))


def inputs(batch, d, dt, seed=2):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((batch, d), generator=g) * torch.exp(torch.randn(d, generator=g))).to(dt).cuda()


def run(hip, w, packed, x, dt=None, x_scales=None):
    out = torch.full((x.shape[0] + 1, packed.rows + 3), 9.0, dtype=dt or x.dtype, device="cuda")
    hip.w4_matmul_rows(out[:x.shape[0], :packed.rows], packed, x, x_scales)
    assert bool((out[x.shape[0]:] == 9).all()) and bool((out[:, packed.rows:] == 9).all())
    return out[:x.shape[0], :packed.rows]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,d", [(32, 32), (32, 96), (32, 672), (64, 64), (64, 832), (128, 128), (128, 2048), (256, 1536),
                                     (160, 160), (2048, 2048), (1184, 1184)])
def test_groups_and_columns(hip, name, zeros, group, d):
    for n in (1, 16, 37):
        w = weights(n, d, group, zeros)
        packed = on_gpu(hip, w)
        for batch in (1, 3):
            x = inputs(batch, d, TYPES[name])
            assert ref.w4_close(run(hip, w, packed, x), ref.f64(x), w), (n, batch)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("batch", [1, 2, 5, 6, 10, 11, 16, 17, 21, 22, 32, 33, 64, 65, 80, 130])
def test_batches(hip, name, batch):
    for n, d, group, zeros in ((200, 1280, 64, True), (48, 3200, 128, False), (33, 512, 32, True)):
        w = weights(n, d, group, zeros)
        x = inputs(batch, d, TYPES[name])
        assert ref.w4_close(run(hip, w, on_gpu(hip, w), x), ref.f64(x), w), (n, d)


@pytest.mark.parametrize("n", [2048, 8192, 40000])
@pytest.mark.parametrize("name", TYPES)
def test_waves_of_a_tile(hip, name, n):
    """Row counts that change how many waves share a tile."""
    w = weights(n, 1152, 128, True)
    packed = on_gpu(hip, w)
    for batch in (1, 9):
        x = inputs(batch, 1152, TYPES[name])
        assert ref.w4_close(run(hip, w, packed, x), ref.f64(x), w)


@pytest.mark.parametrize("batch", [1, 16, 70])
def test_deep_rows(hip, batch):
    """More columns than a workgroup holds of the inputs at once."""
    w = weights(20, 16384, 128, True)
    packed = on_gpu(hip, w)
    for dt in TYPES.values():
        x = inputs(batch, 16384, dt)
        assert ref.w4_close(run(hip, w, packed, x), ref.f64(x), w)


def test_bf16_scales(hip):
    w = weights(50, 512, 64, True, dt=torch.bfloat16)
    x = inputs(4, 512, torch.float32)
    assert ref.w4_close(run(hip, w, on_gpu(hip, w), x), ref.f64(x), w)


@pytest.mark.parametrize("x_group", [0, 32, 64, 128, 256, 512])
@pytest.mark.parametrize("group", [32, 64, 128, 1024])
@pytest.mark.parametrize("batch", [1, 8, 33, 65])
def test_8_bit_inputs(hip, x_group, group, batch):
    d = 1024
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-127, 128, (batch, d), dtype=torch.int8, generator=g)
    s = torch.rand((batch, d // (x_group or d)), generator=g) + 0.1
    w = weights(45, d, group, True)
    packed = on_gpu(hip, w)
    wide = ref.f64(x) * ref.f64(s).repeat_interleave(x_group or d, 1)
    for dt in TYPES.values():
        assert ref.w4_close(run(hip, w, packed, x.cuda(), dt, s.cuda()), wide, w)


def test_8_bit_inputs_that_end_inside_a_step(hip):
    for d, group, x_group in ((96, 32, 32), (320, 64, 64), (416, 32, 0), (1184, 1184, 32)):
        g = torch.Generator().manual_seed(4)
        x = torch.randint(-128, 128, (3, d), dtype=torch.int8, generator=g)
        s = torch.rand((3, d // (x_group or d)), generator=g)
        w = weights(19, d, group, True)
        wide = ref.f64(x) * ref.f64(s).repeat_interleave(x_group or d, 1)
        assert ref.w4_close(run(hip, w, on_gpu(hip, w), x.cuda(), torch.float32, s.cuda()), wide, w)


def test_8_bit_sums_are_exact(hip):
    """With scales of one the products are whole numbers below 2^24."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-128, 128, (5, 2048), dtype=torch.int8, generator=g)
    codes = torch.randint(0, 256, (70, 1024), dtype=torch.uint8, generator=g)
    zeros = torch.randint(0, 16, (70, 16), dtype=torch.uint8, generator=g)
    w = (codes, torch.ones((70, 16), dtype=torch.float16), zeros)
    out = run(hip, w, on_gpu(hip, w), x.cuda(), torch.float32, torch.ones(5, device="cuda"))
    assert torch.equal(ref.f64(out), ref.f64(x) @ ref.w4_dense(*w).T)


@pytest.mark.parametrize("name", TYPES)
def test_every_code_and_zero(hip, name):
    """One column at a time: x picks a column, scales of one: c - z itself."""
    d = 256
    codes = (torch.arange(16 * d // 2) * 37 % 256).to(torch.uint8).view(16, d // 2)
    zeros = (torch.arange(16 * 8) % 16).to(torch.uint8).view(16, 8)
    w = (codes, torch.ones((16, 8), dtype=torch.float16), zeros)
    x = torch.eye(d, dtype=TYPES[name]).cuda()
    assert torch.equal(ref.f64(run(hip, w, on_gpu(hip, w), x)), ref.w4_dense(*w).T)


def test_range_of_f32_inputs(hip):
    """24 bits of each input, however large or small (a group's sum without its scale is an f32 number)."""
    w = weights(40, 256, 64, False)
    packed = on_gpu(hip, w)
    for scale in (1e34, 1e-30):
        x = inputs(2, 256, torch.float32).clamp(-8, 8) * scale
        assert ref.w4_close(run(hip, w, packed, x), ref.f64(x), w), scale


def test_no_number_stays_in_its_row(hip):
    w = weights(40, 512, 128, False)
    packed = on_gpu(hip, w)
    for dt in TYPES.values():
        x = inputs(7, 512, dt)
        want = run(hip, w, packed, x).clone()
        x[3, 100] = float("inf")
        x[5, 7] = float("nan")
        out = run(hip, w, packed, x)
        keep = [0, 1, 2, 4, 6]
        assert torch.equal(out[keep], want[keep]) and not bool(out[5].isfinite().any())
        assert not bool(out[3].isfinite().any())


@pytest.mark.parametrize("name", TYPES)
def test_strided_inputs(hip, name):
    w = weights(30, 320, 64, True)
    x = inputs(6, 333, TYPES[name])[:, 5:325]
    assert ref.w4_close(run(hip, w, on_gpu(hip, w), x), ref.f64(x), w)


def test_no_inputs(hip):
    w = weights(30, 320, 64, True)
    packed = on_gpu(hip, w)
    out = torch.empty((0, 30), device="cuda")
    hip.w4_matmul_rows(out, packed, torch.empty((0, 320), device="cuda"))


def test_more_blocks_than_one(hip):
    """A batch of several blocks of inputs."""
    w = weights(100, 384, 128, True)
    for dt in TYPES.values():
        x = inputs(1000, 384, dt)
        assert ref.w4_close(run(hip, w, on_gpu(hip, w), x), ref.f64(x), w)


@pytest.mark.parametrize("batch", [1, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 128])
def test_sums_keep_the_bits_of_f32(hip, batch, group):
    """The root mean square of the errors, each over the root of its products'
    squares. Partial sums are about that root; some 60 sums of a value each round
    to 2^-24 of it (random: 5 2^-24), 22-bit inputs add 2.3 2^-24: 2^-20 in all is
    twice that. (Sums of 17 bits give 2^-17.)"""
    d = 4096
    w = weights(300, d, group, True)
    packed, dense = on_gpu(hip, w), ref.w4_dense(*w)
    x = inputs(batch, d, torch.float32)
    g = torch.Generator().manual_seed(6)
    c = torch.randint(-127, 128, (batch, d), dtype=torch.int8, generator=g)
    s = torch.rand((batch, d // 128), generator=g) + 0.1
    wide = ref.f64(c) * ref.f64(s).repeat_interleave(128, 1)
    for out, v in ((run(hip, w, packed, x), ref.f64(x)),
                   (run(hip, w, packed, c.cuda(), torch.float32, s.cuda()), wide)):
        error = (ref.f64(out) - v @ dense.T) / torch.sqrt((v * v) @ (dense * dense).T)
        assert float(error.square().mean().sqrt()) < 2.0 ** -20
