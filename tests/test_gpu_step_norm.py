"""Root-mean-square norms of rows against 64 bits: both outputs, residuals,
strides, every way that a row is spread over lanes and waves."""
from __future__ import annotations

import pytest
import torch

import step_refs as ref
from step_refs import TYPES

pytestmark = pytest.mark.gpu


def make(shape, dt, seed, wide=0):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(torch.randn(shape[-1], generator=g))
    x = torch.randn((*shape[:-1], shape[-1] + wide), generator=g)
    return (x * torch.cat([spread, torch.ones(wide)])).to(dt).cuda()[..., :shape[-1]]


def weight(dim, seed=9):
    return (1 + 0.3 * torch.randn(dim, generator=torch.Generator().manual_seed(seed))).cuda()


# lanes of a wave from one to all, waves from 2 to 16, 1 to 4 chunks a thread, and
# rows that are read twice; sizes that end inside a chunk
DIMS = [1, 7, 8, 9, 31, 64, 65, 127, 250, 512, 513, 1000, 2048, 8191, 8192, 8200, 16384, 16390, 32768, 32771, 70001]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("name", TYPES)
def test_rows(hip, name, dim):
    dt, rows = TYPES[name], 5 if dim < 4000 else 2
    x, r, w = make((rows, dim), dt, 1), make((rows, dim), dt, 2), weight(dim)
    out, s = torch.empty_like(x), torch.empty_like(x)
    hip.rms_norm(out, x, w, 1e-5, residual=r, residual_out=s)
    want_s, want = ref.norm(x, w, 1e-5, r)
    assert ref.norm_close(out, want) and ref.sum_close(s, want_s)
    plain = torch.empty_like(x)
    hip.rms_norm(plain, x, w, 1e-6)
    assert ref.norm_close(plain, ref.norm(x, w, 1e-6)[1])


@pytest.mark.parametrize("rows", [0, 1, 3, 4, 63, 1025])
def test_row_counts(hip, rows):
    for dim in (24, 640):
        x, w = make((rows, dim), torch.bfloat16, 3), weight(dim)
        out = torch.empty_like(x)
        hip.rms_norm(out, x, w)
        if rows:
            assert ref.norm_close(out, ref.norm(x, w, 1e-5)[1])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 64), (5, 33), (2, 700)])
def test_heads_of_a_fused_projection(hip, name, heads, dim):
    """[rows, heads, dim] with other columns between heads and rows, which stay."""
    dt = TYPES[name]
    g = torch.Generator().manual_seed(4)
    fused = torch.randn((7, heads + 2, dim + 3), generator=g).to(dt).cuda()
    before = fused.clone()
    x, w = fused[:, 1:1 + heads, 2:2 + dim], weight(dim)
    out = torch.full((7, heads + 1, dim), 5.0, dtype=dt, device="cuda")
    want = ref.norm(x, w, 1e-5)[1]
    hip.rms_norm(out[:, :heads], x, w)
    assert ref.norm_close(out[:, :heads], want) and bool((out[:, heads:] == 5).all())
    hip.rms_norm(x, x, w)  # in place
    assert torch.equal(x, out[:, :heads])
    before[:, 1:1 + heads, 2:2 + dim] = x
    assert torch.equal(before, fused)


@pytest.mark.parametrize("dim", [40, 2048, 40000])
def test_residual_in_place(hip, dim):
    x, r, w = make((3, dim), torch.bfloat16, 5), make((3, dim), torch.bfloat16, 6), weight(dim)
    out, s = torch.empty_like(x), torch.empty_like(x)
    hip.rms_norm(out, x, w, residual=r, residual_out=s)
    hip.rms_norm(x, x, w, residual=r, residual_out=r)
    assert torch.equal(x, out) and torch.equal(r, s)


def test_large_and_small_values(hip):
    """Squares past f32 and far below it; rows of zeros; an infinity stays in its row."""
    x = make((6, 200), torch.float32, 7)
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2] = 0
    x[3, 17] = float("inf")
    x[4, 5] = float("nan")
    w = weight(200)
    out = torch.empty_like(x)
    hip.rms_norm(out, x, w, 1e-30)
    want = ref.norm(x, w, 1e-30)[1]
    for i in (0, 1, 2, 5):
        assert ref.norm_close(out[i], want[i]), i
    assert out[4].isnan().all() and bool((out[3].cpu().isnan() == want[3].isnan()).all())


@pytest.mark.parametrize("group", [0, 32, 64, 128, 256, 512])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_8_bits(hip, name, group, residual):
    """Codes equal the definition's, ties among them (16-bit values with weights
    that are powers of two)."""
    dt = TYPES[name]
    for dim in ([512, 1536, 8704, 16384, 17408] if group else [1, 100, 512, 4099, 16384, 16401]):
        rows = 3 if dim < 9000 else 2
        x, w = make((rows, dim), dt, 8), weight(dim)
        if dim == 512:
            w = torch.exp2(torch.arange(dim) % 3).float().cuda()
        r = make((rows, dim), dt, 9) if residual else None
        s = torch.empty_like(x) if residual else None
        codes = torch.empty((rows, dim), dtype=torch.int8, device="cuda")
        scales = torch.empty((rows, dim // group if group else 1), device="cuda")
        hip.rms_norm_q8(codes, scales, x, w, 1e-5, residual=r, residual_out=s)
        want_c, want_s = ref.norm_q8(x, w, 1e-5, group, r)
        assert torch.equal(codes.cpu().double(), want_c), (dim, (codes.cpu().double() != want_c).sum())
        # rounded to f32 once; its 64-bit factors may differ in their last bits
        assert bool(((ref.f64(scales) - want_s).abs() <= want_s * ref.U * 1.0001).all())
        if residual:
            assert ref.sum_close(s, ref.f64(x) + ref.f64(r))


def test_8_bits_of_ties(hip):
    """Every multiple of half a code, at several largest values."""
    tops = torch.tensor([127.0, 2.0, 254.0, 3.0, 127 * 0.375])
    x = torch.zeros((5, 512))
    half = torch.arange(-254, 255) / 254
    x[:, :509] = tops[:, None] * half
    x[:, 511] = tops
    x = x.cuda()
    codes, scales = torch.empty((5, 512), dtype=torch.int8, device="cuda"), torch.empty((5, 1), device="cuda")
    w = torch.ones(512, device="cuda")
    hip.rms_norm_q8(codes, scales, x, w)
    assert torch.equal(codes.cpu().double(), ref.norm_q8(x, w, 1e-5, 0)[0])


@pytest.mark.parametrize("group", [0, 64])
def test_8_bits_of_nothing_and_of_infinities(hip, group):
    x, w = make((5, 640), torch.float32, 11), weight(640)
    x[0] = 0
    x[1, 64:128] = 0
    x[2, 70] = float("inf")
    x[3, 600] = float("nan")
    w2 = w.clone()
    w2[130] = float("nan")
    codes = torch.empty((5, 640), dtype=torch.int8, device="cuda")
    scales = torch.empty((5, 640 // (group or 640)), device="cuda")
    hip.rms_norm_q8(codes, scales, x, w)
    assert bool((codes[0] == 0).all()) and bool((scales[0] == 0).all())
    want_c, want_s = ref.norm_q8(x, w, 1e-5, group)
    for i in (1, 4):
        assert torch.equal(codes[i].cpu().double(), want_c[i])
    for i in (2, 3):
        assert bool((codes[i] == 0).all()) and bool(scales[i].isnan().all())
    if group:
        assert float(scales[1, 1]) == 0
    hip.rms_norm_q8(codes, scales, x, w2)
    bad = slice(128, 192) if group else slice(None)
    assert bool((codes[4, bad] == 0).all()) and int(scales[4].isnan().sum()) == 1
    if group:
        keep = torch.ones(640, dtype=torch.bool)
        keep[bad] = False
        assert torch.equal(codes[4].cpu().double()[keep], want_c[4][keep])
