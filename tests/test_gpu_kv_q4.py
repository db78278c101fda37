"""The paged 4-bit cache against its definition in 64 bits: rows written and
read back, and attention over what is held."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def held(x):
    """The values that x[..., hd] is held as, in 64 bits, from the definition."""
    x = x.double().cpu().numpy()
    x = np.clip(np.where(np.isnan(x), 0.0, x), -21760.0, 21760.0)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = x.max(-1), x.min(-1)
    y = np.clip(np.where(hi >= -lo, hi, lo) / -8, -2720.0, 2720.0)
    man, ex = np.frexp(y)
    d = np.ldexp(np.rint(man * 256), ex - 8)          # 8 significant bits
    d = d.astype(np.float16).astype(np.float64)[..., None]  # fp16's exponents
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(d == 0, 0.0, np.clip(np.rint(x / d), -8, 7))
    return torch.from_numpy((n * d).reshape(*x.shape[:-2], x.shape[-2] * 32))


class Batch:
    """A cache of `kv` heads with shuffled pages, filled with `fill` bytes."""

    def __init__(self, hip, rows, lens, kv, hd, page, cap=None, fill=0xFF, seed=0):
        r = np.random.RandomState(seed)
        per = max(1, -(-(cap or max(max(lens), 1)) // page))
        n = len(lens)
        self.ids = r.permutation(n * per + 2)[:n * per].reshape(n, per)
        self.data = torch.full(((n * per + 2) * hip.kv_q4_page_bytes(kv, hd, page),), fill, dtype=torch.uint8,
                               device="cuda")
        self.pages = torch.from_numpy(self.ids.astype(np.int32)).cuda()
        self.cache = hip.KvCacheQ4(self.data, self.pages, kv, hd, page)
        self.rows, self.lens, self.kv, self.hd, self.page = list(rows), list(lens), kv, hd, page
        self.starts_t, self.lens_t = self.tensors(rows, lens)

    @staticmethod
    def tensors(rows, lens):
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        return torch.from_numpy(starts).cuda(), torch.tensor(list(lens), dtype=torch.int32, device="cuda")

    def fill(self, hip, seed=1, scale=1.0, dtype=torch.float32):
        """Every position of every sequence written; what is held [n][kv, len, hd] in 64 bits."""
        g = torch.Generator().manual_seed(seed)
        total = sum(self.lens)
        k = (torch.randn((total, self.kv, self.hd), generator=g) * scale).to(dtype)
        v = (torch.randn((total, self.kv, self.hd), generator=g) * scale).to(dtype)
        if total:
            s, l = self.tensors(self.lens, self.lens)
            hip.kv_q4_append(self.cache, k.cuda(), v.cuda(), s, l)
        at = np.concatenate([[0], np.cumsum(self.lens)])
        hk, hv = held(k), held(v)
        return [(hk[a:b].transpose(0, 1), hv[a:b].transpose(0, 1)) for a, b in zip(at[:-1], at[1:])]


def reference(q, kvs, rows, lens, scale, window=0):
    """(outputs, bound terms) per row and head in 64 bits: the outputs, sum of
    w |v| and the largest |q| |k| sum of the row times the scale."""
    q = q.double().cpu()
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    top = torch.zeros(q.shape[:2], dtype=torch.float64)
    at = 0
    for (k, v), n, t in zip(kvs, rows, lens):
        g = q.shape[1] // k.shape[0]
        for i in range(n):
            pos = t - n + i
            lo = max(0, pos + 1 - window) if window else 0
            if pos < 0 or pos + 1 > k.shape[1]:
                continue
            kk, vv = k[:, lo:pos + 1].repeat_interleave(g, 0), v[:, lo:pos + 1].repeat_interleave(g, 0)
            s = (kk @ q[at + i][:, :, None])[..., 0] * scale
            w = torch.softmax(s, -1)
            out[at + i] = (w[:, None] @ vv)[:, 0]
            mag[at + i] = (w[:, None] @ vv.abs())[:, 0]
            top[at + i] = (kk.abs() @ q[at + i].abs()[:, :, None])[..., 0].amax(-1) * abs(scale)
        at += n
    return out, mag, top


def check_attention(got, want, mag, top, dtype, hd, longest, big=6.0):
    """Weights: a score is off by its products' f32 sums (hd + 4 roundings of
    2^-24 of sum |q k|), by the queries' planes (2^-22 in f32, none in the
    others) and by three roundings of the exponent; its weight by as much
    relative to itself, plus 2^-22 of the exponential, plus 2^-11 where weights
    are one fp16 plane and 2^-22 where two. Numerator and denominator: twice
    that. Sums over the tokens: no chain is longer than one in four of them
    plus the joins. A weight is an fp16 number times 2^-11 of the row's reference,
    which is no larger than its largest weight: the last plane of one so small
    that it is a denormal is off by half of 2^-24 there, 2^-36 of the largest and
    so of the denominator; over `longest` tokens of values up to `big` that is
    longest * 2^-36 * big. Then half a step of the output's type."""
    u = 2.0 ** -24
    planes = 2.0 ** -22 if dtype == torch.float32 else 0.0
    eps = top[..., None] * ((hd + 8) * u + planes) + 2.0 ** -21
    eps = eps + (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11)
    bound = mag * (2 * eps + (longest / 4 + 64) * u) + longest * 2.0 ** -36 * big
    bound = bound + (want.abs() + bound) * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / bound).max().item()
    assert worst <= 1.0, worst


# ------------------------------------------------------- writing, reading
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd,page,rows,lens", [
    (1, 32, 32, [1], [1]),
    (2, 64, 64, [1, 1, 1], [1, 64, 65]),
    (3, 96, 96, [5, 0, 33], [5, 7, 200]),
    (8, 64, 256, [130], [300]),
    (2, 128, 32, [31, 32, 33, 64], [31, 40, 33, 100]),
    (1, 192, 64, [70, 2], [70, 129]),
    (2, 256, 128, [3, 40], [130, 40]),
])
def test_rows_written_and_read_back(hip, name, kv, hd, page, rows, lens):
    b = Batch(hip, rows, lens, kv, hd, page, fill=0x5A)
    g = torch.Generator().manual_seed(hd)
    dt = TYPES[name]
    x = torch.randn((sum(rows), 2 * kv, hd), generator=g).to(dt)
    k, v = x[:, :kv], x[:, kv:]  # strided: parts of one projection
    xc = x.cuda()
    before = b.data.clone()
    hip.kv_q4_append(b.cache, xc[:, :kv], xc[:, kv:], b.starts_t, b.lens_t)
    for out_t in (torch.float32, dt):
        ko, vo = (torch.empty((sum(rows), kv, hd), dtype=out_t, device="cuda") for _ in range(2))
        hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
        assert torch.equal(ko.cpu(), held(k).to(out_t)) and torch.equal(vo.cpu(), held(v).to(out_t))
    # two nibbles and two scales a dimension pair, and nothing else, were written
    changed = (b.data != before).sum().item()
    assert changed <= sum(rows) * kv * (hd + hd // 32 * 4)
    used = {int(b.ids[s, p // page]) for s, (n, t) in enumerate(zip(rows, lens)) for p in range(t - n, t)}
    per_page = (b.data != before).view(-1, hip.kv_q4_page_bytes(kv, hd, page)).any(1).nonzero().flatten().tolist()
    assert set(per_page) <= used


def test_layout_of_a_group(hip):
    """The documented order of a group's bytes, by hand for hd 64."""
    hd = 64
    b = Batch(hip, [32], [32], 1, hd, 32, fill=0)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn((32, 1, hd), generator=g), torch.randn((32, 1, hd), generator=g)
    hip.kv_q4_append(b.cache, k.cuda(), v.cuda(), b.starts_t, b.lens_t)
    size = hip.kv_q4_page_bytes(1, hd, 32)
    raw = b.data.cpu().numpy()[int(b.ids[0, 0]) * size:][:size]
    sc = raw[32 * hd:].view(np.float16).astype(np.float64)
    hk, hv = held(k)[:, 0].numpy(), held(v)[:, 0].numpy()
    for t in range(32):
        for d in range(hd):
            blk, i = d // 32, d % 32
            lane = t % 16 + 16 * (i // 8)
            word = raw[lane * 16 + blk * 8 + t // 16 * 4:][:4].view("<u4")[0]
            e = i % 8
            code = int(word) >> (4 * (e // 2) + 16 * (e % 2)) & 15
            assert (code - 8) * sc[t % 16 * 4 + t // 16 * 2 + blk] == hk[t, d]
            lane = i % 16 + 16 * (t % 16 // 4)
            byte = raw[16 * hd + lane * 16 + blk * 8 + t // 16 * 4 + [0, 2, 1, 3][t % 4]]
            code = int(byte) >> (4 * (i // 16)) & 15
            assert (code - 8) * sc[hd + blk * 32 + t % 16 // 4 * 8 + t // 16 * 4 + t % 4] == hv[t, d]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_values_at_the_edges(hip, name):
    """NaN, infinities, values past the largest, denormals, ties of the scale and of the codes."""
    dt = TYPES[name]
    g = torch.Generator().manual_seed(5)
    x = torch.randn((16, 2, 64), generator=g)
    x[0, 0, 3] = math.nan
    x[1, 0, 40] = math.inf
    x[1, 1, 2] = -math.inf
    x[2] = 0.0
    x[3] *= 1e-6
    x[4] *= 1e-7
    x[5] = 3e38 if dt != torch.float16 else 65504.0
    x[6, 0] = -65504.0
    x[7, :, ::2] = 2.0
    x[7, :, 1::2] = -2.0                                  # a tie of the two ends
    x[8] = (torch.arange(64) % 33 - 16).float() / 2       # quotients of one half
    x[9] = -(torch.arange(64) % 33 - 16).float() / 2
    x[10] = math.nan
    x[11] = -2720.0 * 8
    x[12] = torch.rand((2, 64), generator=g) * 8192 * 2 ** -24
    x[13, 0, :32] = 1.0
    x[13, 0, 5] = 1 + 2.0 ** -8 + 2.0 ** -9               # the scale rounds up, down, and at a tie
    x[13, 0, 32:] = 1 + 2.0 ** -8
    x[13, 1, :32] = 1 + 3 * 2.0 ** -8
    x[14, :, 7] = 1e4
    x = x.to(dt)
    b = Batch(hip, [16], [16], 2, 64, 32)
    hip.kv_q4_append(b.cache, x.cuda(), x.cuda().flip(0).contiguous(), b.starts_t, b.lens_t)
    ko, vo = (torch.empty((16, 2, 64), device="cuda") for _ in range(2))
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    want = held(x)
    assert torch.isfinite(want).all()
    assert torch.equal(ko.cpu().double(), want) and torch.equal(vo.cpu().double(), want.flip(0))


def test_codes_next_to_a_half(hip):
    """f32 values one step either side of a code's border, for many scales."""
    g = torch.Generator().manual_seed(6)
    m = (1 + torch.randint(0, 256, (4096, 1), generator=g) / 256) * 2.0 ** torch.randint(-6, 7, (4096, 1), generator=g)
    d = -(m / -8).double()
    half = (torch.randint(-8, 7, (4096, 32), generator=g) + 0.5) * d
    x = half.float()
    way = torch.randint(0, 3, x.shape, generator=g)
    x = torch.where(way == 0, torch.nextafter(x, torch.tensor(9e9)), torch.where(way == 1, torch.nextafter(x, torch.tensor(-9e9)), x))
    x[:, 0] = m[:, 0]  # the scale's own value
    x = x.view(1024, 2, 64)
    b = Batch(hip, [1024], [1024], 2, 64, 64)
    hip.kv_q4_append(b.cache, x.cuda(), (-x).cuda(), b.starts_t, b.lens_t)
    ko, vo = (torch.empty((1024, 2, 64), device="cuda") for _ in range(2))
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    assert torch.equal(ko.cpu().double(), held(x)) and torch.equal(vo.cpu().double(), held(-x))


def test_rows_without_a_position_or_page(hip):
    """Positions below zero or past the table, and ids that are no page: not written, read as zeros; rows outside the
    sequences left alone."""
    kv, hd, page = 2, 64, 32
    b = Batch(hip, [4, 4, 4], [2, 66, 10], kv, hd, page, cap=64, fill=0x11)
    pages = b.pages.clone()
    pages[2, 0] = -1
    b.cache.set_pages(pages)
    # starts from 2: rows 0, 1 and the last 3 belong to no sequence
    starts = torch.tensor([2, 6, 10, 14], dtype=torch.int32, device="cuda")
    lens = torch.tensor([2, 66, 10], dtype=torch.int32, device="cuda")
    x = torch.randn((17, kv, hd), generator=torch.Generator().manual_seed(1))
    before = b.data.clone()
    hip.kv_q4_append(b.cache, x.cuda(), x.cuda(), starts, lens)
    ko, vo = (torch.full((17, kv, hd), 7.0, device="cuda") for _ in range(2))
    hip.kv_q4_read(b.cache, ko, vo, starts, lens)
    want = torch.full((17, kv, hd), 7.0, dtype=torch.float64)
    want[2:14] = 0
    want[4:6] = held(x[4:6])    # sequence 0: rows 2, 3 are positions -2, -1
    want[6:8] = held(x[6:8])    # sequence 1: positions 62, 63; 64, 65 are past the table
    assert torch.equal(ko.cpu().double(), want) and torch.equal(vo.cpu().double(), want)
    touched = (b.data != before).view(-1, hip.kv_q4_page_bytes(kv, hd, page)).any(1).nonzero().flatten().tolist()
    assert set(touched) <= {int(b.ids[0, 0]), int(b.ids[1, 1])}
    pages[2, 0] = 1 << 30
    hip.kv_q4_append(b.cache, x.cuda(), x.cuda(), starts, lens)
    hip.kv_q4_read(b.cache, ko, vo, starts, lens)
    assert torch.equal(ko.cpu().double(), want)


@pytest.mark.parametrize("heads_outer", [False, True])
def test_strided_and_unaligned_rows(hip, heads_outer):
    kv, hd, rows = 3, 96, 37
    b = Batch(hip, [rows], [rows + 5], kv, hd, 32)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((rows, kv, hd), generator=g).to(torch.bfloat16)

    def place(t):  # 2 bytes off 16, rows apart by an odd number of elements
        if heads_outer:
            buf = torch.full((1 + kv * (rows * hd + 3),), 9.0, dtype=t.dtype, device="cuda")
            view = buf[1:].as_strided((rows, kv, hd), (hd, rows * hd + 3, 1))
        else:
            buf = torch.full((1 + rows * (kv * hd + 5),), 9.0, dtype=t.dtype, device="cuda")
            view = buf[1:].as_strided((rows, kv, hd), (kv * hd + 5, hd, 1))
        view.copy_(t)
        return buf, view
    _, kc = place(x)
    _, vc = place(-x)
    hip.kv_q4_append(b.cache, kc, vc, b.starts_t, b.lens_t)
    buf, ko = place(torch.zeros_like(x))
    _, vo = place(torch.zeros_like(x))
    edge = buf.clone()
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    assert torch.equal(ko.cpu(), held(x).to(x.dtype)) and torch.equal(vo.cpu(), held(-x).to(x.dtype))
    ko.zero_()
    assert torch.equal(buf, edge)  # nothing between the rows was written


# ----------------------------------------------------------- attention
CASES = [
    # heads, kv, hd, page, rows, lens, window
    (1, 1, 32, 32, [1], [1], 0),
    (4, 1, 64, 64, [1], [33], 0),
    (32, 8, 64, 64, [1, 1], [4096, 1], 0),
    (8, 8, 64, 32, [1, 1, 1], [0, 31, 32], 0),
    (7, 1, 96, 32, [1, 1], [700, 63], 0),
    (14, 2, 96, 96, [1, 1], [1000, 97], 40),
    (6, 2, 128, 128, [1, 3, 0, 2], [129, 300, 50, 2], 0),
    (16, 1, 128, 64, [1, 1], [515, 2000], 0),
    (40, 2, 128, 32, [2], [100], 33),
    (4, 2, 192, 64, [1, 5], [250, 65], 0),
    (8, 1, 256, 64, [1, 4], [400, 4], 0),
    (3, 3, 256, 32, [17], [40], 5),
    (4, 2, 64, 64, [64, 100], [64, 333], 0),
    (2, 2, 128, 32, [200], [200], 0),
    (8, 2, 128, 64, [70, 1, 129], [500, 900, 129], 0),
    (4, 4, 64, 64, [150], [400], 64),
    (4, 1, 96, 32, [90, 33], [91, 40], 1),
    (6, 1, 32, 32, [66, 0, 3], [66, 9, 300], 0),
    (12, 2, 192, 64, [40, 41], [100, 41], 0),
    (4, 1, 256, 64, [65], [129], 0),
    (4, 2, 64, 32, [6, 90], [3, 50], 0),   # rows before the sequence's start
]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page,rows,lens,window", CASES)
def test_attention(hip, name, heads, kv, hd, page, rows, lens, window):
    dt = TYPES[name]
    b = Batch(hip, rows, lens, kv, hd, page)  # 0xFF: what is not written holds NaN scales
    kvs = b.fill(hip)
    g = torch.Generator().manual_seed(hd + heads)
    q = (torch.randn((sum(rows), heads, hd), generator=g) * 2).to(dt)
    qc, out = q.cuda(), torch.full((sum(rows), heads, hd), 5.0, dtype=dt, device="cuda")
    hip.kv_q4_attention(out, qc, b.cache, b.starts_t, b.lens_t, max(rows), hd ** -0.5, window)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5, window)
    check_attention(out, want, mag, top, dt, hd, max(lens))
    again = torch.empty_like(out)
    hip.kv_q4_attention(again, qc, b.cache, b.starts_t, b.lens_t, max(rows), hd ** -0.5, window)
    assert torch.equal(out, again)  # no sum depends on an order that changes


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_peaked_and_large(hip, name, rows):
    """Scores in the hundreds (one token has all the weight), values up to the largest held."""
    dt = TYPES[name]
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [rows], [600], kv, hd, 64)
    kvs = b.fill(hip, scale=30.0)
    q = (torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * 4).to(dt)
    out = torch.empty((rows, heads, hd), dtype=dt, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, [rows], [600], hd ** -0.5)
    check_attention(out, want, mag, top, dt, hd, 600, max(x.abs().max().item() for kv_ in kvs for x in kv_))
    big = Batch(hip, [rows], [600], kv, hd, 64)
    kvs = big.fill(hip, scale=2e4)  # some at the limit
    q = (q.float() * 2.0 ** -12).to(dt)
    hip.kv_q4_attention(out, q.cuda(), big.cache, big.starts_t, big.lens_t)
    want, mag, top = reference(q, kvs, [rows], [600], hd ** -0.5)
    if dt == torch.float32:
        check_attention(out, want, mag, top, dt, hd, 600, max(x.abs().max().item() for kv_ in kvs for x in kv_))


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_attention_queries_of_any_range(hip, rows, scale):
    heads, kv, hd = 4, 2, 64
    b = Batch(hip, [rows], [100], kv, hd, 64)
    kvs = b.fill(hip)
    q = torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * scale
    out = torch.empty((rows, heads, hd), device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, None, 0.125 / scale)
    want, mag, top = reference(q, kvs, [rows], [100], 0.125 / scale)
    check_attention(out, want, mag, top, torch.float32, hd, 100)


@pytest.mark.parametrize("rows,lens", [([1, 1], [300, 40]), ([20, 50], [300, 60])])
def test_attention_nan_and_inf_in_a_query_stay_there(hip, rows, lens):
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, rows, lens, kv, hd, 32)
    kvs = b.fill(hip)
    q = torch.randn((sum(rows), heads, hd), generator=torch.Generator().manual_seed(4))
    bad = q.clone()
    bad[0, 3, 7], bad[sum(rows) - 1, 5, 1] = math.nan, math.inf
    out = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, bad.cuda(), b.cache, b.starts_t, b.lens_t)
    clean = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(clean, q.cuda(), b.cache, b.starts_t, b.lens_t)
    assert torch.isnan(out[0, 3]).all() and torch.isnan(out[-1, 5]).all()
    out[0, 3], out[-1, 5] = clean[0, 3], clean[-1, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("rows", [[1, 1], [70, 45]])
def test_attention_pages_that_are_missing(hip, rows):
    """Ids that are no page are not attended to, wherever they lie; rows whose
    every page is missing are zero; rows of no sequence are left alone."""
    heads, kv, hd, page, lens = 4, 2, 64, 32, [200, 100]
    b = Batch(hip, rows, lens, kv, hd, page)
    kvs = b.fill(hip)
    pages = b.pages.clone()
    pages[0, 1], pages[0, 3], pages[1, :] = -7, 1 << 29, -1
    b.cache.set_pages(pages)
    n = sum(rows)
    q = torch.randn((n + 3, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.full(q.shape, 5.0, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    assert (out[n:] == 5).all() and (out[rows[0]:n] == 0).all()
    keep = torch.tensor([t // page not in (1, 3) for t in range(200)])
    k, v = kvs[0]
    for i in range(rows[0]):
        see = keep.clone()
        see[200 - rows[0] + i + 1:] = False
        s = (k[:, see].repeat_interleave(2, 0) @ q[i].double()[:, :, None])[..., 0] * hd ** -0.5
        w = torch.softmax(s, -1)
        want = (w[:, None] @ v[:, see].repeat_interleave(2, 0))[:, 0]
        assert (out[i].cpu().double() - want).abs().max() < 1e-5  # sums of 200 terms of order one in f32


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (8, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("rows", [[1, 2], [20, 3], [150, 40]])
def test_attention_positions_before_every_window(hip, name, heads, kv, hd, rows):
    """What no row's window reaches may never have been written (NaN scales here),
    also where it shares a group of 32 with what some row sees."""
    dt, page, lens, window = TYPES[name], 64, [307, 117], 45
    b = Batch(hip, rows, lens, kv, hd, page)
    have = [min(n + window - 1, t) for n, t in zip(rows, lens)]  # positions that some row sees
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn((sum(have), kv, hd), generator=g) for _ in range(2))
    hip.kv_q4_append(b.cache, k.cuda(), v.cuda(), *Batch.tensors(have, lens))
    kvs, at = [], 0
    for n, t in zip(have, lens):
        kvs.append([torch.cat([torch.zeros(kv, t - n, hd, dtype=torch.float64), held(x[at:at + n]).transpose(0, 1)], 1)
                    for x in (k, v)])
        at += n
    q = torch.randn((sum(rows), heads, hd), generator=g).to(dt)
    out = torch.empty_like(q, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, max(rows), hd ** -0.5, window)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5, window)
    check_attention(out, want, mag, top, dt, hd, window)


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 1, 20]])
def test_attention_lengths_past_the_table_and_rows_past_the_limit(hip, rows):
    heads, kv, hd, page = 4, 2, 64, 32
    lens = [64, 64, 64]
    b = Batch(hip, rows, lens, kv, hd, page)
    kvs = b.fill(hip)
    n = sum(rows)
    q = torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.full(q.shape, 5.0, device="cuda")
    # sequence 1 claims a length far past its two pages: its row sees all 64
    claim = torch.tensor([64, 5000, 64], dtype=torch.int32, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, claim, min(max(rows), 30))
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    if rows[0] > 30:
        assert (out[30:rows[0]] == 5).all()  # not computed
        out[30:rows[0]] = want[30:rows[0]].float().cuda()
    check_attention(out, want, mag, top, torch.float32, hd, 64)
    negative = torch.tensor([-5, 0, -2 ** 31], dtype=torch.int32, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, negative)
    assert (out == 0).all()


def test_attention_strided_unaligned_queries_and_outputs(hip):
    heads, kv, hd, rows, lens = 6, 2, 96, [3, 30], [50, 77]
    n = sum(rows)
    b = Batch(hip, rows, lens, kv, hd, 32)
    kvs = b.fill(hip)
    q = torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(4)).to(torch.float16)
    qb = torch.zeros(1 + n * (heads * hd + 7), dtype=torch.float16, device="cuda")
    qv = qb[1:].as_strided((n, heads, hd), (heads * hd + 7, hd, 1))
    qv.copy_(q)
    ob = torch.full((3 + heads * (n * hd + 5),), 9.0, dtype=torch.float16, device="cuda")
    ov = ob[3:].as_strided((n, heads, hd), (hd, n * hd + 5, 1))
    hip.kv_q4_attention(ov, qv, b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    check_attention(ov, want, mag, top, torch.float16, hd, 77)
    ov.fill_(9.0)
    assert (ob == 9.0).all()


def test_shared_pages_and_one_sequence_twice(hip):
    """Two sequences over the same pages (a shared prefix) see the same tokens."""
    heads, kv, hd = 4, 2, 64
    b = Batch(hip, [1], [100], kv, hd, 32)
    kvs = b.fill(hip)
    two = b.pages.repeat(2, 1)
    b.cache.set_pages(two)
    s, l = Batch.tensors([1, 1], [100, 60])
    q = torch.randn((2, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, s, l)
    want, mag, top = reference(q, [kvs[0], tuple(x[:, :60] for x in kvs[0])], [1, 1], [100, 60], hd ** -0.5)
    check_attention(out, want, mag, top, torch.float32, hd, 100)


def test_a_cache_past_four_gigabytes(hip):
    """Pages behind 2^32 bytes of the cache."""
    kv, hd, page, heads = 8, 128, 1024, 16
    size = hip.kv_q4_page_bytes(kv, hd, page)
    n_pages = (1 << 32) // size + 40
    data = torch.empty(n_pages * size, dtype=torch.uint8, device="cuda")
    pages = torch.tensor([[n_pages - 1, 0, n_pages - 3]], dtype=torch.int32, device="cuda")
    cache = hip.KvCacheQ4(data, pages, kv, hd, page)
    t = 2500
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((t, kv, hd), generator=g) for _ in range(2))
    s, l = Batch.tensors([t], [t])
    hip.kv_q4_append(cache, k.cuda(), v.cuda(), s, l)
    ko, vo = (torch.empty((t, kv, hd), device="cuda") for _ in range(2))
    hip.kv_q4_read(cache, ko, vo, s, l)
    hk, hv = held(k), held(v)
    assert torch.equal(ko.cpu().double(), hk) and torch.equal(vo.cpu().double(), hv)
    s, l = Batch.tensors([1], [t])
    q = torch.randn((1, heads, hd), generator=g)
    out = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), cache, s, l)
    want, mag, top = reference(q, [(hk.transpose(0, 1), hv.transpose(0, 1))], [1], [t], hd ** -0.5)
    check_attention(out, want, mag, top, torch.float32, hd, t)


@pytest.mark.parametrize("n,kv,heads,most,few", [
    (70, 2, 8, 400, 1),      # more sequences than a wave has lanes
    (300, 1, 1, 130, 1),
    (65, 3, 6, 3000, 1),
    (130, 2, 16, 90, 5),
    (3, 70, 70, 1500, 1),    # more heads than a wave has lanes
    (2, 66, 132, 2100, 9),
])
def test_attention_of_many_sequences_and_heads(hip, n, kv, heads, most, few):
    """Ragged batches over tables of different spare room: lengths of zero, one
    and the table's, sequences without rows."""
    r = np.random.RandomState(n)
    lens = r.randint(0, most + 1, n)
    lens[r.randint(0, n, 2)] = most
    lens[n // 2], lens[n - 1] = 0, 1
    rows = r.randint(0, few + 1, n) if few > 1 else np.where(r.rand(n) < 0.2, 0, 1)
    rows[0] = few
    for cap in (most, 4 * most):
        b = Batch(hip, rows.tolist(), lens.tolist(), kv, 32, 32, cap=cap, seed=n)
        kvs = b.fill(hip)
        q = torch.randn((int(rows.sum()), heads, 32), generator=torch.Generator().manual_seed(n))
        for window in (0, 50):
            out = torch.full(q.shape, 5.0, device="cuda")
            hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, few, 0.2, window)
            want, mag, top = reference(q, kvs, rows.tolist(), lens.tolist(), 0.2, window)
            check_attention(out, want, mag, top, torch.float32, 32, most)


@pytest.mark.parametrize("n,rows_of", [(70, lambda r, n: r.randint(0, 40, n)), (200, lambda r, n: r.randint(5, 15, n)),
                                       (200, lambda r, n: np.where(r.rand(n) < 0.3, 0, 1))])
def test_rows_of_many_sequences_written_and_read_back(hip, n, rows_of):
    r = np.random.RandomState(n)
    rows = rows_of(r, n)
    lens = rows + r.randint(0, 100, n)
    b = Batch(hip, rows.tolist(), lens.tolist(), 3, 32, 64, seed=n)
    x = torch.randn((int(rows.sum()), 6, 32), generator=torch.Generator().manual_seed(n)).cuda()
    hip.kv_q4_append(b.cache, x[:, :3], x[:, 3:], b.starts_t, b.lens_t)
    ko, vo = (torch.full((x.shape[0], 3, 32), 9.0, device="cuda") for _ in range(2))
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    assert torch.equal(ko.cpu().double(), held(x[:, :3])) and torch.equal(vo.cpu().double(), held(x[:, 3:]))


@pytest.mark.parametrize("rows", [1, 3, 30, 60])
def test_attention_negative_and_zero_scales(hip, rows):
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [rows], [1500], kv, hd, 64)
    kvs = b.fill(hip)
    q = torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.empty(q.shape, device="cuda")
    for scale in (-0.3, 0.0, 1e-38):
        hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, rows, scale)
        want, mag, top = reference(q, kvs, [rows], [1500], scale)
        check_attention(out, want, mag, top, torch.float32, hd, 1500)


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 16), (128, 1, 8), (256, 1, 4)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_attention_of_every_form(hip, name, hd, kv, heads):
    """Row counts on both sides of each form's limits, over a table of 40 groups
    and a window that starts inside one."""
    dt = TYPES[name]
    g = heads // kv
    for pairs in (16, 24, 64, 72, 128, 136, 256, 520):
        rows = -(-pairs // g)
        b = Batch(hip, [rows, 1], [1280, 700], kv, hd, 32)
        kvs = b.fill(hip)
        q = torch.randn((rows + 1, heads, hd), generator=torch.Generator().manual_seed(pairs)).to(dt)
        for window in (0, 333):
            out = torch.empty(q.shape, dtype=dt, device="cuda")
            hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, rows, None, window)
            want, mag, top = reference(q, kvs, [rows, 1], [1280, 700], hd ** -0.5, window)
            check_attention(out, want, mag, top, dt, hd, 1280)


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_attention_rows_of_many_heads(hip, name):
    """Enough heads for the largest workgroups of 16-bit types; the second tile
    of a head has a few rows only."""
    dt = TYPES[name]
    heads, kv, hd, rows, lens = 64, 64, 128, [260] + [1] * 7, [300] + [33] * 7
    b = Batch(hip, rows, lens, kv, hd, 64)
    kvs = b.fill(hip)
    q = torch.randn((sum(rows), heads, hd), generator=torch.Generator().manual_seed(4)).to(dt)
    out = torch.empty(q.shape, dtype=dt, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, 260)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    check_attention(out, want, mag, top, dt, hd, 300)


# ------------------------------------------------------- as they are used
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_prompts_in_passes_then_single_tokens(hip, name):
    """A batch whose prompts arrive in ragged passes, then steps of one token
    each: every call's outputs against attention over all tokens so far."""
    dt = TYPES[name]
    heads, kv, hd, page = 8, 2, 64, 32
    b = Batch(hip, [0, 0, 0], [200, 200, 200], kv, hd, page)
    g = torch.Generator().manual_seed(9)
    toks = [[(torch.empty((kv, 0, hd), dtype=torch.float64),) * 2][0] for _ in range(3)]
    lens = [0, 0, 0]
    for rows in ([50, 0, 33], [31, 7, 60], [1, 64, 1]) + ([1, 1, 1],) * 4:
        lens = [a + r for a, r in zip(lens, rows)]
        s, l = Batch.tensors(rows, lens)
        n = sum(rows)
        qkv = torch.randn((n, heads + 2 * kv, hd), generator=g).to(dt)
        x = qkv.cuda()
        hip.kv_q4_append(b.cache, x[:, heads:heads + kv], x[:, heads + kv:], s, l)
        out = torch.empty((n, heads, hd), dtype=dt, device="cuda")
        hip.kv_q4_attention(out, x[:, :heads], b.cache, s, l, max(rows))
        at = 0
        for i, r in enumerate(rows):
            kk, vv = (held(qkv[at:at + r, o:o + kv]).transpose(0, 1) for o in (heads, heads + kv))
            toks[i] = (torch.cat([toks[i][0], kk], 1), torch.cat([toks[i][1], vv], 1))
            at += r
        want, mag, top = reference(qkv[:, :heads], toks, rows, lens, hd ** -0.5)
        check_attention(out, want, mag, top, dt, hd, max(lens))
    # and the whole of it read back
    s, l = Batch.tensors(lens, lens)
    ko, vo = (torch.empty((sum(lens), kv, hd), device="cuda") for _ in range(2))
    hip.kv_q4_read(b.cache, ko, vo, s, l)
    assert torch.equal(ko.cpu().double(), torch.cat([t[0] for t in toks], 1).transpose(0, 1))
    assert torch.equal(vo.cpu().double(), torch.cat([t[1] for t in toks], 1).transpose(0, 1))


def test_captured_steps_follow_their_lengths(hip):
    """Append and attention captured once, replayed with new rows, lengths and
    pages; two graphs with workspaces of their own, replayed in turn and with
    eager calls between."""
    heads, kv, hd, page = 8, 2, 64, 32
    b = Batch(hip, [1, 1], [300, 300], kv, hd, page)
    kvs = b.fill(hip)
    g = torch.Generator().manual_seed(9)
    starts, lens = Batch.tensors([1, 1], [100, 200])
    graphs = []
    for _ in range(2):
        qkv = torch.randn((2, heads + 2 * kv, hd), generator=g).cuda()
        out = torch.empty((2, heads, hd), device="cuda")
        need = hip.lib().mivi_hip_kv_q4_attention_workspace(2, 2, 1, heads, kv, hd, b.pages.shape[1] * page, 0)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")

        def step():
            hip.kv_q4_append(b.cache, qkv[:, heads:heads + kv], qkv[:, heads + kv:], starts, lens)
            hip.kv_q4_attention(out, qkv[:, :heads], b.cache, starts, lens, 1, workspace=ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, qkv, out))
    kvs = [tuple(x.clone() for x in kv_) for kv_ in b.fill(hip)]
    for turn in range(4):
        for graph, qkv, out in graphs:
            now = [57 + 60 * turn, 1 + turn]
            lens.copy_(torch.tensor(now, dtype=torch.int32))
            qkv.copy_(torch.randn(qkv.shape, generator=g))
            graph.replay()
            for i, t in enumerate(now):
                kvs[i][0][:, t - 1] = held(qkv[i, heads:heads + kv])
                kvs[i][1][:, t - 1] = held(qkv[i, heads + kv:])
            want, mag, top = reference(qkv[:, :heads], [tuple(x[:, :t] for x in kv_) for kv_, t in zip(kvs, now)], [1, 1],
                                       now, hd ** -0.5)
            check_attention(out, want, mag, top, torch.float32, hd, 300)
            eager = torch.empty_like(out)
            hip.kv_q4_attention(eager, qkv[:, :heads], b.cache, starts, lens, 1)
            assert torch.equal(out, eager)


def test_two_streams_at_once(hip):
    """Calls on streams of their own, over caches of their own: the default workspace is each stream's."""
    heads, kv, hd = 8, 2, 128
    jobs = []
    for i in range(2):
        b = Batch(hip, [1] * 3, [900, 500, 77], kv, hd, 64, seed=i)
        kvs = b.fill(hip, seed=i)
        q = torch.randn((3, heads, hd), generator=torch.Generator().manual_seed(i))
        jobs.append((b, q, q.cuda(), torch.empty((3, heads, hd), device="cuda"), torch.cuda.Stream(),
                     reference(q, kvs, b.rows, b.lens, hd ** -0.5)))
    torch.cuda.synchronize()
    for turn in range(8):
        for b, _, qc, out, stream, _ in jobs:
            # one by a stream's object, one by its handle
            hip.kv_q4_attention(out, qc, b.cache, b.starts_t, b.lens_t, 1,
                                stream=stream if turn % 2 else stream.cuda_stream)
    torch.cuda.synchronize()
    for b, q, _, out, _, (want, mag, top) in jobs:
        check_attention(out, want, mag, top, torch.float32, hd, 900)


def test_python_refusals(hip):
    b = Batch(hip, [1], [10], 2, 64, 32)
    x = torch.zeros((1, 2, 64), device="cuda")
    q = torch.zeros((1, 4, 64), device="cuda")
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x, x.half(), b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x[..., ::2], x[..., ::2], b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x, x[:, :1], b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x.double(), x.double(), b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x, x, b.starts_t.long(), b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x, x, b.starts_t, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        hip.kv_q4_append(b.cache, x.cpu(), x.cpu(), b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_attention(q[:, :3], q, b.cache, b.starts_t, b.lens_t)
    with pytest.raises(hip.QuantError):
        hip.kv_q4_attention(q[:, :3].contiguous(), q[:, :3].contiguous(), b.cache, b.starts_t, b.lens_t)
    with pytest.raises(ValueError):
        hip.kv_q4_attention(q, q, b.cache, b.starts_t, b.lens_t, window=-1)
    with pytest.raises(ValueError):
        b.cache.set_pages(b.pages.long())
    with pytest.raises(hip.QuantError):
        hip.kv_q4_read(b.cache, x.expand(3, 2, 64), x.expand(3, 2, 64), b.starts_t, b.lens_t)
    assert hip.kv_q4_attention(torch.empty((0, 4, 64), device="cuda"), torch.empty((0, 4, 64), device="cuda"), b.cache,
                               b.starts_t, b.lens_t).shape[0] == 0


def test_a_batch_of_no_sequences(hip):
    b = Batch(hip, [1], [10], 2, 64, 32)
    b.cache.set_pages(torch.empty((0, 4), dtype=torch.int32, device="cuda"))
    starts, lens = Batch.tensors([], [])
    for rows in (0, 3):  # rows of no sequence are left alone
        x = torch.full((rows, 2, 64), 5.0, device="cuda")
        before = b.data.clone()
        hip.kv_q4_append(b.cache, x, x, starts, lens)
        hip.kv_q4_read(b.cache, x, torch.empty_like(x), starts, lens)
        out = torch.full((rows, 4, 64), 5.0, device="cuda")
        hip.kv_q4_attention(out, torch.zeros_like(out), b.cache, starts, lens)
        assert torch.equal(b.data, before) and (x == 5).all() and (out == 5).all()
