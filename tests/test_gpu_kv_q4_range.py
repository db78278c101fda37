"""Attention over the 4-bit cache at the ends of what its arguments can hold:
scores far past fp32's integers, scales next to the largest float, values at
the cache's limit; and how near 16-bit outputs come to their own rounding."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_kv_q4 import TYPES, Batch, check_attention, held, reference

pytestmark = pytest.mark.gpu


def check_hull(got, q, kvs, rows, lens, scale, dtype, longest):
    """For scores whose f32 rounding is larger than one: softmax weighs a row's
    tokens by scores that are off by at most e = sum |q k| scale * ((hd + 8)
    2^-24 and 2^-22 for f32 queries in two planes), so that a token more than
    2 e + 40 below the largest has less than e^-40 of its weight, which fp16
    weights hold as zero, and the output lies between the least and the largest
    value of the tokens that are left, up to the f32 sums (one in four of the
    tokens and 64 more roundings) and half a step of the type. With one token
    left this is its value."""
    q = q.double().cpu()
    hd = q.shape[-1]
    assert torch.isfinite(got).all()
    got = got.double().cpu()
    at, alone = 0, 0
    for (k, v), n, t in zip(kvs, rows, lens):
        g = q.shape[1] // k.shape[0]
        for i in range(n):
            kk, vv = (x[:, :t - n + i + 1].repeat_interleave(g, 0) for x in (k, v))
            s = (kk @ q[at + i][:, :, None])[..., 0] * scale
            top = (kk.abs() @ q[at + i].abs()[:, :, None])[..., 0].amax(-1, keepdim=True) * abs(scale)
            e = top * ((hd + 8) * 2.0 ** -24 + (2.0 ** -22 if dtype == torch.float32 else 0.0))
            left = s >= s.amax(-1, keepdim=True) - 2 * e - 40
            alone += (left.sum(-1) == 1).sum().item()
            lo = torch.where(left[..., None], vv, math.inf).amin(1)
            hi = torch.where(left[..., None], vv, -math.inf).amax(1)
            room = (torch.maximum(lo.abs(), hi.abs()) * ((longest / 4 + 64) * 2.0 ** -24 + torch.finfo(dtype).eps / 2)
                    + torch.finfo(dtype).tiny)
            assert (got[at + i] >= lo - room).all() and (got[at + i] <= hi + room).all()
        at += n
    return alone


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("cap", [600, 4096])   # one part, and shares with a join
@pytest.mark.parametrize("name,by,kscale", [
    ("f32", 3e7, 1.0), ("f32", 1e9, 1.0), ("f32", 1e20, 1.0), ("f32", 1e36, 1.0),
    ("bf16", 1e8, 1.0), ("bf16", 1e36, 1.0), ("f16", 1.5e4, 2e4),
])
def test_attention_of_scores_past_the_integers_of_fp32(hip, name, by, kscale, cap, rows):
    """Finite queries give finite outputs, of the tokens with the largest scores."""
    dt = TYPES[name]
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [rows], [600], kv, hd, 64, cap=cap)
    kvs = b.fill(hip, scale=kscale)
    q = (torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * by).clamp(-3e38, 3e38)
    q = (q.clamp(-65504, 65504) if dt == torch.float16 else q).to(dt)
    out = torch.empty((rows, heads, hd), dtype=dt, device="cuda")
    for scale in (hd ** -0.5, -0.125):
        hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, rows, scale)
        alone = check_hull(out, q, kvs, [rows], [600], scale, dt, 600)
        assert alone > rows * heads / 2  # most rows have one token only


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_large_scores_leaves_the_other_rows_alone(hip, rows):
    """Rows beside one of very large scores are as exact as ever."""
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [rows], [600], kv, hd, 64)
    kvs = b.fill(hip)
    q = torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4))
    far = q.clone()
    far[0, 1] *= 1e9
    out = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, far.cuda(), b.cache, b.starts_t, b.lens_t)
    assert torch.isfinite(out).all()
    want, mag, top = reference(q, kvs, [rows], [600], hd ** -0.5)
    out[0, 1] = want[0, 1].float()
    check_attention(out, want, mag, top, torch.float32, hd, 600)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("scale,by", [(3.4e38, 1e-38), (3.4e38, 1e-39), (-3e38, 2e-38), (2.5e38, 1e-20), (3.4e38, 1.0),
                                      (1e30, 1e30), (3.4e38, 0.0)])
def test_attention_of_scales_next_to_the_largest_float(hip, rows, scale, by):
    """scale log2(e) passes the largest float, and scale q k does."""
    heads, kv, hd = 4, 2, 64
    b = Batch(hip, [rows], [100], kv, hd, 64)
    kvs = b.fill(hip)
    q = (torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * by).clamp(-3e38, 3e38)
    out = torch.empty((rows, heads, hd), device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t, rows, scale)
    if abs(scale) * by < 100:
        want, mag, top = reference(q, kvs, [rows], [100], float(np.float32(scale)))
        check_attention(out, want, mag, top, torch.float32, hd, 100)
    else:
        check_hull(out, q, kvs, [rows], [100], float(np.float32(scale)), torch.float32, 100)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [600, 4096])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_values_at_the_limit(hip, name, rows, cap):
    """Values up to 21760, in every type: the bounds of check_attention."""
    dt = TYPES[name]
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [rows], [600], kv, hd, 64, cap=cap)
    kvs = b.fill(hip, scale=2e4)  # some at the limit
    q = (torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * 2.0 ** -10).to(dt)
    out = torch.empty((rows, heads, hd), dtype=dt, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, [rows], [600], hd ** -0.5)
    check_attention(out, want, mag, top, dt, hd, 600, max(x.abs().max().item() for kv_ in kvs for x in kv_))


@pytest.mark.parametrize("heads,kv,hd,rows,length,by", [
    (28, 4, 96, 1, 4097, 0.3), (8, 2, 64, 6, 100, 0.3), (8, 2, 128, 1, 8192, 0.3), (16, 2, 128, 70, 400, 0.3),
    (8, 2, 64, 40, 300, 0.0), (4, 2, 256, 9, 500, 0.3), (2, 1, 192, 60, 500, 1.0), (4, 4, 32, 120, 300, 0.3),
])
def test_fp16_outputs_are_as_near_as_their_rounding(hip, heads, kv, hd, rows, length, by):
    """Nearly uniform weights, whose outputs are small beside the values: the
    error is that of rounding the exact output. Before that rounding an output
    is off by less than 2^-20 of the values' mean magnitude (weights to 22 bits
    and the f32 sums), under a third of a rounding's rms here; in quadrature 6 %."""
    b = Batch(hip, [rows], [length], kv, hd, 64)
    kvs = b.fill(hip)
    q = (torch.randn((rows, heads, hd), generator=torch.Generator().manual_seed(4)) * by).half()
    out = torch.empty((rows, heads, hd), dtype=torch.float16, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, [rows], [length], hd ** -0.5)
    rms = lambda x: x.square().mean().sqrt().item()  # noqa: E731
    got, best = rms(out.cpu().double() - want), rms(want.half().double() - want)
    print(heads, kv, hd, rows, length, got / best)
    assert got <= 1.1 * best


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_queries_of_wide_range(hip, name, rows):
    """Dimensions of one query far apart: the large ones meet keys of zero, so
    that the small ones decide. A query is held to 2^-39 of its row's largest
    magnitude (half of fp16's smallest step beside 2^14), two planes or one."""
    dt = TYPES[name]
    heads, kv, hd, length = 4, 2, 64, 100
    b = Batch(hip, [rows], [length], kv, hd, 64)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn((length, kv, hd), generator=g), torch.randn((length, kv, hd), generator=g)
    k[..., :32] = 0.0
    s, l = Batch.tensors([length], [length])
    hip.kv_q4_append(b.cache, k.cuda(), v.cuda(), s, l)
    kvs = [(held(k).transpose(0, 1), held(v).transpose(0, 1))]
    q = torch.randn((rows, heads, hd), generator=g)
    far = 2.0 ** 12 if dt == torch.float16 else 2.0 ** 24
    q[..., :32] *= far
    q = q.to(dt)
    out = torch.empty((rows, heads, hd), dtype=dt, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, [rows], [length], hd ** -0.5)
    # what the queries lack, times the keys
    most = q.double().abs().amax(-1)
    lack = most * 2.0 ** -39 * hd * kvs[0][0].abs().amax().item() * hd ** -0.5
    check_attention(out, want, mag, top + lack / 2.0 ** -22, dt, hd, length)


@pytest.mark.parametrize("rows", [[1, 1], [20, 50], [300, 2]])
def test_a_table_without_pages(hip, rows):
    """No row has a position: nothing is written, rows read and attend as zeros."""
    heads, kv, hd = 4, 2, 64
    b = Batch(hip, rows, [400, 400], kv, hd, 64)
    b.cache.set_pages(torch.empty((2, 0), dtype=torch.int32, device="cuda"))
    n = sum(rows)
    x = torch.randn((n, kv, hd), device="cuda")
    before = b.data.clone()
    hip.kv_q4_append(b.cache, x, x, b.starts_t, b.lens_t)
    assert torch.equal(b.data, before)
    ko, vo = torch.full_like(x, 5.0), torch.full_like(x, 5.0)
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    assert (ko == 0).all() and (vo == 0).all()
    q = torch.randn((n, heads, hd), device="cuda")
    out = torch.full_like(q, 5.0)
    hip.kv_q4_attention(out, q, b.cache, b.starts_t, b.lens_t, max(rows))
    assert (out == 0).all()


@pytest.mark.parametrize("rows", [[1, 1], [9, 3]])
def test_rows_more_than_two_billion_elements_apart(hip, rows):
    """Offsets past 32 bits, in elements and in bytes, in every tensor."""
    heads, kv, hd, lens = 4, 2, 64, [1500, 700]
    n = sum(rows)
    b = Batch(hip, rows, lens, kv, hd, 64)
    kvs = [tuple(x.clone() for x in kv_) for kv_ in b.fill(hip, dtype=torch.bfloat16)]
    apart = 2 ** 31 // (n - 1) + 64
    buf = torch.empty((n - 1) * apart + 3 * heads * hd, dtype=torch.bfloat16, device="cuda")

    def view(first, h):
        return buf[first * hd:].as_strided((n, h, hd), (apart, hd, 1))
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn((n, h, hd), generator=g).to(torch.bfloat16) for h in (heads, kv, kv))
    view(0, heads).copy_(q), view(heads, kv).copy_(k), view(heads + kv, kv).copy_(v)
    hip.kv_q4_append(b.cache, view(heads, kv), view(heads + kv, kv), b.starts_t, b.lens_t)
    ko, vo = view(heads + 2 * kv, kv), view(heads + 3 * kv, kv)
    hip.kv_q4_read(b.cache, ko, vo, b.starts_t, b.lens_t)
    assert torch.equal(ko.cpu(), held(k).to(ko.dtype)) and torch.equal(vo.cpu(), held(v).to(vo.dtype))
    out = view(2 * heads, heads)
    hip.kv_q4_attention(out, view(0, heads), b.cache, b.starts_t, b.lens_t, max(rows))
    at = 0
    for i, (r, t) in enumerate(zip(rows, lens)):
        kvs[i][0][:, t - r:t], kvs[i][1][:, t - r:t] = (held(x[at:at + r]).transpose(0, 1) for x in (k, v))
        at += r
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    check_attention(out.contiguous(), want, mag, top, torch.bfloat16, hd, max(lens))
