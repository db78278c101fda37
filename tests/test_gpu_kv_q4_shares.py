"""Attention over the 4-bit cache where its work is cut into shares and joined
(tables past 32 groups): the uses that a workspace, the cut or the join could
break. Every test asserts that its call needs a workspace."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_kv_q4 import TYPES, Batch, check_attention, held, reference

pytestmark = pytest.mark.gpu


def need_of(hip, b, rows, heads, max_rows=None, window=0):
    n = sum(rows)
    need = hip.lib().mivi_hip_kv_q4_attention_workspace(
        len(rows), n, n if max_rows is None else max_rows, heads, b.kv, b.hd, b.cache.pages.shape[1] * b.page, window)
    assert need > 0
    return need


FORMS = [[1, 1], [5, 3], [30, 2], [70, 45]]  # one tile of 16 pairs, of 64, two of 64, three of 128 (4 heads over 2)


@pytest.mark.parametrize("rows", FORMS)
def test_pages_that_are_missing_over_whole_shares(hip, rows):
    heads, kv, hd, page, lens = 4, 2, 64, 32, [4000, 2100]
    b = Batch(hip, rows, lens, kv, hd, page, cap=4096)
    need_of(hip, b, rows, heads)
    kvs = b.fill(hip)
    pages = b.pages.clone()
    pages[0, 10:70], pages[0, 100:], pages[1, :] = -7, 1 << 29, -1
    b.cache.set_pages(pages)
    n = sum(rows)
    q = torch.randn((n + 3, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.full(q.shape, 5.0, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, b.lens_t)
    assert (out[n:] == 5).all() and (out[rows[0]:n] == 0).all()
    keep = torch.tensor([t // page < 10 or 70 <= t // page < 100 for t in range(4000)])
    kept = [tuple(x[:, keep] for x in kvs[0])]
    length = int(keep.sum())
    for i in range(rows[0]):  # all rows are past the last page that is there
        want, mag, top = reference(q[i:i + 1], kept, [1], [length], hd ** -0.5)
        check_attention(out[i:i + 1], want, mag, top, torch.float32, hd, 4000)


@pytest.mark.parametrize("rows", FORMS)
def test_nan_and_inf_in_a_query_stay_there_over_shares(hip, rows):
    heads, kv, hd, lens = 4, 2, 64, [4000, 77]
    b = Batch(hip, rows, lens, kv, hd, 32, cap=4096)
    need_of(hip, b, rows, heads)
    b.fill(hip)
    q = torch.randn((sum(rows), heads, hd), generator=torch.Generator().manual_seed(4))
    bad = q.clone()
    bad[0, 3, 7], bad[sum(rows) - 1, 1, 1], bad[0, 0, 2] = math.nan, math.inf, -math.inf
    out, clean = torch.empty(q.shape, device="cuda"), torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, bad.cuda(), b.cache, b.starts_t, b.lens_t)
    hip.kv_q4_attention(clean, q.cuda(), b.cache, b.starts_t, b.lens_t)
    assert torch.isnan(out[0, 3]).all() and torch.isnan(out[-1, 1]).all() and torch.isnan(out[0, 0]).all()
    out[0, 3], out[-1, 1], out[0, 0] = clean[0, 3], clean[-1, 1], clean[0, 0]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("rows", [[3, 30], [1, 2]])
@pytest.mark.parametrize("hd", [32, 96, 192, 256])
def test_strided_unaligned_queries_and_outputs_of_a_join(hip, hd, rows):
    heads, kv, lens = 6, 2, [1900, 77]
    n = sum(rows)
    b = Batch(hip, rows, lens, kv, hd, 32, cap=2048)
    need_of(hip, b, rows, heads)
    kvs = b.fill(hip)
    q = torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(4)).to(torch.float16)
    qb = torch.zeros(1 + n * (heads * hd + 7), dtype=torch.float16, device="cuda")
    qv = qb[1:].as_strided((n, heads, hd), (heads * hd + 7, hd, 1))
    qv.copy_(q)
    ob = torch.full((3 + heads * (n * hd + 5),), 9.0, dtype=torch.float16, device="cuda")
    ov = ob[3:].as_strided((n, heads, hd), (hd, n * hd + 5, 1))
    hip.kv_q4_attention(ov, qv, b.cache, b.starts_t, b.lens_t)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    check_attention(ov, want, mag, top, torch.float16, hd, 1900)
    ov.fill_(9.0)
    assert (ob == 9.0).all()


@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 1, 2], [40, 1, 20], [90, 1, 20]])
def test_lengths_past_the_table_and_rows_past_the_limit_of_a_join(hip, rows):
    heads, kv, hd, page, limit = 4, 2, 64, 32, 30
    lens = [2048, 2048, 2048]
    b = Batch(hip, rows, lens, kv, hd, page)
    kvs = b.fill(hip)
    n, most = sum(rows), min(max(rows), limit)
    need_of(hip, b, rows, heads, most)
    q = torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(4))
    out = torch.full(q.shape, 5.0, device="cuda")
    # sequence 1 claims a length far past its table: its row sees all of it
    claim = torch.tensor([2048, 5000, 2048], dtype=torch.int32, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, claim, most)
    want, mag, top = reference(q, kvs, rows, lens, hd ** -0.5)
    if rows[0] > limit:
        assert (out[limit:rows[0]] == 5).all()  # not computed, not joined
        out[limit:rows[0]] = want[limit:rows[0]].float().cuda()
    check_attention(out, want, mag, top, torch.float32, hd, 2048)
    negative = torch.tensor([-5, 0, -2 ** 31], dtype=torch.int32, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, b.starts_t, negative)
    assert (out == 0).all()


def test_shared_pages_over_shares(hip):
    """A shared prefix, and one sequence twice, in one batch."""
    heads, kv, hd = 4, 2, 64
    b = Batch(hip, [1], [3000], kv, hd, 32)
    kvs = b.fill(hip)
    b.cache.set_pages(b.pages.repeat(3, 1))
    lens = [3000, 1700, 3000]
    s, l = Batch.tensors([1, 2, 1], lens)
    need_of(hip, b, [1, 2, 1], heads, 2)
    q = torch.randn((4, heads, hd), generator=torch.Generator().manual_seed(4))
    q[3] = q[0]
    out = torch.empty(q.shape, device="cuda")
    hip.kv_q4_attention(out, q.cuda(), b.cache, s, l, 2)
    want, mag, top = reference(q, [tuple(x[:, :t] for x in kvs[0]) for t in lens], [1, 2, 1], lens, hd ** -0.5)
    check_attention(out, want, mag, top, torch.float32, hd, 3000)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_prompts_in_passes_then_single_tokens_under_a_long_table(hip, name):
    """As a server runs: a table for the largest context, prompts in ragged
    passes, then single tokens, every call's outputs against all tokens so far."""
    dt = TYPES[name]
    heads, kv, hd, page = 8, 2, 64, 32
    b = Batch(hip, [0, 0, 0], [4096, 4096, 4096], kv, hd, page)
    g = torch.Generator().manual_seed(9)
    toks = [(torch.empty((kv, 0, hd), dtype=torch.float64),) * 2 for _ in range(3)]
    lens = [0, 0, 0]
    for rows in ([900, 0, 33], [31, 7, 60], [1, 1500, 1]) + ([1, 1, 1],) * 4:
        lens = [a + r for a, r in zip(lens, rows)]
        s, l = Batch.tensors(rows, lens)
        n = sum(rows)
        need_of(hip, b, rows, heads, max(rows))
        qkv = torch.randn((n, heads + 2 * kv, hd), generator=g).to(dt)
        x = qkv.cuda()
        hip.kv_q4_append(b.cache, x[:, heads:heads + kv], x[:, heads + kv:], s, l)
        out = torch.empty((n, heads, hd), dtype=dt, device="cuda")
        hip.kv_q4_attention(out, x[:, :heads], b.cache, s, l, max(rows))
        at, checked = 0, []
        for i, r in enumerate(rows):
            kk, vv = (held(qkv[at:at + r, o:o + kv]).transpose(0, 1) for o in (heads, heads + kv))
            toks[i] = (torch.cat([toks[i][0], kk], 1), torch.cat([toks[i][1], vv], 1))
            for j in sorted({0, r // 2, r - 1}) if r else ():  # first, middle and last row of each
                checked.append((i, j, at + j))
            at += r
        for i, j, row in checked:
            t = lens[i] - rows[i] + j + 1
            want, mag, top = reference(qkv[row:row + 1, :heads], [tuple(x[:, :t] for x in toks[i])], [1], [t], hd ** -0.5)
            check_attention(out[row:row + 1], want, mag, top, dt, hd, t)


@pytest.mark.parametrize("rows", [[1, 1], [5, 5], [70, 70]])
def test_captured_steps_follow_their_lengths_over_shares(hip, rows):
    """Append and attention captured once, replayed with rows and lengths that
    change the cut; two graphs with workspaces of their own, replayed in turn
    and with eager calls between."""
    heads, kv, hd, page = 8, 2, 64, 32
    n = sum(rows)
    b = Batch(hip, rows, [4096, 4096], kv, hd, page)
    g = torch.Generator().manual_seed(9)
    starts, lens = Batch.tensors(rows, [100, 200])
    need = need_of(hip, b, rows, heads, max(rows))
    graphs = []
    for _ in range(2):
        qkv = torch.randn((n, heads + 2 * kv, hd), generator=g).cuda()
        out = torch.empty((n, heads, hd), device="cuda")
        ws = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")

        def step():
            hip.kv_q4_append(b.cache, qkv[:, heads:heads + kv], qkv[:, heads + kv:], starts, lens)
            hip.kv_q4_attention(out, qkv[:, :heads], b.cache, starts, lens, max(rows), workspace=ws[:need])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, qkv, out, ws))
    kvs = [tuple(x.clone() for x in kv_) for kv_ in b.fill(hip)]
    for turn, (long, short) in enumerate(((4096, 90), (2000, 2000), (80, 4096), (3000, 1100))):
        for graph, qkv, out, ws in graphs:
            now = [long - turn, short]
            lens.copy_(torch.tensor(now, dtype=torch.int32))
            qkv.copy_(torch.randn(qkv.shape, generator=g))
            graph.replay()
            at = 0
            for i, (r, t) in enumerate(zip(rows, now)):
                for z, o in enumerate((heads, heads + kv)):
                    kvs[i][z][:, t - r:t] = held(qkv[at:at + r, o:o + kv]).transpose(0, 1)
                at += r
            for row, i, t in ((0, 0, now[0] - rows[0] + 1), (n - 1, 1, now[1])):
                want, mag, top = reference(qkv[row:row + 1, :heads], [tuple(x[:, :t] for x in kvs[i])], [1], [t], hd ** -0.5)
                check_attention(out[row:row + 1], want, mag, top, torch.float32, hd, 4096)
            eager = torch.empty_like(out)
            hip.kv_q4_attention(eager, qkv[:, :heads], b.cache, starts, lens, max(rows))
            assert torch.equal(out, eager)
            assert (ws[need:] == 0xAB).all()


@pytest.mark.parametrize("rows", [1, 6])
def test_two_streams_at_once_with_workspaces(hip, rows):
    """Calls on streams of their own, over caches of their own: the default
    workspace is each stream's."""
    heads, kv, hd = 8, 2, 128
    jobs = []
    for i in range(2):
        b = Batch(hip, [rows] * 3, [4000, 500, 77], kv, hd, 64, cap=4096, seed=i)
        need_of(hip, b, b.rows, heads, rows)
        kvs = b.fill(hip, seed=i)
        q = torch.randn((3 * rows, heads, hd), generator=torch.Generator().manual_seed(i))
        jobs.append((b, q.cuda(), [torch.empty(q.shape, device="cuda") for _ in range(8)], torch.cuda.Stream(),
                     reference(q, kvs, b.rows, b.lens, hd ** -0.5)))
    torch.cuda.synchronize()
    for turn in range(8):
        for b, qc, outs, stream, _ in jobs:
            # one by a stream's object, one by its handle
            hip.kv_q4_attention(outs[turn], qc, b.cache, b.starts_t, b.lens_t, rows,
                                stream=stream if turn % 2 else stream.cuda_stream)
    torch.cuda.synchronize()
    for b, q, outs, _, (want, mag, top) in jobs:
        check_attention(outs[0], want, mag, top, torch.float32, hd, 4000)
        for out in outs[1:]:
            assert torch.equal(out, outs[0])


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,rows,lens", [
    (32, 8, 128, [1] * 9, [1, 8192, 700, 4001, 63, 2900, 5555, 33, 8000]),
    (28, 4, 96, [5, 1, 3], [6000, 33, 8192]),
    (8, 2, 128, [300], [4096]),
])
def test_the_same_call_gives_the_same_bits(hip, name, heads, kv, hd, rows, lens):
    """No sum's order changes between calls, whatever ran before."""
    dt = TYPES[name]
    b = Batch(hip, rows, lens, kv, hd, 64, cap=8192)
    b.fill(hip)
    q = torch.randn((sum(rows), heads, hd), generator=torch.Generator().manual_seed(4)).to(dt).cuda()
    outs = []
    for _ in range(4):
        ws = torch.full((max(1, hip.lib().mivi_hip_kv_q4_attention_workspace(
            len(rows), sum(rows), max(rows), heads, kv, hd, 8192, 0)),), np.random.randint(256), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        hip.kv_q4_attention(out, q, b.cache, b.starts_t, b.lens_t, max(rows), workspace=ws)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


def test_the_default_workspace_of_the_null_stream(hip, monkeypatch):
    """stream=0 is the device's default stream: the workspace comes from its
    memory, which nothing else reuses ahead of the work."""
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [1], [3000], kv, hd, 64)
    need_of(hip, b, [1], heads)
    kvs = b.fill(hip)
    q = torch.randn((1, heads, hd), generator=torch.Generator().manual_seed(4))
    qc, out = q.cuda(), torch.empty(q.shape, device="cuda")
    seen, empty = [], torch.empty

    def record(*args, **kw):
        seen.append(torch.cuda.current_stream().cuda_stream)
        return empty(*args, **kw)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        monkeypatch.setattr(torch, "empty", record)
        hip.kv_q4_attention(out, qc, b.cache, b.starts_t, b.lens_t, 1, stream=0)
        monkeypatch.undo()
    torch.cuda.synchronize()
    assert seen == [0]
    want, mag, top = reference(q, kvs, [1], [3000], hd ** -0.5)
    check_attention(out, want, mag, top, torch.float32, hd, 3000)


def test_captured_steps_on_their_default_workspaces(hip):
    """Two captured steps that name no workspace, replayed in turn with eager
    work and other allocations between."""
    heads, kv, hd = 8, 2, 64
    b = Batch(hip, [1, 2], [4096, 2000], kv, hd, 64)
    need_of(hip, b, [1, 2], heads, 2)
    kvs = b.fill(hip)
    gen = torch.Generator().manual_seed(4)
    jobs = []
    for _ in range(2):
        q = torch.randn((3, heads, hd), generator=gen).cuda()
        out = torch.empty(q.shape, device="cuda")
        hip.kv_q4_attention(out, q, b.cache, b.starts_t, b.lens_t, 2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.kv_q4_attention(out, q, b.cache, b.starts_t, b.lens_t, 2)
        jobs.append((graph, q, out))
    for _ in range(4):
        for graph, q, out in jobs:
            q.copy_(torch.randn(q.shape, generator=gen))
            out.fill_(9.0)
            graph.replay()
            torch.full((1 << 20,), 7.0, device="cuda")
            eager = torch.empty_like(out)
            hip.kv_q4_attention(eager, q, b.cache, b.starts_t, b.lens_t, 2)
            assert torch.equal(out, eager)
    _, q, out = jobs[0]
    want, mag, top = reference(q, kvs, [1, 2], [4096, 2000], hd ** -0.5)
    check_attention(out, want, mag, top, torch.float32, hd, 4096)
