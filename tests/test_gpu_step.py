"""The step's operators together, as a host that drives its own layers uses them:
a layer over the 4-bit cache, then verification of drafted tokens; eager, captured
and replayed, on streams, next to each other."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu

KV, HEADS, HD, DIM, VOCAB, PAGE, GROUP = 2, 6, 64, 512, 1000, 64, 128


def w4(hip, n, d, seed):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, generator=g), (torch.rand((n, d // GROUP), generator=g) * 0.01 + 0.001).half(),
         torch.randint(5, 11, (n, d // GROUP), dtype=torch.uint8, generator=g))
    return t, hip.W4Weights(*(x.cuda() for x in t))


class Layer:
    """Weights, cache and every buffer of a step of ragged rows; `step` makes the
    calls, on the buffers alone."""

    def __init__(self, hip, rows, lens, dt=torch.bfloat16, seed=0):
        self.hip, self.rows, self.dt = hip, list(rows), dt
        g = torch.Generator().manual_seed(seed)
        self.g = g
        n, seqs = sum(rows), len(rows)
        self.wqkv, self.qkv_w = w4(hip, (HEADS + 2 * KV) * HD, DIM, 1)
        self.wo, self.o_w = w4(hip, DIM, HEADS * HD, 2)
        self.whead, self.head_w = w4(hip, VOCAB, DIM, 3)
        self.norms = [(1 + 0.1 * torch.randn(d, generator=g)).cuda() for d in (DIM, HD, HD, DIM)]
        self.freqs = hip.rope_frequencies(HD, 1e6, "yarn", 8.0, 4096)
        per = -(-max(lens) // PAGE) + 2
        self.data = torch.zeros(seqs * per * hip.kv_q4_page_bytes(KV, HD, PAGE), dtype=torch.uint8, device="cuda")
        self.cache = hip.KvCacheQ4(self.data, torch.randperm(seqs * per, generator=g).to(torch.int32).view(seqs, per).cuda(),
                                   KV, HD, PAGE)
        self.starts = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        old = [t - r for r, t in zip(rows, lens)]
        if sum(old):
            k, v = (torch.randn((sum(old), KV, HD), generator=g).to(dt).cuda() for _ in range(2))
            hip.kv_q4_append(self.cache, k, v, torch.from_numpy(np.concatenate([[0], np.cumsum(old)]).astype(np.int32)).cuda(),
                             torch.tensor(old, dtype=torch.int32, device="cuda"))
        e = lambda *s, t=dt: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        self.x, self.residual, self.stream_in = e(n, DIM), e(n, DIM), e(n, DIM)
        self.codes, self.scales = e(n, DIM, t=torch.int8), e(n, DIM // GROUP, t=torch.float32)
        self.qkv, self.attended, self.delta, self.normed = e(n, HEADS + 2 * KV, HD), e(n, HEADS, HD), e(n, DIM), e(n, DIM)
        self.logits = e(n, VOCAB, t=torch.float32)
        self.normed32 = e(n, DIM, t=torch.float32)
        self.draft = torch.empty_like(self.logits)
        self.drafted, self.accept, self.pick = e(n, t=torch.int32), e(n, t=torch.float32), e(seqs, t=torch.float32)
        self.tokens, self.counts = e(n, t=torch.int32), e(seqs, t=torch.int32)
        self.workspace = e(hip.lib().mivi_hip_verify_rows_workspace(VOCAB, seqs), t=torch.uint8)
        need = hip.lib().mivi_hip_kv_q4_attention_workspace(seqs, n, max(rows), HEADS, KV, HD, per * PAGE, 0)
        self.attn_ws = e(max(need, 16), t=torch.uint8)
        self.inputs(seed)

    def inputs(self, seed):
        g = torch.Generator().manual_seed(seed + 100)
        n = self.x.shape[0]
        self.x.copy_(torch.randn((n, DIM), generator=g))
        self.stream_in.copy_(torch.randn((n, DIM), generator=g))
        self.draft.copy_(torch.softmax(3 * torch.randn((n, VOCAB), generator=g), -1))
        self.drafted.copy_(torch.multinomial(self.draft.cpu(), 1, generator=g)[:, 0])
        self.accept.copy_(torch.rand(n, generator=g) * 0.1)
        self.pick.copy_(torch.rand(len(self.rows), generator=g))

    def step(self):
        h = self.hip
        self.residual.copy_(self.stream_in)
        h.rms_norm_q8(self.codes, self.scales, self.x, self.norms[0], residual=self.residual, residual_out=self.residual)
        h.w4_matmul_rows(self.qkv.view(self.qkv.shape[0], -1), self.qkv_w, self.codes, self.scales)
        q, k, v = self.qkv[:, :HEADS], self.qkv[:, HEADS:HEADS + KV], self.qkv[:, HEADS + KV:]
        h.rms_norm(q, q, self.norms[1])
        h.rms_norm(k, k, self.norms[2])
        h.rope(q, k, self.freqs, starts=self.starts, lens=self.lens, scale=1.2)
        h.kv_q4_append(self.cache, k, v, self.starts, self.lens)
        h.kv_q4_attention(self.attended, q, self.cache, self.starts, self.lens, max(self.rows), workspace=self.attn_ws)
        h.w4_matmul_rows(self.delta, self.o_w, self.attended.view(self.attended.shape[0], -1))
        h.rms_norm(self.normed, self.delta, self.norms[3], residual=self.residual, residual_out=self.residual)
        self.normed32.copy_(self.normed)
        h.w4_matmul_rows(self.logits, self.head_w, self.normed32)
        torch.softmax(self.logits, -1, out=self.logits)
        h.verify_rows(self.tokens, self.counts, self.logits, self.drafted, self.accept, self.pick, self.starts,
                      draft=self.draft, workspace=self.workspace)

    OUTS = ("residual", "codes", "scales", "qkv", "attended", "delta", "normed", "logits", "tokens", "counts", "data")

    def outs(self):
        torch.cuda.synchronize()
        return {k: getattr(self, k).clone() for k in self.OUTS}


def positions(layer):
    return torch.cat([torch.arange(t - r, t) for r, t in zip(layer.rows, layer.lens.tolist())])


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [1, 300, 64]), ([5, 1, 3, 5], [5, 200, 65, 1000]), ([70, 2], [70, 90])])
def test_each_call_of_a_step(hip, rows, lens, dt):
    """Every call against 64 bits on what the call before left."""
    L = Layer(hip, rows, lens, dt)
    n = sum(rows)
    want_c, want_s = ref.norm_q8(L.x, L.norms[0], 1e-5, GROUP, L.stream_in)
    L.step()
    assert torch.equal(L.codes.cpu().double(), want_c)
    assert bool(((ref.f64(L.scales) - want_s).abs() <= want_s * ref.U * 1.0001).all())
    # the projection again, for q and k before their norms
    wide = ref.f64(L.codes) * ref.f64(L.scales).repeat_interleave(GROUP, 1)
    qkv = torch.empty((n, (HEADS + 2 * KV) * HD), dtype=dt, device="cuda")
    hip.w4_matmul_rows(qkv, L.qkv_w, L.codes, L.scales)
    assert ref.w4_close(qkv, wide, L.wqkv)
    qkv = qkv.view(n, -1, HD)
    assert torch.equal(qkv[:, HEADS + KV:], L.qkv[:, HEADS + KV:])
    for at, w in ((slice(0, HEADS), L.norms[1]), (slice(HEADS, HEADS + KV), L.norms[2])):
        turned = torch.empty_like(qkv[:, at])
        hip.rms_norm(turned, qkv[:, at], w)
        assert ref.norm_close(turned, ref.norm(qkv[:, at], w, 1e-5)[1])
        assert ref.rope_close(L.qkv[:, at], *ref.rope(turned, positions(L), L.freqs.cpu(), False, float(np.float32(1.2))))
    assert ref.w4_close(L.delta, ref.f64(L.attended).view(n, -1), L.wo)
    before = torch.empty_like(L.residual)
    hip.rms_norm_q8(torch.empty_like(L.codes), torch.empty_like(L.scales), L.x, L.norms[0], residual=L.stream_in,
                    residual_out=before)
    want_sum, want = ref.norm(L.delta, L.norms[3], 1e-5, before)
    assert ref.norm_close(L.normed, want) and ref.sum_close(L.residual, want_sum)
    tokens, counts = ref.verify(L.logits, L.drafted.cpu(), L.accept.cpu(), L.pick.cpu(), L.starts.cpu(), L.draft)
    assert L.tokens.tolist() == tokens.tolist() and L.counts.tolist() == counts.tolist()


@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [100, 300, 64]), ([5, 1, 3, 5], [5, 200, 65, 1000])])
def test_captured_step(hip, rows, lens):
    """Replays follow the buffers: other inputs, then longer sequences."""
    L, E = Layer(hip, rows, lens), Layer(hip, rows, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.step()
    for i in range(4):
        for x in (L, E):
            x.inputs(i)
            if i:
                x.lens += 1  # a token more: the rows' positions move on
        graph.replay()
        E.step()
        a, b = L.outs(), E.outs()
        for k in a:
            assert torch.equal(a[k], b[k]), (i, k)


def test_two_steps_at_once(hip):
    """On two streams, each with its own buffers, as alone."""
    kinds = (([5, 1, 3, 5], [5, 200, 65, 1000]), ([1] * 6, [7, 90, 1, 64, 128, 300]))
    alone = []
    for i, (r, t) in enumerate(kinds):
        L = Layer(hip, r, t, seed=i)
        L.step()
        alone.append(L.outs())
    layers = [Layer(hip, r, t, seed=i) for i, (r, t) in enumerate(kinds)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(5):
        for L, s in zip(layers, streams):
            with torch.cuda.stream(s):
                L.step()
    for L, want in zip(layers, alone):
        for k, v in L.outs().items():
            assert torch.equal(v, want[k]), k


def test_streams_and_handles(hip):
    """A stream object, its handle, and the null stream's 0; a default workspace
    is taken from the given stream's memory."""
    g = torch.Generator().manual_seed(3)
    p = torch.softmax(torch.randn((6, 5000), generator=g), -1).cuda()
    q = torch.softmax(torch.randn((6, 5000), generator=g), -1).cuda()
    t = torch.randint(0, 5000, (6,), generator=g, dtype=torch.int32).cuda()
    u, pick, starts = torch.rand(6, generator=g).cuda(), torch.rand(2, generator=g).cuda(), torch.tensor([0, 4, 6], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (None, side, side.cuda_stream, 0):
        tokens, counts = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        hip.verify_rows(tokens, counts, p, t, u, pick, starts, draft=q, stream=s)
        torch.cuda.synchronize()
        got.append((tokens.tolist(), counts.tolist()))
    assert all(x == got[0] for x in got)
    w = w4(hip, 64, 256, 5)
    x = torch.randn((3, 256), generator=g).cuda()
    want = torch.empty((3, 64), device="cuda")
    hip.w4_matmul_rows(want, w[1], x)
    for s in (side, side.cuda_stream):
        torch.cuda.synchronize()
        packed = hip.W4Weights(*(v.cuda() for v in w[0]))
        torch.cuda.synchronize()
        out = torch.zeros_like(want)
        torch.cuda.synchronize()
        hip.w4_matmul_rows(out, packed, x, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_same_bits_from_the_same_call(hip):
    L = Layer(hip, [5, 1, 3, 5], [5, 200, 65, 1000])
    L.step()
    a = L.outs()
    L.step()
    b = L.outs()
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_refused_tensors(hip):
    x = torch.randn((4, 2, 64), device="cuda")
    w, f = torch.ones(64, device="cuda"), hip.rope_frequencies(64)
    pos, starts = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    one = torch.tensor([9], dtype=torch.int32, device="cuda")
    q8 = torch.empty((4, 64), dtype=torch.int8, device="cuda")
    sc = torch.empty((4, 2), device="cuda")
    wt = w4(hip, 32, 128, 1)[1]
    xb = torch.randn((4, 128), device="cuda")
    bad = [
        lambda: hip.rms_norm(x.half(), x, w), lambda: hip.rms_norm(x[:3], x, w), lambda: hip.rms_norm(x, x, w[:63]),
        lambda: hip.rms_norm(x, x, w.double()), lambda: hip.rms_norm(x, x, w.cpu()), lambda: hip.rms_norm(x, x, None),
        lambda: hip.rms_norm(x.double(), x.double(), w), lambda: hip.rms_norm(x.transpose(0, 2), x.transpose(0, 2), w),
        lambda: hip.rms_norm(x, x, w, residual=x[:, :1]), lambda: hip.rms_norm(x[0, 0], x[0, 0], w),
        lambda: hip.rms_norm_q8(q8, sc, x[:, 0].cpu(), w), lambda: hip.rms_norm_q8(q8.float(), sc, x[:, 0], w),
        lambda: hip.rms_norm_q8(q8, sc[:3], x[:, 0], w), lambda: hip.rms_norm_q8(q8[:, :32], sc, x[:, 0], w),
        lambda: hip.rope(x, x[:3], f, positions=pos), lambda: hip.rope(x, x.half(), f, positions=pos),
        lambda: hip.rope(x, None, f.float(), positions=pos), lambda: hip.rope(x, None, f),
        lambda: hip.rope(x, None, f, positions=pos, starts=starts, lens=one), lambda: hip.rope(x, None, f, starts=starts),
        lambda: hip.rope(x, None, f, positions=pos.long()), lambda: hip.rope(x, None, f, positions=pos[:3]),
        lambda: hip.rope(x, None, f, starts=starts, lens=pos), lambda: hip.rope(x[:, 0], None, f, positions=pos),
        lambda: hip.rope(x, None, f, positions=pos, q_out=x.half()), lambda: hip.rope(x, None, f, starts=starts[:0], lens=one),
        lambda: hip.w4_matmul_rows(torch.empty((4, 32), device="cuda"), wt, xb[:, :64]),
        lambda: hip.w4_matmul_rows(torch.empty((4, 31), device="cuda"), wt, xb),
        lambda: hip.w4_matmul_rows(torch.empty((3, 32), device="cuda"), wt, xb),
        lambda: hip.w4_matmul_rows(torch.empty((4, 32), device="cuda").half(), wt, xb),
        lambda: hip.w4_matmul_rows(torch.empty((4, 32), device="cuda"), wt, xb, sc),
        lambda: hip.w4_matmul_rows(torch.empty((4, 32)), wt, xb),
        lambda: hip.verify_rows(pos, one, xb, pos, xb[:, 0].contiguous(), xb[0, :1], starts, draft=xb[:, :64]),
        lambda: hip.verify_rows(pos, one, xb, pos[:3], xb[:, 0].contiguous(), xb[0, :1], starts),
        lambda: hip.verify_rows(pos, one, xb.half(), pos, xb[:, 0].contiguous(), xb[0, :1], starts),
        lambda: hip.verify_rows(pos, one, xb, pos, xb[:, 0], xb[0, :1], starts),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(hip.QuantError):  # 34 columns
        hip.W4Weights(torch.zeros((4, 17), dtype=torch.uint8, device="cuda"),
                      torch.ones((4, 1), dtype=torch.float16, device="cuda"))
