"""The step's calls validate on the host before anything is launched (CPU only:
no device pointer is dereferenced)."""
from __future__ import annotations

import math

import pytest
import torch

import mivi_hip

LIB = mivi_hip.lib()
A = 1 << 20  # an aligned address that nothing reads
HUGE = 1 << 60


def t4(p=A, n=HUGE, row=256, head=64):
    return [p, n, row, head]


def norm(typ=0, out=None, x=None, r=None, s=None, w=A, w_len=64, eps=1e-5, rows=3, heads=2, dim=64):
    return LIB.mivi_hip_rms_norm(typ, *(out or t4(2 * A)), *(x or t4()), *(r or t4(None)), *(s or t4(None)), w, w_len, eps,
                                 rows, heads, dim, None)


def norm_q8(typ=0, codes=A, codes_len=HUGE, scales=A, scales_len=HUGE, group=32, x=None, r=None, s=None, w=A, w_len=256,
            eps=1e-5, rows=3, dim=256):
    return LIB.mivi_hip_rms_norm_q8(typ, codes, codes_len, scales, scales_len, group, *(x or t4())[:3],
                                    *(r or t4(None))[:3], *(s or t4(None))[:3], w, w_len, eps, rows, dim, None)


def rope(typ=0, qo=None, q=None, heads=2, ko=None, k=None, kv=1, rows=3, hd=64, rot=64, half=0, freqs=A, freqs_len=32,
         scale=1.0, pos=A, pos_len=3, starts=None, lens=None, n_seq=0):
    return LIB.mivi_hip_rope(typ, *(qo or t4(2 * A)), *(q or t4()), heads, *(ko or t4(4 * A)), *(k or t4(3 * A)), kv, rows,
                             hd, rot, half, freqs, freqs_len, scale, pos, pos_len, starts, lens, n_seq, None)


def pack(codes=A, codes_len=HUGE, st=1, scales=A, scales_len=HUGE, zeros=None, zeros_len=0, packed=A, packed_len=HUGE, n=20,
         d=256, group=64):
    return LIB.mivi_hip_w4_pack(codes, codes_len, st, scales, scales_len, zeros, zeros_len, packed, packed_len, n, d,
                                group, None)


def w4(typ=0, out=A, out_len=HUGE, out_row=20, packed=A, packed_len=HUGE, st=1, zeros=0, x=A, x_len=HUGE, x_row=256,
       batch=3, n=20, d=256, group=64):
    return LIB.mivi_hip_w4_matmul_rows(typ, out, out_len, out_row, packed, packed_len, st, zeros, x, x_len, x_row, batch,
                                       n, d, group, None)


def w4_q8(typ=0, out=A, out_len=HUGE, out_row=20, packed=A, packed_len=HUGE, st=1, zeros=0, x=A, x_len=HUGE, xs=A,
          xs_len=HUGE, xg=128, batch=3, n=20, d=256, group=64):
    return LIB.mivi_hip_w4_matmul_rows_q8(typ, out, out_len, out_row, packed, packed_len, st, zeros, x, x_len, xs, xs_len,
                                          xg, batch, n, d, group, None)


def verify(tokens=A, tokens_len=7, counts=A, counts_len=2, p=A, p_len=HUGE, p_row=100, q=A, q_len=HUGE, q_row=100,
           drafted=A, drafted_len=7, accept=A, accept_len=7, pick=A, pick_len=2, starts=A, n_seq=2, rows=7, n=100, ws=A,
           ws_len=HUGE):
    return LIB.mivi_hip_verify_rows(tokens, tokens_len, counts, counts_len, p, p_len, p_row, q, q_len, q_row, drafted,
                                    drafted_len, accept, accept_len, pick, pick_len, starts, n_seq, rows, n, ws, ws_len,
                                    None)


@pytest.mark.parametrize("call", [norm, norm_q8, rope, w4, w4_q8])
def test_types(call):
    for t in (2, 8, 12, 14, -1):
        assert call(typ=t) == 1 and mivi_hip.last_error().type_id == t & 0xFFFFFFFF


def test_norm_refusals():
    assert norm(dim=0) == 101 and norm(heads=0) == 101
    for eps in (0.0, -1e-5, 1e-31, math.inf, math.nan):
        assert norm(eps=eps) == 101 and norm_q8(eps=eps) == 101, eps
    assert norm(w=None) == 101 and norm(w=A + 2) == 101
    assert norm(w_len=63) == 2 and mivi_hip.last_error().expected == 64
    need = 2 * 256 + 64 + 64
    for name in ("x", "out", "r", "s"):
        p = 2 * A if name == "out" else A if name == "x" else 5 * A
        assert norm(**{name: t4(p, need - 1)}) == 2 and mivi_hip.last_error().expected == need, name
        assert norm(**{name: t4(p + 2, need)}) == 101, name
    assert norm(x=t4(None)) == 101 and norm(out=t4(None)) == 101
    assert norm(out=t4(2 * A, HUGE, 128, 32)) == 101      # heads inside one another
    assert norm(s=t4(5 * A, HUGE, 100, 64)) == 101        # rows inside one another
    assert norm(rows=1 << 30, heads=4) == 4 and norm(dim=1 << 31) == 4
    assert norm(x=[A, HUGE, 1 << 62, 64]) == 4
    assert norm(rows=0) == 0


def test_norm_in_place():
    """Over itself a tensor has its own strides; out and the sum are two tensors."""
    assert norm(out=t4(A, HUGE, 512, 64)) == 101
    assert norm(s=t4(A, HUGE, 256, 128), out=t4(2 * A)) == 101
    assert norm(r=t4(5 * A), s=t4(5 * A, HUGE, 512, 64)) == 101
    assert norm(s=t4(2 * A), out=t4(2 * A)) == 101
    assert norm_q8(r=t4(5 * A), s=t4(5 * A, HUGE, 512)) == 101


def test_norm_q8_refusals():
    for group in (1, 16, 48, 96, 1024):
        assert norm_q8(group=group) == 101, group
    assert norm_q8(group=512) == 3 and mivi_hip.last_error().block_size == 512
    assert norm_q8(codes=None) == 101 and norm_q8(scales=None) == 101 and norm_q8(scales=A + 2) == 101
    assert norm_q8(codes_len=3 * 256 - 1) == 2 and norm_q8(scales_len=3 * 8 - 1) == 2
    assert norm_q8(group=0, scales_len=2) == 2 and mivi_hip.last_error().expected == 3
    assert norm_q8(rows=1 << 31) == 4 and norm_q8(rows=0) == 0


def test_rope_refusals():
    assert rope(heads=0, kv=0) == 101 and rope(heads=65536) == 101
    assert rope(hd=0, rot=0) == 101 and rope(hd=513) == 101
    assert rope(rot=63) == 3 and mivi_hip.last_error().block_size == 2
    assert rope(rot=0) == 101 and rope(rot=66, freqs_len=33) == 101
    assert rope(freqs=None) == 101 and rope(freqs=A + 4) == 101 and rope(freqs_len=31) == 2
    assert rope(pos=None) == 101
    assert rope(pos=None, starts=A, n_seq=1) == 101 and rope(pos=None, lens=A, n_seq=1) == 101
    assert rope(pos=None, starts=A, lens=None, n_seq=1) == 101
    assert rope(starts=A, lens=A, n_seq=1) == 101                  # both
    assert rope(pos=A + 2) == 101 and rope(pos_len=2) == 2
    assert rope(pos=None, starts=A + 2, lens=A, n_seq=1) == 101
    for name in ("q", "qo", "k", "ko"):
        n = 2 * 256 + (64 if name[0] == "q" else 0) + 64
        p = dict(q=A, qo=2 * A, k=3 * A, ko=4 * A)[name]
        assert rope(**{name: t4(p, n - 1)}) == 2 and mivi_hip.last_error().expected == n, name
        assert rope(**{name: t4(None)}) == 101, name
        assert rope(**{name: t4(p + 1)}) == 101, name
    assert rope(qo=t4(2 * A, HUGE, 64, 64)) == 101
    assert rope(qo=t4(A, HUGE, 512, 64)) == 101                    # in place with other strides
    assert rope(qo=t4(4 * A)) == 101                               # q and k to one place
    assert rope(rows=1 << 31) == 4 and rope(pos=None, starts=A, lens=A, n_seq=1 << 31) == 4
    assert rope(rows=0) == 0 and rope(pos=None, starts=A, lens=None, n_seq=0) == 0
    assert rope(rows=1 << 30, heads=65535, q=t4(A, HUGE, 1 << 23), qo=t4(2 * A, HUGE, 1 << 23), pos_len=1 << 30) == 4


def test_frequencies():
    f = LIB.mivi_hip_rope_frequencies
    out = torch.empty(32, dtype=torch.float64)
    ok = [0, 1e4, 1.0, 4096, 64, out.data_ptr(), 32]
    assert f(*ok) == 0
    for i, bad, rc in ((0, 5, 101), (0, -1, 101), (1, 1.0, 101), (1, math.inf, 101), (1, math.nan, 101), (2, 0.0, 101),
                       (2, math.inf, 101), (4, 63, 3), (4, 0, 3), (5, None, 101), (6, 31, 2)):
        args = list(ok)
        args[i] = bad
        assert f(*args) == rc, (i, bad)
    for kind in (3, 4):
        assert f(kind, 1e4, 2.0, 0, 64, out.data_ptr(), 32) == 101
    plain = mivi_hip.rope_frequencies(64, 1e6, device="cpu")
    assert torch.allclose(plain, 1e6 ** -(torch.arange(32, dtype=torch.float64) / 32), rtol=1e-13, atol=0)
    # a factor of one or less changes nothing; the fast end stays, the slow end is divided
    for kind in ("linear", "base", "yarn", "model"):
        assert torch.equal(mivi_hip.rope_frequencies(64, 1e6, kind, 1.0, device="cpu"), plain), kind
    for kind in ("yarn", "model"):
        g = mivi_hip.rope_frequencies(64, 1e6, kind, 8.0, 4096, device="cpu")
        assert float(g[0]) == 1.0 and abs(float(g[-1] * 8 / plain[-1]) - 1) < 1e-12
        assert bool((g[:-1] > g[1:]).all())
    base = mivi_hip.rope_frequencies(64, 1e6, "base", 8.0, device="cpu")
    assert abs(float(base[-1] * 8 / plain[-1]) - 1) < 1e-12 and float(base[0]) == 1.0


def test_model_frequencies_are_the_models():
    """rope.rs:50-122 with model.rs:194-206, as the model handles form them in f32."""
    dim, base, scale = 64, 1e6, 31.25
    f = mivi_hip.rope_frequencies(dim, base, "model", scale, 4096, device="cpu")
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        ramp = min(max((2 * math.pi / plain - 128) / (4096 - 128), 0), 1)
        assert abs(float(f[i]) / ((1 - ramp) * plain + ramp * plain / scale) - 1) < 1e-12


def test_w4_sizes():
    size = LIB.mivi_hip_w4_packed_size
    # tiles of 16 rows and steps of 128 columns: 1024 bytes of codes, 32 of scales and
    # 16 of zeros a unit
    assert size(20, 256, 64, 0) == 2 * 2 * (1024 + 64) and size(20, 256, 64, 1) == 2 * 2 * (1024 + 96)
    assert size(16, 96, 32, 0) == 1024 + 128 and size(1, 160, 160, 0) == 2 * (1024 + 32)
    for n, d, g in ((0, 256, 64), (16, 0, 64), (16, 250, 50), (16, 256, 0), (16, 256, 96), (16, 256, 192), (16, 320, 128),
                    (1 << 31, 256, 64), (16, 1 << 40, 64)):
        assert size(n, d, g, 0) == 0, (n, d, g)
    # workgroups have up to 16 tiles: indexes of rows behind the last stay within 32 bits
    assert size((1 << 31) - 1024, 32, 32, 0) == ((1 << 27) - 64) * (1024 + 128) and size((1 << 31) - 1023, 32, 32, 0) == 0


@pytest.mark.parametrize("call", [pack, w4, w4_q8])
def test_w4_geometry_refusals(call):
    assert call(n=0) == 101
    assert call(d=0) in (101, 3)
    assert call(d=272, group=272) == 3 and call(group=48) == 101 and call(group=0) == 101
    assert call(d=320, group=128) == 3
    assert call(st=0) == 1 and call(st=12) == 1
    n = LIB.mivi_hip_w4_packed_size(20, 256, 64, 0)
    assert call(packed_len=n - 1) == 2 and mivi_hip.last_error().expected == n
    assert call(packed=None) == 101 and call(packed=A + 8) == 101
    assert call(n=1 << 31, **({} if call is pack else dict(out_row=1 << 31))) == 4


def test_pack_refusals():
    assert pack(codes=None) == 101 and pack(scales=None) == 101 and pack(scales=A + 1) == 101
    assert pack(codes_len=20 * 128 - 1) == 2 and pack(scales_len=79) == 2
    assert pack(zeros=A, zeros_len=79) == 2


def test_w4_refusals():
    assert w4(x=None) == 101 and w4(x=A + 2) == 101 and w4(out=None) == 101 and w4(out=A + 2) == 101
    assert w4(x_len=2 * 256 + 255) == 2 and w4(out_len=2 * 20 + 19) == 2
    assert w4(out_row=19) == 101
    assert w4(batch=1 << 31, x_row=256) == 4
    assert w4(batch=0) == 0 and w4_q8(batch=0) == 0
    assert w4_q8(x=None) == 101 and w4_q8(xs=None) == 101 and w4_q8(xs=A + 2) == 101
    assert w4_q8(x_len=3 * 256 - 1) == 2 and w4_q8(xs_len=5) == 2 and w4_q8(xg=0, xs_len=2) == 2
    for xg in (1, 16, 48, 1024):
        assert w4_q8(xg=xg) == 101, xg
    assert w4_q8(xg=512) == 3


def test_verify_refusals():
    assert verify(n=0) == 101
    for name in ("tokens", "counts", "p", "drafted", "accept", "pick", "starts"):
        assert verify(**{name: None}) == 101, name
        assert verify(**{name: A + 2}) == 101, name
    assert verify(q=A + 2) == 101
    for name, need in (("tokens", 7), ("counts", 2), ("drafted", 7), ("accept", 7), ("pick", 2), ("p", 700), ("q", 700)):
        assert verify(**{name + "_len": need - 1}) == 2 and mivi_hip.last_error().expected == need, name
    need = LIB.mivi_hip_verify_rows_workspace(100, 2)
    assert need == 2 * (16 + 4) and verify(ws_len=need - 1) == 2 and mivi_hip.last_error().expected == need
    assert verify(ws=None) == 101 and verify(ws=A + 8) == 101
    assert verify(n=1 << 31) == 4 and verify(rows=1 << 31) == 4 and verify(n_seq=65536) == 4
    assert verify(n=1 << 30, n_seq=65535, p_row=1 << 30, q_row=1 << 30, counts_len=65535, pick_len=65535) == 4
    assert verify(n_seq=0) == 0
    assert LIB.mivi_hip_verify_rows_workspace(1 << 40, 2) == 0 and LIB.mivi_hip_verify_rows_workspace(100, 65536) == 0


def test_python_refusals_on_host_tensors():
    x, w = torch.zeros(2, 64), torch.ones(64)
    with pytest.raises(ValueError):
        mivi_hip.rms_norm(torch.empty_like(x), x, w)
    with pytest.raises(ValueError):
        mivi_hip.rope(x.view(2, 1, 64), None, torch.ones(32, dtype=torch.float64),
                      positions=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        mivi_hip.rope(None, None, torch.ones(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        mivi_hip.W4Weights(torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 1), dtype=torch.float16))
    with pytest.raises(ValueError):
        mivi_hip.verify_rows(*(torch.zeros(1) for _ in range(2)), torch.zeros(1, 5), *(torch.zeros(1) for _ in range(3)),
                             torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        mivi_hip.rope_frequencies(64, kind="none", device="cpu")
