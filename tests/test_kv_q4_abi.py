"""The 4-bit cache's calls validate on the host before anything is launched
(CPU only: no device pointer is dereferenced)."""
from __future__ import annotations

import pytest
import torch

import mivi_hip

LIB = mivi_hip.lib()
A = 1 << 20  # an aligned address that nothing reads


def geometry(cache=A, cache_len=None, kv=2, hd=64, page=64, pages=A, pstride=4, per=4, nseq=3, starts=A, lens=A):
    n = mivi_hip.kv_q4_page_bytes(kv, hd, page)
    return [cache, 5 * n if cache_len is None else cache_len, kv, hd, page, pages, pstride, per, nseq, starts, lens]


def rows_args(kv=2, hd=64, rows=7, typ=0, p=A, n=None, rs=None, hs=None):
    rs, hs = kv * hd if rs is None else rs, hd if hs is None else hs
    n = (rows - 1) * rs + (kv - 1) * hs + hd if n is None else n
    return [p, n, rs, hs]


def kv_call(fn, geo=None, k=None, v=None, typ=0, rows=7):
    return fn(*(geo or geometry()), typ, *(k or rows_args()), *(v or rows_args()), rows, None)


def attn(geo=None, out=None, q=None, typ=0, rows=7, max_rows=7, heads=4, window=0, ws=A, ws_bytes=1 << 40,
         scale=0.125):
    return LIB.mivi_hip_kv_q4_attention(typ, *(out or rows_args(kv=4)), *(q or rows_args(kv=4)), rows, max_rows, heads,
                                        scale, window, *(geo or geometry()), ws, ws_bytes, None)


CALLS = [lambda **k: kv_call(LIB.mivi_hip_kv_q4_append, **k), lambda **k: kv_call(LIB.mivi_hip_kv_q4_read, **k), attn]


def test_page_bytes():
    # 32 tokens of one head: K and V codes 16 hd bytes each, scales 2 hd each
    for kv, hd, page in ((1, 32, 32), (8, 64, 64), (3, 96, 96), (2, 256, 1024)):
        assert mivi_hip.kv_q4_page_bytes(kv, hd, page) == kv * page // 32 * 36 * hd
    for kv, hd, page in ((0, 64, 64), (8, 48, 64), (8, 160, 64), (8, 64, 0), (8, 64, 48), (8, 64, 2048)):
        assert mivi_hip.kv_q4_page_bytes(kv, hd, page) == 0


@pytest.mark.parametrize("call", CALLS)
def test_geometry_refusals(call):
    assert call(geo=geometry(hd=48)) == 3 and mivi_hip.last_error().block_size == 32
    assert call(geo=geometry(hd=160)) == 116
    assert call(geo=geometry(page=48)) == 3 and mivi_hip.last_error().dim == 48
    assert call(geo=geometry(page=0)) == 101
    assert call(geo=geometry(page=2048)) == 101
    assert call(geo=geometry(kv=0)) == 101
    n = mivi_hip.kv_q4_page_bytes(2, 64, 64)
    assert call(geo=geometry(cache_len=n - 1)) == 2 and mivi_hip.last_error().expected == n
    for name in ("cache", "pages", "starts", "lens"):
        assert call(geo=geometry(**{name: None})) == 101, name
    assert call(geo=geometry(cache=A + 8)) == 101
    for name in ("pages", "starts", "lens"):
        assert call(geo=geometry(**{name: A + 2})) == 101, name
    assert call(geo=geometry(pstride=3)) == 101
    assert call(geo=geometry(per=1 << 31, pstride=1 << 31)) == 4
    assert call(geo=geometry(per=1 << 26, pstride=1 << 26)) == 4  # positions past 31 bits
    assert call(geo=geometry(nseq=1 << 31)) == 4
    assert call(rows=1 << 31) == 4


@pytest.mark.parametrize("call", CALLS)
def test_type_refusals(call):
    for t in (2, 8, 12, 14):
        assert call(typ=t) == 1 and mivi_hip.last_error().type_id == t


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("call", CALLS[:2])
def test_row_refusals(call, which):
    full = rows_args()
    assert call(**{which: [A, full[1] - 1] + full[2:]}) == 2 and mivi_hip.last_error().expected == full[1]
    assert call(**{which: [None] + full[1:]}) == 101
    assert call(**{which: [A + 2] + full[1:]}) == 101
    assert call(**{which: [A, 1 << 62, 1 << 62, 64]}) == 4


def test_written_rows_may_not_overlap():
    read = CALLS[1]
    assert read(k=rows_args(rs=64, hs=64)) == 101       # rows inside one another
    assert read(k=rows_args(rs=128, hs=32)) == 101      # heads inside one another
    assert read(k=rows_args(rs=0)) == 101
    assert attn(out=rows_args(kv=4, rs=128)) == 101


def test_attention_refusals():
    assert attn(heads=5) == 101 and attn(heads=0) == 101
    for scale in (float("inf"), float("-inf"), float("nan")):
        assert attn(scale=scale) == 101
    full = rows_args(kv=4)
    assert attn(q=[A, full[1] - 1] + full[2:]) == 2
    assert attn(out=[None] + full[1:]) == 101
    geo = geometry(page=1024, pstride=64, per=64)
    need = LIB.mivi_hip_kv_q4_attention_workspace(3, 7, 7, 4, 2, 64, 64 * 1024, 0)
    assert need > 0
    assert attn(geo=geo, ws_bytes=need - 1) == 2 and mivi_hip.last_error().expected == need
    assert attn(geo=geo, ws=None, ws_bytes=need) == 101
    assert attn(geo=geo, ws=A + 4, ws_bytes=need) == 101


def test_nothing_to_do_is_ok():
    for call in CALLS:
        assert call(rows=0) == 0
        assert call(geo=geometry(nseq=0)) == 0
    assert attn(max_rows=0) == 0


@pytest.mark.parametrize("call", CALLS)
def test_no_sequences_need_no_table(call):
    assert call(geo=geometry(nseq=0, pages=None, lens=None)) == 0  # what an empty tensor's address is
    assert call(geo=geometry(nseq=0, starts=None)) == 101


def test_workspace_grows_with_the_batch():
    f = LIB.mivi_hip_kv_q4_attention_workspace
    assert f(0, 7, 7, 4, 2, 64, 256, 0) == 0 and f(1, 0, 0, 4, 2, 64, 256, 0) == 0
    assert f(1, 1, 1, 5, 2, 64, 256, 0) == 0 and f(1, 1, 1, 4, 0, 64, 256, 0) == 0
    assert f(1, 1, 1, 32, 8, 64, 4096, 0) > 0


def test_python_refusals_on_host_tensors():
    data = torch.zeros(mivi_hip.kv_q4_page_bytes(2, 64, 64), dtype=torch.uint8)
    with pytest.raises(ValueError):
        mivi_hip.KvCacheQ4(data, torch.zeros((1, 1), dtype=torch.int32), 2, 64, 64)
