"""The 4-bit cache's largest sizes are refused on the host, as overflows, where
a launch could not hold them (CPU only: nothing is launched)."""
from __future__ import annotations

import pytest

from test_kv_q4_abi import A, CALLS, LIB, attn, geometry, rows_args

HUGE = 1 << 40


def tensor(rs, hs):
    return [A, HUGE, rs, hs]


@pytest.mark.parametrize("call", CALLS[:2])
@pytest.mark.parametrize("n_seq,rows", [
    (1 << 26, 1 << 26),          # 8 values a thread: more than 2^32 threads
    (1 << 24, (1 << 27) + 5),    # whole groups: more than 2^24 workgroups
])
def test_more_rows_than_a_launch_holds(call, n_seq, rows):
    geo = geometry(kv=8, pstride=1, per=1, nseq=n_seq)
    assert call(geo=geo, k=tensor(512, 64), v=tensor(512, 64), rows=rows) == 4


@pytest.mark.parametrize("n_seq,rows,max_rows,per", [
    (1 << 23, 1 << 23, 1, 1),           # a workgroup a sequence and head: 2^24
    (1 << 22, (1 << 22) + 9, 9, 1),     # and of 72 pairs two of each
    (1 << 21, 1 << 21, 1, 32),          # joined by 2^24 workgroups
])
def test_more_attention_than_a_launch_holds(n_seq, rows, max_rows, per):
    """2 kv heads, 32 heads: the largest form of 64 dimensions, and the join."""
    geo = geometry(pstride=per, per=per, nseq=n_seq)
    args = dict(geo=geo, q=tensor(2048, 64), out=tensor(2048, 64), rows=rows, max_rows=max_rows, heads=32)
    assert attn(ws_bytes=1 << 60, **args) == 4


def test_workspace_of_sizes_that_no_call_has():
    f = LIB.mivi_hip_kv_q4_attention_workspace
    big = (1 << 64) - 1
    for i, value in ((0, big), (1, big), (3, 1 << 16), (5, 48), (5, big), (6, big), (6, 1 << 31)):
        args = [3, 7, 7, 4, 2, 64, 65536, 0]
        assert f(*args) > 0
        args[i] = value
        assert f(*args) == 0, (i, value)
    # a window or a row limit past everything is one that limits nothing
    for i in (2, 7):
        args = [3, 7, 7, 4, 2, 64, 65536, 0]
        want = f(*args)
        args[i] = big
        assert f(*args) == want
