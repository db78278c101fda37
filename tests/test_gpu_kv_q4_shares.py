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
