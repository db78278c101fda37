"""A paged key/value cache held in 4 bits: `kv_q4_append`, `kv_q4_read` and
`kv_q4_attention` over a `KvCacheQ4` (values and conventions:
include/mivi_hip.h, the mivi_hip_kv_q4_* calls).

A batch is ragged: rows starts[s] .. starts[s+1] - 1 of the tensors belong to
sequence s and are its last positions, lens[s] - n .. lens[s] - 1. A step of a
model appends its rows' K and V, then attends with the same starts and lens.
"""
from __future__ import annotations

from . import _check, _lib

torch = None  # imported by the first cache: the rest of the package works without it
_TYPES = {}   # torch dtype -> GgmlType
_needs = {}   # a call's sizes -> the bytes of its workspace
_append = _lib.mivi_hip_kv_q4_append
_read = _lib.mivi_hip_kv_q4_read
_attention = _lib.mivi_hip_kv_q4_attention
_workspace = _lib.mivi_hip_kv_q4_attention_workspace


def kv_q4_page_bytes(n_kv_heads: int, head_dim: int, page_tokens: int) -> int:
    """Bytes of a page (0: no such geometry)."""
    return int(_lib.mivi_hip_kv_q4_page_bytes(n_kv_heads, head_dim, page_tokens))


class KvCacheQ4:
    """One layer's cache: `data` (contiguous u8 GPU tensor of whole pages) and
    `pages` (int32 GPU tensor [n_seq, pages_per_seq], rows contiguous, read at
    every call: change its contents freely, or set another tensor with
    `set_pages`). Both stay the caller's."""

    def __init__(self, data, pages, n_kv_heads: int, head_dim: int, page_tokens: int):
        global torch
        if torch is None:
            import torch as t
            _TYPES.update({t.float32: 0, t.float16: 1, t.bfloat16: 30})
            torch = t
        if data.dtype != torch.uint8 or not data.is_contiguous() or not data.is_cuda:
            raise ValueError("data is a contiguous u8 GPU tensor")
        self.data, self.n_kv_heads, self.head_dim, self.page_tokens = data, n_kv_heads, head_dim, page_tokens
        self.device = data.device
        self._geometry = (data.data_ptr(), data.numel(), n_kv_heads, head_dim, page_tokens)
        self.set_pages(pages)

    def set_pages(self, pages):
        if pages.dtype != torch.int32 or pages.dim() != 2 or (pages.shape[1] > 1 and pages.stride(1) != 1):
            raise ValueError("pages is a 2-D int32 tensor with contiguous rows")
        if pages.device != self.device:
            raise ValueError("pages and data are on different devices")
        self.pages = pages
        self._table = (pages.data_ptr(), pages.stride(0), pages.shape[1], pages.shape[0])

    def _batch(self, starts, lens):
        n = self._table[3]
        if starts.dtype != torch.int32 or lens.dtype != torch.int32 or not starts.is_contiguous() \
                or not lens.is_contiguous():
            raise ValueError("starts and lens are contiguous int32 tensors")
        if starts.numel() != n + 1 or lens.numel() != n:
            raise ValueError(f"{n} sequences: starts has {starts.numel()} values, lens {lens.numel()}")
        if starts.device != self.device or lens.device != self.device:
            raise ValueError("starts, lens and the cache are on different devices")
        return self._geometry + self._table + (starts.data_ptr(), lens.data_ptr())

    def _rows(self, t, heads: int, what: str):
        shape, strides = t.shape, t.stride()
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or strides[2] != 1:
            raise ValueError(f"{what} is [rows, {heads}, {self.head_dim}] with a contiguous last dimension")
        if t.device != self.device:
            raise ValueError(f"{what} and the cache are on different devices")
        rs, hs = strides[0], strides[1]
        # the elements from the first to the last: what a strided view spans
        span = (shape[0] - 1) * rs + (heads - 1) * hs + self.head_dim if shape[0] else 0
        return t.data_ptr(), span, rs, hs


def _type(a, b):
    t = _TYPES.get(a.dtype)
    if t is None or b.dtype != a.dtype:
        raise ValueError("tensors of one type: float32, float16 or bfloat16")
    return t


def _call(fn, args, device, stream):
    """fn(*args, stream) on `device`: the given stream, or the current one there."""
    if stream is None:
        raw = torch._C._cuda_getCurrentRawStream(device.index)
    elif isinstance(stream, int):
        raw = stream
    else:
        if stream.device != device:
            raise ValueError("the stream is on another device than the cache")
        raw = stream.cuda_stream
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(*args, raw)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw)
    if rc:
        _check(rc)


def _stream_of(stream, device):
    """The torch stream of an object or a handle (0: the default stream, which
    ExternalStream would take for a new one)."""
    if not isinstance(stream, int):
        return stream
    return torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)


def _kv(fn, cache, k, v, starts, lens, stream):
    if k.shape != v.shape:
        raise ValueError("k and v are of one shape")
    args = cache._batch(starts, lens) + (_type(k, v),) + cache._rows(k, cache.n_kv_heads, "k") \
        + cache._rows(v, cache.n_kv_heads, "v") + (k.shape[0],)
    _call(fn, args, cache.device, stream)


def kv_q4_append(cache: KvCacheQ4, k, v, starts, lens, stream=None):
    """Quantises the rows of k and v ([rows, n_kv_heads, head_dim], float32,
    float16 or bfloat16) into the cache as the sequences' last positions."""
    _kv(_append, cache, k, v, starts, lens, stream)


def kv_q4_read(cache: KvCacheQ4, k, v, starts, lens, stream=None):
    """Reads the sequences' last positions back into k and v (exact in float32
    and float16)."""
    _kv(_read, cache, k, v, starts, lens, stream)


def kv_q4_attention(out, q, cache: KvCacheQ4, starts, lens, max_rows: int | None = None, scale: float | None = None,
                    window: int = 0, workspace=None, stream=None):
    """out = softmax(scale q K^T) V per row and head of q ([rows, n_heads,
    head_dim]) over the cache, which holds the rows' own tokens already; a row
    at position p sees 0 .. p, or the last `window` of them. max_rows: at least
    the rows of any one sequence (default: all rows); scale: default
    head_dim ** -0.5. workspace: a u8 GPU tensor of at least the bytes that
    mivi_hip_kv_q4_attention_workspace names (allocated here by default); calls
    that may overlap need their own. Returns out."""
    shape = q.shape
    if shape != out.shape or len(shape) != 3:
        raise ValueError("q and out are [rows, n_heads, head_dim]")
    rows, heads, _ = shape
    max_rows = rows if max_rows is None else min(max_rows, rows)
    if window < 0 or max_rows < 0:
        raise ValueError("window and max_rows are not negative")
    batch = cache._batch(starts, lens)
    sizes = (cache._table[3], rows, max_rows, heads, cache.n_kv_heads, cache.head_dim,
             cache._table[2] * cache.page_tokens, window)
    need = _needs.get(sizes)
    if need is None:
        if len(_needs) >= 1024:
            _needs.clear()
        need = _needs[sizes] = _workspace(*sizes)
    device = cache.device
    if workspace is None and need:
        if stream is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        else:  # from that stream's memory: reused only behind its work
            with torch.cuda.stream(_stream_of(stream, device)):
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
    if workspace is not None and (workspace.device != device or not workspace.is_contiguous()):
        raise ValueError("workspace is a contiguous tensor on the cache's device")
    ws = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    args = (_type(q, out),) + cache._rows(out, heads, "out") + cache._rows(q, heads, "q") \
        + (rows, max_rows, heads, cache.head_dim ** -0.5 if scale is None else scale, window) + batch + ws
    _call(_attention, args, device, stream)
    return out
