"""The parts of a step around the paged 4-bit cache, for a host that drives its
own layers: `rms_norm`, `rms_norm_q8`, `rope` (with `rope_frequencies`),
`w4_matmul_rows` over `W4Weights`, and `verify_rows` (values and conventions:
include/mivi_hip.h, the mivi_hip_* calls of the same names).

Tensors are GPU tensors of one device; work is enqueued on `stream`, or on the
device's current one.
"""
from __future__ import annotations

from . import _check, _lib, kv_q4
from .kv_q4 import _TYPES, _stream_of

torch = None  # imported by the first call: the rest of the package works without it
ROPE_KINDS = {"plain": 0, "linear": 1, "base": 2, "yarn": 3, "model": 4}


def _load():
    global torch
    torch = kv_q4._load()


def _call(fn, args, device, stream):
    if device.type != "cuda":
        raise ValueError("tensors are on a GPU")
    kv_q4._call(fn, args, device, stream)


def _type(t):
    k = _TYPES.get(t.dtype)
    if k is None:
        raise ValueError("tensors are float32, float16 or bfloat16")
    return k


def _rows(t, like, what):
    """(pointer, span, row stride, head stride) of [rows, (heads,) dim] of the
    shape, type and device of `like`."""
    shape, st = t.shape, t.stride()
    if shape != like.shape or t.dtype != like.dtype:
        raise ValueError(f"{what} is of shape {tuple(like.shape)} and {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{what} is on another device")
    if shape[-1] > 1 and st[-1] != 1:
        raise ValueError(f"{what} has a contiguous last dimension")
    if len(shape) == 2:
        return t.data_ptr(), (shape[0] - 1) * st[0] + shape[1] if shape[0] else 0, st[0], 0
    if shape[0] == 0 or shape[1] == 0:
        return t.data_ptr(), 0, st[0], st[1]
    return t.data_ptr(), (shape[0] - 1) * st[0] + (shape[1] - 1) * st[1] + shape[2], st[0], st[1]


def _array(t, dtype, device, what, numel=None):
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} is a contiguous {dtype} tensor")
    if t.device != device:
        raise ValueError(f"{what} is on another device")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{what} has {t.numel()} values, not {numel}")
    return t.data_ptr(), t.numel()


def rms_norm(out, x, weight, eps: float = 1e-5, residual=None, residual_out=None, stream=None):
    """out = s weight / sqrt(mean s^2 + eps) over the last dimension of s = x
    (+ residual), [rows, dim] or [rows, heads, dim]; s into residual_out where
    given (residual itself, to update it). weight: f32. Returns out."""
    if torch is None:
        _load()
    if x.dim() not in (2, 3):
        raise ValueError("x is [rows, dim] or [rows, heads, dim]")
    d = x.device
    rows, heads, dim = x.shape[0], 1 if x.dim() == 2 else x.shape[1], x.shape[-1]
    none = (None, 0, 0, 0)
    args = (_type(x),) + _rows(out, x, "out") + _rows(x, x, "x") \
        + (none if residual is None else _rows(residual, x, "residual")) \
        + (none if residual_out is None else _rows(residual_out, x, "residual_out")) \
        + _array(weight, torch.float32, d, "weight", dim) + (eps, rows, heads, dim)
    _call(_lib.mivi_hip_rms_norm, args, d, stream)
    return out


def rms_norm_q8(codes, scales, x, weight, eps: float = 1e-5, residual=None, residual_out=None, stream=None):
    """rms_norm of [rows, dim] in 8 bits: codes int8 [rows, dim], scales f32
    [rows, dim / group] (a group of 32 to 512 dimensions, or the whole row where
    scales is [rows, 1] or [rows])."""
    if torch is None:
        _load()
    if x.dim() != 2 or codes.shape != x.shape:
        raise ValueError("x and codes are [rows, dim]")
    d = x.device
    rows, dim = x.shape
    none = (None, 0, 0)
    args = (_type(x),) + _array(codes, torch.int8, d, "codes") + _array(scales, torch.float32, d, "scales") \
        + (_group(scales, rows, dim, "scales"),) + _rows(x, x, "x")[:3] \
        + (none if residual is None else _rows(residual, x, "residual")[:3]) \
        + (none if residual_out is None else _rows(residual_out, x, "residual_out")[:3]) \
        + _array(weight, torch.float32, d, "weight", dim) + (eps, rows, dim)
    _call(_lib.mivi_hip_rms_norm_q8, args, d, stream)


def _group(scales, rows, dim, what):
    """Dimensions of a scale (0: one a row)."""
    n = 1 if scales.dim() == 1 else scales.shape[1]
    if scales.dim() not in (1, 2) or scales.shape[0] != rows or n == 0 or dim % n:
        raise ValueError(f"{what} is [rows, dim / group]")
    return 0 if n == 1 else dim // n


def rope_frequencies(rot_dim: int, base: float = 10000.0, kind: str = "plain", factor: float = 1.0,
                     context: int = 4096, device="cuda"):
    """Frequencies for `rope` as an f64 tensor: kind "plain", "linear", "base",
    "yarn" or "model" (see MIVI_ROPE_*) for a context `factor` times the trained
    one of `context` tokens."""
    if torch is None:
        _load()
    if kind not in ROPE_KINDS:
        raise ValueError(f"kind is one of {', '.join(ROPE_KINDS)}")
    f = torch.empty(max(rot_dim // 2, 0), dtype=torch.float64)
    _check(_lib.mivi_hip_rope_frequencies(ROPE_KINDS[kind], base, factor, context, rot_dim, f.data_ptr(), f.numel()))
    return f.to(device)


def rope(q, k, freqs, positions=None, starts=None, lens=None, half: bool = False, scale: float = 1.0, q_out=None,
         k_out=None, stream=None):
    """Turns the pairs of q's and k's heads ([rows, heads, head_dim]; either may be
    None) by position times freqs (f64, one for each of the first dimensions'
    pairs): (2 i, 2 i + 1), or (i, i + len(freqs)) with half. positions: int32
    [rows]; or starts and lens of a batch, as kv_q4_append takes them. In place
    without q_out and k_out. Returns (q_out, k_out)."""
    if torch is None:
        _load()
    one = q if q is not None else k
    if one is None:
        raise ValueError("neither q nor k")
    d, rows, hd = one.device, one.shape[0], one.shape[-1]
    args = (_type(one),)
    outs = []
    for t, o, what in ((q, q_out, "q"), (k, k_out, "k")):
        if t is None:
            args += (None, 0, 0, 0, None, 0, 0, 0, 0)
            outs.append(None)
            continue
        if t.dim() != 3 or t.shape[0] != rows or t.shape[2] != hd or t.dtype != one.dtype or t.device != d:
            raise ValueError("q and k are [rows, heads, head_dim], of one type and device")
        o = t if o is None else o
        outs.append(o)
        args += _rows(o, t, what + "_out") + _rows(t, t, what) + (t.shape[1],)
    f, n = _array(freqs, torch.float64, d, "freqs")
    args += (rows, hd, 2 * n, int(half), f, n, scale)
    if (positions is None) == (starts is None) or (starts is None) != (lens is None):
        raise ValueError("either positions, or starts and lens")
    if positions is not None:
        args += _array(positions, torch.int32, d, "positions", rows) + (None, None, 0)
    else:
        s, m = _array(starts, torch.int32, d, "starts")
        args += (None, 0, s, _array(lens, torch.int32, d, "lens", m - 1)[0], m - 1)
    _call(_lib.mivi_hip_rope, args, d, stream)
    return tuple(outs)


class W4Weights:
    """4-bit weights laid out for `w4_matmul_rows`: codes u8 [rows, cols / 2] (the
    even column in the low nibble), scales float16 or bfloat16 [rows, cols /
    group], zeros u8 (0..15) of that shape or None (8). The inputs are not kept."""

    def __init__(self, codes, scales, zeros=None, stream=None):
        if torch is None:
            _load()
        if codes.dim() != 2 or scales.dim() != 2 or scales.shape[0] != codes.shape[0] or scales.shape[1] == 0:
            raise ValueError("codes is [rows, cols / 2], scales [rows, cols / group]")
        if scales.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("scales are float16 or bfloat16")
        if zeros is not None and zeros.shape != scales.shape:
            raise ValueError("zeros are of the scales' shape")
        self.rows, self.cols = codes.shape[0], codes.shape[1] * 2
        if self.cols % scales.shape[1]:
            raise ValueError("scales is [rows, cols / group]")
        self.group, self.device, self.has_zeros = self.cols // scales.shape[1], codes.device, zeros is not None
        self.scale_type = _TYPES[scales.dtype]
        d = self.device
        args = _array(codes, torch.uint8, d, "codes") + (self.scale_type,) + _array(scales, scales.dtype, d, "scales") \
            + ((None, 0) if zeros is None else _array(zeros, torch.uint8, d, "zeros"))
        n = _lib.mivi_hip_w4_packed_size(self.rows, self.cols, self.group, int(self.has_zeros))
        if n == 0:
            _check(_lib.mivi_hip_w4_pack(*args, None, 0, self.rows, self.cols, self.group, None))
        if stream is None:
            self.data = torch.empty(n, dtype=torch.uint8, device=d)
        else:
            with torch.cuda.stream(_stream_of(stream, d)):
                self.data = torch.empty(n, dtype=torch.uint8, device=d)
        self._args = (self.data.data_ptr(), n, self.scale_type, int(self.has_zeros))
        _call(_lib.mivi_hip_w4_pack, args + (self.data.data_ptr(), n, self.rows, self.cols, self.group), d, stream)


def w4_matmul_rows(out, weights: W4Weights, x, x_scales=None, stream=None):
    """out[batch, rows] = x[batch, cols] W^T: x of out's type, or int8 codes with
    x_scales (f32 [batch, cols / group]) as rms_norm_q8 leaves them. Returns out."""
    w = weights
    if out.dim() != 2 or x.dim() != 2 or out.shape[0] != x.shape[0]:
        raise ValueError("x is [batch, cols], out [batch, rows]")
    batch = x.shape[0]
    if x.shape[1] != w.cols or out.shape[1] != w.rows:
        raise ValueError(f"weights are {w.rows} x {w.cols}")
    if x.device != w.device:
        raise ValueError("x is on another device than the weights")
    o = _rows(out, out, "out")[:3]
    if out.device != w.device:
        raise ValueError("out is on another device than the weights")
    if x_scales is None:
        if x.dtype != out.dtype:
            raise ValueError("x and out are of one type")
        _call(_lib.mivi_hip_w4_matmul_rows, (_type(out),) + o + w._args + _rows(x, x, "x")[:3]
              + (batch, w.rows, w.cols, w.group), w.device, stream)
    else:
        _call(_lib.mivi_hip_w4_matmul_rows_q8, (_type(out),) + o + w._args + _array(x, torch.int8, w.device, "x")
              + _array(x_scales, torch.float32, w.device, "x_scales")
              + (_group(x_scales, batch, w.cols, "x_scales"), batch, w.rows, w.cols, w.group), w.device, stream)
    return out


def verify_rows(tokens, counts, target, drafted, accept, pick, starts, draft=None, workspace=None, stream=None):
    """Verifies drafted tokens: target f32 [rows, vocab] probabilities, drafted
    int32 [rows] (of a sequence's last row unused), accept f32 [rows] and pick f32
    [sequences] uniform numbers, starts int32 [sequences + 1], draft f32 [rows,
    vocab] or None (certain). tokens int32 [rows] receives the accepted tokens, the
    drawn one and -1 behind it, counts int32 [sequences] the accepted. workspace:
    u8 GPU tensor (allocated here by default); calls that may overlap need their
    own."""
    if torch is None:
        _load()
    d = target.device
    if target.dim() != 2 or target.dtype != torch.float32:
        raise ValueError("target is [rows, vocab] of float32")
    rows, n = target.shape
    s, m = _array(starts, torch.int32, d, "starts")
    i32, f32, seqs = torch.int32, torch.float32, m - 1
    if seqs < 0:
        raise ValueError("starts has a value more than there are sequences")
    args = _array(tokens, i32, d, "tokens", rows) + _array(counts, i32, d, "counts", seqs) \
        + _rows(target, target, "target")[:3] + ((None, 0, 0) if draft is None else _rows(draft, target, "draft")[:3]) \
        + _array(drafted, i32, d, "drafted", rows) + _array(accept, f32, d, "accept", rows) \
        + _array(pick, f32, d, "pick", seqs) + (s, seqs, rows, n)
    need = _lib.mivi_hip_verify_rows_workspace(n, seqs)
    if workspace is None and need:
        if stream is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=d)
        else:  # from that stream's memory: reused only behind its work
            with torch.cuda.stream(_stream_of(stream, d)):
                workspace = torch.empty(need, dtype=torch.uint8, device=d)
    if workspace is not None and (workspace.device != d or not workspace.is_contiguous()):
        raise ValueError("workspace is a contiguous tensor on the other tensors' device")
    ws = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _call(_lib.mivi_hip_verify_rows, args + ws, d, stream)
