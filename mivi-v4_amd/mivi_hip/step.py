"""The parts of a step around the paged 4-bit cache, for a host that drives its
own layers: `rms_norm`, `rms_norm_q8`, `rope` (with `rope_frequencies`),
`w4_matmul_rows` over `W4Weights`, and `verify_rows` (values and conventions:
include/mivi_hip.h, the mivi_hip_* calls of the same names).

Tensors are GPU tensors of one device; work is enqueued on `stream`, or on the
device's current one. A tensor used on another stream than its own (a W4Weights
too) is the caller's to keep until that work is done.
"""
from __future__ import annotations

from . import _check, _lib, kv_q4
from .kv_q4 import _TYPES, _stream_of

torch = _step = _raw_stream = _device = None  # set by the first call: the rest of the package works without torch
_needs = {}  # (vocabulary, sequences) -> the bytes of verify_rows' workspace
ROPE_KINDS = {"plain": 0, "linear": 1, "base": 2, "yarn": 3, "model": 4}


def _load():
    global torch, _step, _raw_stream, _device
    torch = kv_q4._load()
    from . import _step as calls  # the checks and calls (csrc/step_calls.cpp)
    _raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
    _step = calls  # last: another thread takes it for the sign that all are there


def _run(fn, of, stream, *args):
    """fn(stream's handle, *args) on the device of the tensor `of`: the given
    stream, or the current one there."""
    index = of.get_device()
    if index < 0:
        raise ValueError("tensors are on a GPU")
    if stream is None:
        raw = _raw_stream(index)
    elif isinstance(stream, int):
        raw = stream
    else:
        if stream.device.index != index:
            raise ValueError("the stream is on another device than the tensors")
        raw = stream.cuda_stream
    if _device() == index:
        rc = fn(raw, *args)
    else:
        with torch.cuda.device(index):
            rc = fn(raw, *args)
    if rc:
        _check(rc)


def rms_norm(out, x, weight, eps: float = 1e-5, residual=None, residual_out=None, stream=None):
    """out = s weight / sqrt(mean s^2 + eps) over the last dimension of s = x
    (+ residual), [rows, dim] or [rows, heads, dim]; s into residual_out where
    given (residual itself, to update it). weight: f32. Returns out."""
    if _step is None:
        _load()
    _run(_step.rms_norm, x, stream, out, x, weight, eps, residual, residual_out)
    return out


def rms_norm_q8(codes, scales, x, weight, eps: float = 1e-5, residual=None, residual_out=None, stream=None):
    """rms_norm of [rows, dim] in 8 bits: codes int8 [rows, dim], scales f32
    [rows, dim / group] (a group of 32 to 512 dimensions, or the whole row where
    scales is [rows, 1] or [rows])."""
    if _step is None:
        _load()
    _run(_step.rms_norm_q8, x, stream, codes, scales, x, weight, eps, residual, residual_out)


def rope_frequencies(rot_dim: int, base: float = 10000.0, kind: str = "plain", factor: float = 1.0,
                     context: int = 4096, device="cuda"):
    """Frequencies for `rope` as an f64 tensor: kind "plain", "linear", "base",
    "yarn" or "model" (see MIVI_ROPE_*) for a context `factor` times the trained
    one of `context` tokens."""
    if _step is None:
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
    if _step is None:
        _load()
    one = q if q is not None else k
    if one is None:
        raise ValueError("neither q nor k")
    _run(_step.rope, one, stream, q, k, freqs, positions, starts, lens, half, scale, q_out, k_out)
    return q if q_out is None else q_out, k if k_out is None else k_out


class W4Weights:
    """4-bit weights laid out for `w4_matmul_rows`: codes u8 [rows, cols / 2] (the
    even column in the low nibble), scales float16 or bfloat16 [rows, cols /
    group], zeros u8 (0..15) of that shape or None (8). The inputs are not kept."""

    def __init__(self, codes, scales, zeros=None, stream=None):
        if _step is None:
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
        for t, dtype, what in ((codes, torch.uint8, "codes"), (scales, scales.dtype, "scales"),
                               (zeros, torch.uint8, "zeros")):
            if t is not None and (t.dtype != dtype or not t.is_contiguous()):
                raise ValueError(f"{what} is a contiguous {dtype} tensor")
            if t is not None and t.device != d:
                raise ValueError(f"{what} is on another device")
        if d.type != "cuda":
            raise ValueError("tensors are on a GPU")
        args = (codes.data_ptr(), codes.numel(), self.scale_type, scales.data_ptr(), scales.numel(),
                None if zeros is None else zeros.data_ptr(), 0 if zeros is None else zeros.numel())
        n = _lib.mivi_hip_w4_packed_size(self.rows, self.cols, self.group, int(self.has_zeros))
        if n == 0:
            _check(_lib.mivi_hip_w4_pack(*args, None, 0, self.rows, self.cols, self.group, None))
        if stream is None:
            self.data = torch.empty(n, dtype=torch.uint8, device=d)
        else:
            with torch.cuda.stream(_stream_of(stream, d)):
                self.data = torch.empty(n, dtype=torch.uint8, device=d)
        self._args = (self.data, self.scale_type, int(self.has_zeros), self.rows, self.cols, self.group)
        kv_q4._call(_lib.mivi_hip_w4_pack, args + (self.data.data_ptr(), n, self.rows, self.cols, self.group), d, stream)
        if stream is not None:  # the inputs' memory is another stream's: reused only behind this one's work
            for t in (codes, scales, zeros):
                if t is not None:
                    t.record_stream(_stream_of(stream, d))


def w4_matmul_rows(out, weights: W4Weights, x, x_scales=None, stream=None):
    """out[batch, rows] = x[batch, cols] W^T: x of out's type, or int8 codes with
    x_scales (f32 [batch, cols / group]) as rms_norm_q8 leaves them. Returns out."""
    if _step is None:  # (weights may come from another process)
        _load()
    _run(_step.w4_matmul_rows, weights.data, stream, out, *weights._args, x, x_scales)
    return out


def verify_rows(tokens, counts, target, drafted, accept, pick, starts, draft=None, workspace=None, stream=None):
    """Verifies drafted tokens: target f32 [rows, vocab] probabilities, drafted
    int32 [rows] (of a sequence's last row unused), accept f32 [rows] and pick f32
    [sequences] uniform numbers, starts int32 [sequences + 1], draft f32 [rows,
    vocab] or None (certain). tokens int32 [rows] receives the accepted tokens, the
    drawn one and -1 behind it, counts int32 [sequences] the accepted. workspace:
    u8 GPU tensor (allocated here by default); calls that may overlap need their
    own."""
    if _step is None:
        _load()
    if workspace is None:
        sizes = (target.shape[-1], starts.numel() - 1)
        need = _needs.get(sizes)
        if need is None:
            if len(_needs) >= 1024:
                _needs.clear()
            need = _needs[sizes] = _lib.mivi_hip_verify_rows_workspace(max(sizes[0], 0), max(sizes[1], 0))
        if need and stream is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=target.device)
        elif need:  # from that stream's memory: reused only behind its work
            with torch.cuda.stream(_stream_of(stream, target.device)):
                workspace = torch.empty(need, dtype=torch.uint8, device=target.device)
    _run(_step.verify_rows, target, stream, tokens, counts, target, drafted, accept, pick, starts, draft, workspace)