"""The step's operators from their definitions in 64 bits, on the CPU, and the
errors that their roundings can add up to."""
from __future__ import annotations

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24                                               # half a step of f32
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def f64(t):
    return t.detach().cpu().double()


def norm(x, w, eps, r=None):
    """s and s f w in 64 bits."""
    s = f64(x) if r is None else f64(x) + f64(r)
    f = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + float(np.float32(eps)))
    return s, s * f * f64(w)


def norm_close(out, want):
    """s, f and two products are rounded to f32, the result to its type."""
    room = want.abs() * (4.1 * U + (0 if out.dtype == torch.float32 else HALF_STEP[out.dtype])) + LEAST[out.dtype]
    return bool(((f64(out) - want).abs() <= room).all())


def sum_close(out, want):
    """Rounded to f32 and to its type."""
    room = want.abs() * (U * 1.001 + (0 if out.dtype == torch.float32 else HALF_STEP[out.dtype])) + LEAST[out.dtype]
    return bool(((f64(out) - want).abs() <= room).all())


def norm_q8(x, w, eps, group, r=None):
    """Codes and scales; each operation is one of the definition's."""
    s = (f64(x) if r is None else f64(x) + f64(r)).numpy()
    f = 1 / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(eps)))
    v = (s * f64(w).numpy()).reshape(s.shape[0], -1, group or s.shape[1])
    top = np.abs(v).max(-1, keepdims=True)
    codes = np.rint(127 * v / np.where(top == 0, 1, top)).reshape(s.shape)
    return torch.from_numpy(codes), torch.from_numpy(top[..., 0] * f / 127)


def rope(x, pos, freqs, half, scale=1.0):
    """The turned heads and, for each value, the error that roundings add up to:
    the angle's eighth of a turn, the polynomials and the products cost 6 U of m
    (|a| + |b|) together; the angle itself is a product of 64 bits."""
    x, n = f64(x), len(freqs)
    angle = pos.double()[:, None] * freqs.double()
    c, s = (scale * angle.cos())[:, None], (scale * angle.sin())[:, None]
    rot = x[..., :2 * n]
    a, b = (rot[..., :n], rot[..., n:]) if half else (rot[..., 0::2], rot[..., 1::2])
    y0, y1 = a * c - b * s, b * c + a * s
    room = (a.abs() + b.abs()) * abs(scale) * (6 * U + 4 * 2.0 ** -53 * angle.abs()[:, None])
    out, err = x.clone(), torch.zeros_like(x)
    if half:
        out[..., :n], out[..., n:2 * n], err[..., :n], err[..., n:2 * n] = y0, y1, room, room
    else:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2], err[..., 0:2 * n:2], err[..., 1:2 * n:2] = y0, y1, room, room
    return out, err


def rope_close(out, want, err):
    room = err + (0 if out.dtype == torch.float32 else HALF_STEP[out.dtype]) * (want.abs() + err) + LEAST[out.dtype]
    return bool(((f64(out) - want).abs() <= room).all())


def w4_dense(codes, scales, zeros):
    """The weights' values in 64 bits."""
    c, s = codes.cpu().numpy(), f64(scales).numpy()
    n, groups = s.shape
    w = np.empty((n, 2 * c.shape[1]))
    w[:, 0::2], w[:, 1::2] = c & 15, c >> 4
    z = np.full_like(s, 8.0) if zeros is None else (zeros.cpu().numpy() & 15).astype(np.float64)
    w = (w.reshape(n, groups, -1) - z[..., None]) * s[..., None]
    return torch.from_numpy(w.reshape(n, -1))


def w4_reach(codes, scales, zeros):
    """(c + z) |s|: what the two sums that a value's product may be taken from,
    s (sum c x - z sum x), add up to."""
    c, s = codes.cpu().numpy(), f64(scales).abs().numpy()
    n, groups = s.shape
    w = np.empty((n, 2 * c.shape[1]))
    w[:, 0::2], w[:, 1::2] = c & 15, c >> 4
    z = np.full_like(s, 8.0) if zeros is None else (zeros.cpu().numpy() & 15).astype(np.float64)
    w = (w.reshape(n, groups, -1) + z[..., None]) * s[..., None]
    return torch.from_numpy(w.reshape(n, -1))


def w4_close(out, x, w):
    """x in 64 bits; w: codes, scales and zeros. An f32 input may enter with 22
    bits, which are off by 2^-22 of it at most. Of cols products at most 32 are
    summed by an instruction, four such in a row, then a wave's steps of 128 and
    eight waves; each sum may be off by a whole step of f32, the factors' products
    by half of one each."""
    want = x @ w4_dense(*w).T
    size = x.abs() @ w4_reach(*w).T
    depth = 32 + 4 + x.shape[1] // 128 + 1 + 8 + 3
    room = size * (depth * 2 * U + 2 * U + 4 * U)
    room = room + (0 if out.dtype == torch.float32 else HALF_STEP[out.dtype]) * (want.abs() + room) + LEAST[out.dtype]
    return bool(((f64(out) - want).abs() <= room).all())


def verify(target, drafted, accept, pick, starts, draft=None):
    """Tokens and counts, row by row."""
    p_all, n = f64(target).numpy(), target.shape[1]
    q_all = None if draft is None else f64(draft).numpy()
    clean = lambda v: np.where(np.isfinite(v) & (v > 0), v, 0.0)  # noqa: E731
    t, u, k, st = drafted.tolist(), f64(accept).numpy(), f64(pick).numpy(), starts.tolist()
    tokens, counts = np.full(len(t), -7, np.int64), np.zeros(len(st) - 1, np.int64)
    for s in range(len(st) - 1):
        lo, hi = st[s], st[s + 1]
        if hi <= lo:
            continue
        row = lo
        while row < hi - 1:
            if not 0 <= t[row] < n:
                break
            p = clean(p_all[row, t[row]])
            q = 1.0 if draft is None else clean(q_all[row, t[row]])
            if not u[row] * q < p:
                break
            row += 1
        p = clean(p_all[row])
        left = p
        if row < hi - 1:
            if draft is None:
                q = np.zeros(n)
                if 0 <= t[row] < n:
                    q[t[row]] = 1
            else:
                q = clean(q_all[row])
            left = np.maximum(p - q, 0)
            if left.sum() == 0:
                left = p
        cum = np.cumsum(left)
        if cum[-1] == 0:
            token = -1
        else:
            hit = np.nonzero(cum > k[s] * cum[-1])[0]
            token = hit[0] if len(hit) else np.nonzero(left)[0][-1]
        tokens[lo:row], tokens[row], tokens[row + 1:hi] = t[lo:row], token, -1
        counts[s] = row - lo
    return tokens, counts
