"""Timed cases of the parts of a step that a host drives itself, around the
paged 4-bit cache: norms, rotary positions, products with 4-bit weights, and
the verification of drafted tokens.

norm    s = x + residual, out = s (mean s^2 + eps)^(-1/2) w over the last
        dimension, and s itself rounded to its type; or out in 8 bits: in each
        group of a row (`group` dimensions, 0 the whole row) with A = max |s w|
        codes rint(127 s w / A) (ties to even), which stand for A (mean s^2 +
        eps)^(-1/2) / 127 times themselves.
rope    pairs (a, b) of the first `rot` dimensions turned by position times
        frequency, dimensions (2 i, 2 i + 1) or (i, i + rot / 2), the others
        copied. Rows are ragged as in the cache: row i of a sequence's n is at
        position len - n + i.
w4      out = x W^T, W's values (c - z) s: codes c in 0..15, a scale s and a
        zero z (8 without zeros) for `group` columns of a row. x in its type or
        as 8-bit codes with a scale for 128 columns.
verify  row i of a sequence's n but the last holds the target's probabilities p
        and the draft's q where token i was drafted; it is accepted if u q < p
        there and all before it are. The next token is drawn from the first row
        that is not: from max(p - q, 0), or from p in the last row (or where
        nothing is left): the first index whose cumulative sum passes u times
        the whole.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # a decode step of eight sequences of the 1.2B model, its norm for an
        # 8-bit product: latency alone
        dict(name="norm_step_8", kind="norm", type="f32", rows=8, heads=1, dim=2048, residual=True, q8=True, group=128),
        # the norm of every query head of a prompt's rows, in a fused projection
        dict(name="norm_heads_f16", kind="norm", type="f16", rows=4099, heads=32, dim=64, residual=False, q8=False, group=0),
        # a 2048-row pass of the model's prompt, for an 8-bit product
        dict(name="norm_tile_2048", kind="norm", type="f32", rows=2048, heads=1, dim=2048, residual=True, q8=True, group=128),
        # prompts of a serving batch, wide rows
        dict(name="norm_prompt_bf16", kind="norm", type="bf16", rows=16384, heads=1, dim=8192, residual=True, q8=False, group=0),
        # single tokens of eight sequences at a context of 32768, the model's heads
        dict(name="rope_step_8", kind="rope", type="f32", seqs=8, rows=1, hi=32768, heads=32, kv=8, hd=64, rot=64, half=False, stretch=8.0),
        # ragged prompts far into long contexts, part of the head
        dict(name="rope_prompt_bf16", kind="rope", type="bf16", seqs=6, rows=8191, hi=1000000, heads=32, kv=8, hd=128, rot=96, half=True, stretch=32.0),
        # one token through the 1.2B model's gate projection
        dict(name="w4_step_1", kind="w4", type="f32", x8=False, batch=1, n=8192, d=2048, group=128, zeros=False),
        # its output head, odd groups of rows, with zeros
        dict(name="w4_head_f16", kind="w4", type="f16", x8=False, batch=1, n=65535, d=2048, group=64, zeros=True),
        # a wide model's gate and up projection for eight sequences, on the norm's codes
        dict(name="w4_codes_8", kind="w4", type="bf16", x8=True, batch=8, n=28672, d=8192, group=128, zeros=False),
        # drafted tokens of sixteen sequences through a projection
        dict(name="w4_verify_80", kind="w4", type="bf16", x8=False, batch=80, n=14336, d=4096, group=32, zeros=True),
        # four drafted tokens of one sequence
        dict(name="verify_1x5", kind="verify", seqs=1, rows=5, vocab=65536, top=40, sure=False),
        # a serving batch, up to eight drafted tokens each, whole distributions
        dict(name="verify_64x9", kind="verify", seqs=64, rows=9, vocab=128256, top=0, sure=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "rope", "w4", "w4", "verify"))
    c = dict(kind=kind)
    if kind == "verify":
        c.update(seqs=_log(rng, 1, 64), rows=rng.randint(1, 9), vocab=_log(rng, 1000, 128256), top=rng.choice((0, 40)),
                 sure=rng.random() < 0.3)
        return c
    c["type"] = rng.choice(("f32", "f16", "bf16"))
    if kind == "norm":
        c["q8"] = rng.random() < 0.5
        c["heads"] = 1 if c["q8"] else rng.choice((1, 1, 4, 8, 32))
        c["dim"] = _log(rng, 16, 16384 if c["heads"] == 1 else 256)
        c["group"] = rng.choice((0, 32, 64, 128)) if c["q8"] else 0
        if c["group"]:
            c["dim"] = max(1, c["dim"] // c["group"]) * c["group"]
        c["rows"] = _log(rng, 1, 67108864 // (c["dim"] * c["heads"]))
        c["residual"] = c["heads"] == 1 and rng.random() < 0.7
        return c
    if kind == "rope":
        c["seqs"] = _log(rng, 1, 64)
        c["rows"] = _log(rng, 1, max(1, 16384 // c["seqs"]))
        c["hi"] = c["rows"] + _log(rng, 1, 1000000)
        c["kv"] = rng.choice((1, 2, 4, 8))
        c["heads"] = c["kv"] * rng.choice((1, 3, 4, 7))
        c["hd"] = rng.choice((32, 64, 80, 96, 128, 192, 256))
        c["rot"] = rng.choice((c["hd"], c["hd"], c["hd"] // 2, c["hd"] // 4))
        c["half"] = rng.random() < 0.5
        c["stretch"] = rng.choice((1.0, 4.0, 32.0))
        return c
    c["x8"] = rng.random() < 0.4
    c["group"] = rng.choice((32, 64, 128, 128))
    unit = 128 if c["x8"] else c["group"]
    c["d"] = unit * _log(rng, 2, 16384 // unit)
    c["batch"] = _log(rng, 1, 80)
    c["n"] = _log(rng, 16, min(131072, (234881024 if c["batch"] <= 8 else 58720256) // c["d"]))
    c["zeros"] = rng.random() < 0.5
    return c


def _ragged(case):
    """Rows and lengths of the sequences: the same for every seed of a case."""
    r = np.random.RandomState(case["seqs"] * 7919 + case["rows"] * 31)
    rows = r.randint(max(1, case["rows"] // 2), case["rows"] + 1, case["seqs"])
    rows[0] = case["rows"]
    hi = case.get("hi", case["rows"])
    lens = np.maximum(r.randint(max(1, hi // 2), hi + 1, case["seqs"]), rows)
    lens[0] = hi
    return rows.astype(np.int64), lens.astype(np.int64)


def work(case):
    kind = case["kind"]
    if kind == "verify":
        rows, _ = _ragged(case)
        # of each sequence one row of both distributions; a bonus row reads one
        return dict(bytes=case["seqs"] * case["vocab"] * 4 * (1 if case["sure"] else 2) + int(rows.sum()) * 20,
                    flops=case["seqs"] * case["vocab"] * 3)
    e = TYPES[case["type"]].itemsize
    if kind == "norm":
        n = case["rows"] * case["heads"] * case["dim"]
        out = n + 4 * case["rows"] * (case["dim"] // case["group"] if case["group"] else 1) if case["q8"] else n * e
        return dict(bytes=n * e * (3 if case["residual"] else 1) + out + 4 * case["dim"], flops=4 * n)
    if kind == "rope":
        n = int(_ragged(case)[0].sum()) * (case["heads"] + case["kv"])
        return dict(bytes=2 * n * case["hd"] * e, flops=3 * n * case["rot"])
    n, d, b = case["n"], case["d"], case["batch"]
    groups = n * (d // case["group"])
    x = b * d + b * (d // 128) * 4 if case["x8"] else b * d * e
    return dict(bytes=n * d // 2 + groups * 2 + (groups // 2 if case["zeros"] else 0) + x + b * n * e, flops=2 * b * n * d)


def _mivi():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mivi-v4_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mivi_hip
    return mivi_hip


def _freqs(case):
    """Radians a position: base 1000000, the slow half of the pairs stretched."""
    half = case["rot"] // 2
    f = 1e6 ** -(np.arange(half, dtype=np.float64) / half)
    ramp = np.clip((np.arange(half) / half - 0.25) * 2, 0, 1)
    return f * (1 - ramp) + f / case["stretch"] * ramp


def _cuda(a, dt):
    return torch.from_numpy(np.ascontiguousarray(a).astype(dt)).to(DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = case["kind"], dict(case=dict(case))

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=gen)

    if kind == "norm":
        dt, rows, heads, dim = TYPES[case["type"]], case["rows"], case["heads"], case["dim"]
        wide = normal(dim) * 0.3 + 1
        # a stream's channels are of different spread, some far out; heads stand
        # in a fused projection's rows, other columns behind them
        spread = torch.exp(0.5 * normal(dim))
        s["x"] = (normal(rows, heads + (heads + 1) // 2 if heads > 1 else 1, dim) * spread).to(dt)[:, :heads]
        s["w"] = wide
        if case["residual"]:
            s["r"] = (normal(rows, heads, dim) * spread * 4).to(dt)
        return s
    if kind == "rope":
        dt, hd = TYPES[case["type"]], case["hd"]
        rows, lens = _ragged(case)
        n = int(rows.sum())
        qkv = normal(n, case["heads"] + 2 * case["kv"], hd).to(dt)
        s["q"], s["k"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + case["kv"]]
        s["starts"], s["lens"] = _cuda(np.concatenate([[0], np.cumsum(rows)]), np.int32), _cuda(lens, np.int32)
        s["freqs"] = _cuda(_freqs(case), np.float64)
        return s
    if kind == "w4":
        n, d, g, b = case["n"], case["d"], case["group"], case["batch"]
        s["codes"] = torch.randint(0, 256, (n, d // 2), dtype=torch.uint8, device=DEV, generator=gen)
        s["scales"] = (0.002 + 0.004 * torch.rand((n, d // g), device=DEV, generator=gen)).to(torch.float16)
        s["zeros"] = torch.randint(5, 12, (n, d // g), dtype=torch.uint8, device=DEV, generator=gen) if case["zeros"] else None
        x = normal(b, d) * torch.exp(0.5 * normal(d))
        if case["x8"]:
            top = x.view(b, -1, 128).abs().amax(-1)
            s["x"] = (x.view(b, -1, 128) * (127 / top[..., None])).round().to(torch.int8).view(b, d)
            s["x_scales"] = top / 127
        else:
            s["x"] = x.to(TYPES[case["type"]])
        if own:  # laid out once, at load
            s["weights"] = _mivi().W4Weights(s["codes"], s["scales"], s["zeros"])
        return s
    rows, _ = _ragged(case)
    starts = np.concatenate([[0], np.cumsum(rows)])
    n, v = int(starts[-1]), case["vocab"]
    logits = 2.5 * normal(n, v)
    p = _chances(logits, case["top"])
    if case["sure"]:  # drafted by a lookup: likely tokens, no distribution
        t = torch.where(torch.rand(n, device=DEV, generator=gen) < 0.6, p.argmax(-1),
                        torch.randint(0, v, (n,), device=DEV, generator=gen))
    else:
        q = s["q"] = _chances(logits.add_(normal(n, v)), case["top"])
        u = torch.rand(n, dtype=torch.float64, device=DEV, generator=gen)
        cum = q.double().cumsum_(-1)
        t = (cum <= u[:, None] * cum[:, -1:]).sum(-1).clamp(max=v - 1)
        del cum
    s["p"], s["t"] = p, t.to(torch.int32)
    s["u"] = torch.rand(n, device=DEV, generator=gen)
    s["pick"] = torch.rand(case["seqs"], device=DEV, generator=gen)
    s["starts"] = _cuda(starts, np.int32)
    return s


def _chances(logits, top):
    if top:
        floor = torch.topk(logits, min(top, logits.shape[-1]), dim=-1).values[:, -1:]
        logits = torch.where(logits < floor, -math.inf, logits)
    return torch.softmax(logits, -1)


def _norm(s):
    c, dt = s["case"], TYPES[s["case"]["type"]]
    y = s["x"].float()
    out = {}
    if c["residual"]:
        y = y + s["r"].float()
        out["residual"] = y.to(dt)
    f = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    if not c["q8"]:
        return dict(out, out=(y * f * s["w"]).to(dt))
    # 64 bits: a quotient next to a half goes the right way
    y = s["x"].double() + s["r"].double() if c["residual"] else s["x"].double()
    y = (y * s["w"].double()).view(c["rows"], -1, c["group"] or c["dim"])
    top = y.abs().amax(-1, keepdim=True)
    codes = (y * 127 / torch.where(top == 0, 1.0, top)).round_()
    scale = (top * f.double() / 127).float()
    return dict(out, out=(codes.float() * scale).view(c["rows"], -1))


def _positions(s):
    row = torch.arange(s["q"].shape[0], device=DEV)
    starts, lens = s["starts"].long(), s["lens"].long()
    seq = (row[:, None] >= starts[1:]).sum(-1)
    return row - starts[seq + 1] + lens[seq]


def _rope(s):
    c = s["case"]
    angle = _positions(s).double()[:, None, None] * s["freqs"]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x):
        x, rot = x.float(), c["rot"]
        at = (slice(0, rot // 2), slice(rot // 2, rot)) if c["half"] else (slice(0, rot, 2), slice(1, rot, 2))
        a, b = x[..., at[0]], x[..., at[1]]
        out = x.clone()
        out[..., at[0]], out[..., at[1]] = a * cos - b * sin, b * cos + a * sin
        return out.to(TYPES[c["type"]])
    return dict(q=turn(s["q"]), k=turn(s["k"]))


def _w4(s):
    c = s["case"]
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(c["n"], -1, c["group"]).float()
    codes -= 8 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = codes.mul_(s["scales"].float()[..., None]).view(c["n"], c["d"])
    x = s["x"].float()
    if c["x8"]:
        x = (x.view(c["batch"], -1, 128) * s["x_scales"][..., None]).view(c["batch"], c["d"])
    return dict(out=torch.matmul(x, w.T).to(TYPES[c["type"]]))


def _verify(s):
    c, p, t = s["case"], s["p"], s["t"].long()
    rows = torch.arange(p.shape[0], device=DEV)
    starts = s["starts"].long()
    # 64 bits: products next to the border go the right way
    qt = 1.0 if c["sure"] else s["q"][rows, t].double()
    taken = s["u"].double() * qt < p[rows, t].double()
    at = starts[:-1, None] + torch.arange(c["rows"] - 1, device=DEV)
    drafted = at < starts[1:, None] - 1
    run_ = (taken[at.clamp(max=p.shape[0] - 1)] & drafted).long().cumprod(-1)
    count = run_.sum(-1)
    row = starts[:-1] + count
    last = row == starts[1:] - 1
    full = p[row].double()
    q = torch.zeros_like(full).scatter_(1, t[row][:, None], 1.0) if c["sure"] else s["q"][row].double()
    left = torch.where(last[:, None], full, (full - q).clamp_(min=0))
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, full)
    cum = left.cumsum(-1)
    pick = (cum <= s["pick"].double()[:, None] * cum[:, -1:]).sum(-1).clamp(max=c["vocab"] - 1)
    seq = (rows[:, None] >= starts[1:]).sum(-1)
    place = rows - starts[seq]
    tokens = torch.where(place < count[seq], t, torch.where(place == count[seq], pick[seq], -1))
    return dict(tokens=tokens.to(torch.int32), counts=count.to(torch.int32))


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if not own:
        return dict(norm=_norm, rope=_rope, w4=_w4, verify=_verify)[kind](s)
    m = _mivi()
    if kind == "norm":
        x, r = s["x"], s.get("r")
        held = None if r is None else torch.empty_like(r)
        out = {} if r is None else dict(residual=held)
        if not c["q8"]:
            y = torch.empty(x.shape, dtype=x.dtype, device=DEV)
            m.rms_norm(y, x, s["w"], EPS, residual=r, residual_out=held)
            return dict(out, out=y)
        x = x[:, 0]
        codes = torch.empty(x.shape, dtype=torch.int8, device=DEV)
        scales = torch.empty((c["rows"], c["dim"] // c["group"] if c["group"] else 1), dtype=torch.float32, device=DEV)
        m.rms_norm_q8(codes, scales, x, s["w"], EPS, residual=None if r is None else r[:, 0],
                      residual_out=None if r is None else held[:, 0])
        return dict(out, out=(codes.view(c["rows"], scales.shape[1], -1) * scales[..., None]).view(c["rows"], -1))
    if kind == "rope":
        q, k = (torch.empty(s[i].shape, dtype=s[i].dtype, device=DEV) for i in "qk")
        m.rope(s["q"], s["k"], s["freqs"], starts=s["starts"], lens=s["lens"], half=c["half"], q_out=q, k_out=k)
        return dict(q=q, k=k)
    if kind == "w4":
        out = torch.empty((c["batch"], c["n"]), dtype=TYPES[c["type"]], device=DEV)
        m.w4_matmul_rows(out, s["weights"], s["x"], s.get("x_scales"))
        return dict(out=out)
    tokens, counts = torch.empty_like(s["t"]), torch.empty(c["seqs"], dtype=torch.int32, device=DEV)
    m.verify_rows(tokens, counts, s["p"], s["t"], s["u"], s["pick"], s["starts"], draft=s.get("q"))
    return dict(tokens=tokens, counts=counts)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        s64 = s["x"].to(torch.float64)
        out = {}
        if "r" in s:
            s64 = s64 + s["r"]
            out["residual"] = s64
        f = 1 / torch.sqrt(torch.einsum("rhd,rhd->rh", s64, s64) / case["dim"] + EPS)
        if not case["q8"]:
            return dict(out, out=s64 * f[..., None] * s["w"])
        v = (s64 * s["w"]).unflatten(-1, (-1, case["group"] or case["dim"]))
        hi, lo = v.amax(-1), v.amin(-1)
        top = torch.maximum(hi, -lo)[..., None]
        codes = torch.where(top > 0, 127 * v / torch.where(top > 0, top, 1.0), 0.0).round()
        return dict(out, out=(codes * (top / 127) * f[..., None, None]).flatten(1))
    if kind == "rope":
        rows, lens = _ragged(case)
        pos = np.concatenate([np.arange(t - n, t) for n, t in zip(rows, lens)])
        angle = torch.from_numpy(np.outer(pos, _freqs(case))).to(DEV)[:, None]
        turn = torch.polar(torch.ones_like(angle), angle)
        rot, out = case["rot"], {}
        for name in "qk":
            x = s[name].to(torch.float64)
            part = x[..., :rot]
            part = part.unflatten(-1, (2, -1)).transpose(-1, -2) if case["half"] else part.unflatten(-1, (-1, 2))
            part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
            part = part.transpose(-1, -2).flatten(-2) if case["half"] else part.flatten(-2)
            out[name] = torch.cat([part, x[..., rot:]], -1)
        return out
    if kind == "w4":
        out = torch.empty((case["batch"], case["n"]), dtype=torch.float64, device=DEV)
        x, g = s["x"].double(), case["group"]
        if case["x8"]:
            x = x * s["x_scales"].double().repeat_interleave(128, -1)
        for a in range(0, case["n"], 8192):
            byte = s["codes"][a:a + 8192].to(torch.int32)
            w = torch.empty((byte.shape[0], case["d"]), dtype=torch.float64, device=DEV)
            w[:, 0::2], w[:, 1::2] = byte % 16, byte // 16
            w -= 8.0 if s["zeros"] is None else s["zeros"][a:a + 8192].double().repeat_interleave(g, -1)
            w *= s["scales"][a:a + 8192].double().repeat_interleave(g, -1)
            out[:, a:a + 8192] = x @ w.T.contiguous()
        return dict(out=out)
    starts = s["starts"].tolist()
    t, u, pick = s["t"].tolist(), s["u"].double().tolist(), s["pick"].double().tolist()
    tokens = np.full(len(t), -1, np.int32)
    counts = np.zeros(case["seqs"], np.int32)
    for i in range(case["seqs"]):
        row = starts[i]
        while row < starts[i + 1] - 1:
            q = 1.0 if case["sure"] else float(s["q"][row, t[row]])
            if not u[row] * q < float(s["p"][row, t[row]]):
                break
            tokens[row] = t[row]
            row += 1
        counts[i] = row - starts[i]
        p = s["p"][row].cpu().numpy().astype(np.float64)
        r = p
        if row < starts[i + 1] - 1:
            q = np.zeros_like(p) if case["sure"] else s["q"][row].cpu().numpy().astype(np.float64)
            if case["sure"]:
                q[t[row]] = 1.0
            r = np.maximum(p - q, 0.0)
            r = r if r.sum() > 0 else p
        cum = np.cumsum(r)
        tokens[row] = min(int(np.searchsorted(cum, pick[i] * cum[-1], side="right")), case["vocab"] - 1)
    return dict(tokens=torch.from_numpy(tokens).to(DEV), counts=torch.from_numpy(counts).to(DEV))
