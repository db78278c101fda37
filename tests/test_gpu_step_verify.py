"""Verification of drafted tokens against the definition, row by row."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_refs as ref

pytestmark = pytest.mark.gpu


def batch(rows, n, seed, top=0, noise=1.0, first=0, behind=0):
    g = torch.Generator().manual_seed(seed)
    starts = np.concatenate([[first], first + np.cumsum(rows)]).astype(np.int32)
    total = int(starts[-1]) + behind

    def chances(x):
        if top and top < n:
            x = torch.where(x < torch.topk(x, top, dim=-1).values[:, -1:], -torch.inf, x)
        return torch.softmax(x, -1)
    logits = 2 * torch.randn((total, n), generator=g)
    p, q = chances(logits), chances(logits + noise * torch.randn((total, n), generator=g))
    t = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32) if total else torch.empty(0, dtype=torch.int32)
    return dict(target=p, drafted=t, accept=torch.rand(total, generator=g), pick=torch.rand(len(rows), generator=g),
                starts=torch.from_numpy(starts), draft=q)


def check(hip, b, **kw):
    tokens = torch.full((b["target"].shape[0],), -7, dtype=torch.int32, device="cuda")
    counts = torch.full((b["starts"].numel() - 1,), -7, dtype=torch.int32, device="cuda")
    c = {k: None if v is None else v.cuda() for k, v in b.items()}
    hip.verify_rows(tokens, counts, c["target"], c["drafted"], c["accept"], c["pick"], c["starts"], draft=c["draft"], **kw)
    want_t, want_c = ref.verify(**b)
    assert counts.tolist() == want_c.tolist()
    assert tokens.tolist() == want_t.tolist()
    return tokens, counts


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 1000, 4095, 4096, 4097, 65536, 128256])
@pytest.mark.parametrize("noise", [0.0, 0.3, 2.0])
def test_sizes(hip, n, noise):
    check(hip, batch([5, 1, 2, 9], n, n, noise=noise))


@pytest.mark.parametrize("rows", [[1], [0], [0, 3, 0, 0, 1], [2] * 300, [700, 1, 600], [257, 258, 256]])
def test_ragged(hip, rows):
    b = batch(rows, 300, 3, noise=0.02, first=2, behind=3)
    check(hip, b)


@pytest.mark.parametrize("top", [1, 40])
def test_cut_distributions(hip, top):
    for seed in range(6):
        check(hip, batch([4, 6, 1, 8], 5000, seed, top=top, noise=0.5))


def test_certain_drafts(hip):
    for seed in range(4):
        b = batch([4, 6, 1, 8], 5000, seed, top=3)
        b["draft"] = None
        b["drafted"] = b["target"].argmax(-1).to(torch.int32)
        check(hip, b)


def test_many_chunks(hip):
    """More chunks than a workgroup has threads."""
    check(hip, batch([2, 2], 256 * 4096 + 4096 * 3 + 5, 1, noise=3.0))


def test_all_accepted_and_none(hip):
    b = batch([5, 5], 1000, 8)
    b["accept"].zero_()
    tokens, counts = check(hip, b)
    assert counts.tolist() == [4, 4]
    b["accept"].fill_(1.0)
    b["draft"] = b["target"] * 1.5
    tokens, counts = check(hip, b)  # nothing is left of max(p - q, 0): drawn from p
    assert counts.tolist() == [0, 0] and bool((tokens[1:5] == -1).all())


def test_borders(hip):
    """u q = p exactly is no acceptance; the smallest step below is one."""
    n = 8
    b = batch([2] * 3, n, 9)
    b["target"].fill_(0.125)
    b["draft"].fill_(0.25)
    for s, u in enumerate((0.5, float(np.nextafter(np.float32(0.5), np.float32(0))), 0.75)):
        b["accept"][2 * s] = u
    b["draft"][:, 0] = 0
    b["drafted"].fill_(3)
    _, counts = check(hip, b)
    assert counts.tolist() == [0, 1, 0]


def test_picks_at_the_ends(hip):
    n = 9000
    for pick in (0.0, float(np.nextafter(np.float32(1), np.float32(0))), 1.0):
        b = batch([1, 2, 1], n, 10)
        b["target"][:, :5000] = 0
        b["target"][:, 8000:] = 0
        b["draft"] = None
        b["drafted"].fill_(6000)
        b["pick"].fill_(pick)
        check(hip, b)


def test_ids_outside_and_values_that_are_no_chances(hip):
    b = batch([3, 3, 3, 2], 700, 11)
    b["drafted"][0], b["drafted"][3] = 700, -1
    b["target"][0, 5], b["target"][0, 6], b["target"][0, 7] = float("nan"), float("inf"), -3.0
    b["draft"][0, 8], b["draft"][3, 9] = float("nan"), -1.0
    b["target"][6, b["drafted"][6]] = float("nan")
    b["target"][9:] = 0
    b["draft"][9:] = 0
    tokens, _ = check(hip, b)
    assert tokens[9] == -1 and tokens[10] == -1


def test_strides_and_workspace(hip):
    b = batch([3, 4], 555, 12)
    wide_p, wide_q = torch.full((7, 600), 9.0), torch.full((7, 777), 9.0)
    wide_p[:, 3:558], wide_q[:, 1:556] = b["target"], b["draft"]
    b["target"], b["draft"] = wide_p[:, 3:558], wide_q[:, 1:556]
    need = hip.lib().mivi_hip_verify_rows_workspace(555, 2)
    c = {k: v.cuda() for k, v in b.items()}
    p, q = wide_p.cuda()[:, 3:558], wide_q.cuda()[:, 1:556]
    tokens, counts = torch.empty(7, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    hip.verify_rows(tokens, counts, p, c["drafted"], c["accept"], c["pick"], c["starts"], draft=q, workspace=ws)
    want_t, want_c = ref.verify(**b)
    assert tokens.tolist() == want_t.tolist() and counts.tolist() == want_c.tolist()


def test_distribution(hip):
    """Drafted and verified tokens have the target's distribution: 5 standard
    deviations of a multinomial count."""
    n, trials = 12, 20000
    g = torch.Generator().manual_seed(13)
    p1, q1 = torch.softmax(torch.randn(n, generator=g), -1), torch.softmax(torch.randn(n, generator=g), -1)
    b = dict(target=p1.expand(2 * trials, n).contiguous().cuda(), draft=q1.expand(2 * trials, n).contiguous().cuda(),
             drafted=torch.multinomial(q1.expand(2 * trials, n), 1, generator=g)[:, 0].to(torch.int32).cuda(),
             accept=torch.rand(2 * trials, generator=g).cuda(), pick=torch.rand(trials, generator=g).cuda(),
             starts=(torch.arange(trials + 1, dtype=torch.int32) * 2).cuda())
    tokens = torch.empty(2 * trials, dtype=torch.int32, device="cuda")
    counts = torch.empty(trials, dtype=torch.int32, device="cuda")
    hip.verify_rows(tokens, counts, b["target"], b["drafted"], b["accept"], b["pick"], b["starts"], draft=b["draft"])
    seen = torch.bincount(tokens[0::2].cpu().long(), minlength=n).double()
    p = p1.double()
    assert bool(((seen - trials * p).abs() <= 5 * torch.sqrt(trials * p * (1 - p))).all())


def test_tokens_over_the_drafted(hip):
    for certain in (False, True):
        b = batch([4, 6, 1, 8], 5000, 14, noise=0.3)
        if certain:
            b["draft"] = None
            b["drafted"] = b["target"].argmax(-1).to(torch.int32)
        c = {k: None if v is None else v.cuda() for k, v in b.items()}
        counts = torch.empty(4, dtype=torch.int32, device="cuda")
        hip.verify_rows(c["drafted"], counts, c["target"], c["drafted"], c["accept"], c["pick"], c["starts"], draft=c["draft"])
        want_t, want_c = ref.verify(**b)
        assert counts.tolist() == want_c.tolist() and c["drafted"].tolist() == want_t.tolist()
