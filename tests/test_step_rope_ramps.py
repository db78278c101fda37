"""The frequencies' ramps against their definition (CPU only)."""
from __future__ import annotations

import math

import pytest
import torch

import mivi_hip


def index_of(turns, dim, base, context):
    """The real index at which a pair turns so many times over the context, by halving."""
    lo, hi = -1000.0 * dim, 1000.0 * dim
    for _ in range(200):
        mid = (lo + hi) / 2
        if context * base ** (-2 * mid / dim) > turns * 2 * math.pi:
            lo = mid
        else:
            hi = mid
    return lo


@pytest.mark.parametrize("dim,base,factor,context", [(64, 1e4, 8.0, 4096), (64, 1e6, 4.0, 32768), (128, 1e4, 32.0, 2048),
                                                     (96, 5e5, 2.5, 8192), (80, 1e4, 16.0, 1000), (32, 1e4, 4.0, 131072),
                                                     (128, 1e6, 1.5, 262144), (2, 1e4, 4.0, 4096)])
def test_yarn(dim, base, factor, context):
    f = mivi_hip.rope_frequencies(dim, base, "yarn", factor, context, device="cpu")
    # whole indexes around the real ones, within the pairs' range
    lo, hi = max(math.floor(index_of(32, dim, base, context)), 0), min(math.ceil(index_of(1, dim, base, context)), dim - 1)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        far = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
        assert abs(float(f[i]) / (plain * (1 - far) + plain / factor * far) - 1) < 1e-12, i


@pytest.mark.parametrize("dim,base,factor", [(64, 1e4, 8.0), (128, 1e6, 2.0), (2, 1e4, 4.0)])
def test_linear_and_base(dim, base, factor):
    """All divided; or of a base whose slowest pair is divided by the factor and whose
    fastest stays (one pair alone is the fastest)."""
    plain = base ** -(torch.arange(dim // 2, dtype=torch.float64) * 2 / dim)
    assert torch.allclose(mivi_hip.rope_frequencies(dim, base, "linear", factor, device="cpu"), plain / factor, rtol=1e-12, atol=0)
    f = mivi_hip.rope_frequencies(dim, base, "base", factor, device="cpu")
    share = torch.arange(dim // 2, dtype=torch.float64) / max(dim // 2 - 1, 1)
    assert torch.allclose(f, plain * factor ** -share, rtol=1e-12, atol=0)
