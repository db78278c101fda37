"""The step calls' Python binding (CPU only): when it is loaded."""
from __future__ import annotations

import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mivi-v4_amd")


def fresh(code: str) -> str:
    """What a new process that has the package prints."""
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=PKG))
    assert r.returncode == 0, r.stderr
    return r.stdout.strip()


def test_a_product_as_the_first_call():
    """Weights from another process (a pickle): no call before has loaded the
    binding. (On the host they are refused, as by a process that has.)"""
    assert fresh("""
        import torch, mivi_hip
        w = object.__new__(mivi_hip.W4Weights)
        w.data = torch.zeros(1088, dtype=torch.uint8)
        w._args = (w.data, 1, 0, 16, 128, 128)
        try:
            mivi_hip.w4_matmul_rows(torch.empty(1, 16), w, torch.zeros(1, 128))
        except ValueError as e:
            print(e)
    """) == "tensors are on a GPU"


def test_a_thread_that_comes_between():
    """Every entry point asks whether _step is there: while it is being loaded, no
    moment shows it without what goes with it."""
    assert fresh("""
        import sys
        import torch
        from mivi_hip import step
        seen = set()

        def trace(frame, event, arg):
            if frame.f_code is not step._load.__code__:
                return None
            frame.f_trace_opcodes = True
            seen.add((step._step is not None, step._raw_stream is not None and step._device is not None
                      and step.torch is not None))
            return trace
        sys.settrace(trace)
        step._load()
        sys.settrace(None)
        print((False, False) in seen, (True, False) in seen, step._step is not None)
    """) == "True False True"
