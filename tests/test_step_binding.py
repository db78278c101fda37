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


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with the compiler replaced: the commands that it would run."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("mivi_build", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    commands = []

    def run(cmd, **_):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(m.subprocess, "run", run)
    (tmp_path / "mivi_hip").mkdir()
    for name, at in (("HERE", tmp_path), ("BUILD", tmp_path / "_build"), ("OUT", tmp_path / "mivi_hip" / "libmivi_hip.so")):
        monkeypatch.setattr(m, name, str(at))
    monkeypatch.setattr(m, "_deps", lambda src: [src])
    m.commands = commands
    return m


def bindings(m):
    n = sum(any(str(a).endswith("step_calls.cpp") for a in c) for c in m.commands)
    m.commands.clear()
    return n


def test_a_build_without_torch(build, monkeypatch):
    """The library is for hosts in any language: it is built, its Python binding is not."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.OUT and os.path.exists(build.OUT)
    assert bindings(build) == 0
    assert not os.path.exists(os.path.join(os.path.dirname(build.OUT), "_step.so"))


def test_a_build_for_another_torch(build, monkeypatch):
    """The binding is built again where torch or Python changed, its source or not."""
    import torch
    build.build()
    assert bindings(build) == 1
    build.build()
    assert bindings(build) == 0
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".next")
    build.build()
    assert bindings(build) == 1
    build.build()
    assert bindings(build) == 0
    monkeypatch.setattr(sys, "version", "3.99 " + sys.version)
    build.build()
    assert bindings(build) == 1
    build.build(force=True)
    assert bindings(build) == 1
