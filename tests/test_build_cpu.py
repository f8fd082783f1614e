"""What `make` builds: the runtime for everyone, the torch module where torch is."""
from __future__ import annotations

import os
import subprocess
import sys

from conftest import PKG


def plan(python):
    """The commands of a build from nothing."""
    r = subprocess.run(["make", "-B", "-n", "-C", os.path.join(PKG, "csrc"), "PY=" + python], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_the_runtime_builds_without_torch():
    """A C caller's Python has no torch (here: no site packages)."""
    p = plan(sys.executable + " -S")
    assert "-o ../libsabah_rt.so" in p and "-o ../_torch_ops.so" not in p and "_torch_ops.so is not built" in p


def test_both_build_with_torch():
    p = plan(sys.executable)
    assert "-o ../libsabah_rt.so" in p and "-o ../_torch_ops.so" in p
