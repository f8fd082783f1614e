"""The host side of the paged attention (csrc/sb_attend.cu) without a GPU: its object
file linked with a CUDA runtime that only writes down what it is asked."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

CSRC = os.path.join(PKG, "csrc")
BASE = 0x10000   # a pointer that nothing follows


@pytest.fixture(scope="module")
def host(rtlib, tmp_path_factory):
    from sabah_moe_accelerator_b200 import rt
    subprocess.run(["make", "-s", "-C", CSRC, "_build/obj/sb_attend.o"], check=True)
    out = str(tmp_path_factory.mktemp("host") / "libattend_host.so")
    cuda = os.environ.get("CUDA_HOME") or os.path.dirname(os.path.dirname(shutil.which("nvcc")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-I" + os.path.join(cuda, "include"),
                    os.path.join(ROOT, "tests", "fake_cuda_host.cpp"), os.path.join(CSRC, "_build", "obj", "sb_attend.o"),
                    "-o", out], check=True)
    lib = ctypes.CDLL(out)
    for name in ("sabah_attend_paged", "sabah_attend_paged_workspace"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = rt.SIGNATURES[name]
    lib.fake_message.restype = ctypes.c_char_p
    return lib


def attend(lib, *, act=0, cache=1, n_pages=64, page=16, width=32, seqs=2, heads=8, kv=2, dim=128, window=0, workspace=None):
    ws = lib.sabah_attend_paged_workspace(heads, kv, dim) if workspace is None else workspace
    row, head = kv * dim * 2, dim * 2
    return lib.sabah_attend_paged(BASE, heads * dim * 4, dim * 4, act, BASE, page * row, row, head, BASE, page * row, row, head,
                                  cache, n_pages, page, BASE, 4 * width, width, BASE, seqs, heads, kv, dim, 0.1, window,
                                  BASE, None, BASE, ws, None)


def test_each_device_is_set_up(host):
    """The shared memory opt-in and the number of SMs are the current device's, whichever came first."""
    sizes = {}
    for dev in (0, 1, 0, 3, 70, 1):   # 70: past what is kept by number
        host.fake_set_device(dev)
        sizes.setdefault(dev, host.sabah_attend_paged_workspace(8, 2, 128))
        assert sizes[dev] == host.sabah_attend_paged_workspace(8, 2, 128)
        before = host.fake_launches()
        for dim in (64, 128, 256):
            assert attend(host, dim=dim) == 0, (dev, dim, host.fake_message())
            assert host.fake_last_grid() == {0: 148}.get(dev, min(148, 100 + dev)), (dev, dim)
        assert host.fake_launches() == before + 6   # the attention and its join
    assert host.fake_refused_launches() == 0
    assert sizes[1] < sizes[3] < sizes[0]
    host.fake_set_device(0)


def test_a_refused_call_leaves_no_timing_open(host):
    """A refusal after the checks of the arguments: the list of steps would be too long."""
    host.fake_set_device(0)
    open_before, launches = host.fake_open_timings(), host.fake_launches()
    assert attend(host, kv=4096, heads=4096, width=1 << 26, page=16) == -1
    assert b"too many" in host.fake_message()
    assert host.fake_open_timings() == open_before and host.fake_launches() == launches
    assert attend(host) == 0 and host.fake_open_timings() == open_before
