"""The arithmetic that cuts a list into parts (csrc/sb_split.cuh), compiled for the
host with overflow checks: every place in one part, whatever the list's length."""
from __future__ import annotations

import os
import shutil
import subprocess

from conftest import PKG

PROGRAM = r"""
#include "sb_split.cuh"
#include <cstdio>
int main() {
    int bad = 0;
    for (int warps : {1, 2, 148, 296, 592, 740, 1184})
        for (int least : {1, 2, 7})
            for (long long at : {1ll, 2ll, 3ll, 147ll, 148ll, 149ll, 1183ll, 1184ll, 1185ll, 5000ll, 4194303ll, 4194304ll,
                                 1ll << 30, 2147483647ll - 1184, 2147483647ll - 1183, 2147483647ll - 1, 2147483647ll}) {
                const int places = (int)at, part = part_of(places, warps, least), n = parts_in(places, part);
                if (part < least || n < 1 || n > warps) { printf("%d places, %d warps: part %d, %d parts\n", places, warps, part, n), ++bad; continue; }
                int end = 0;
                for (int w = 0; w < n; ++w) {
                    if (w * part != end) ++bad;   // starts where the one before ended
                    const int to = part_end(places, part, w);
                    if (to <= end || to > places || (w + 1 < n && to - end != part)) ++bad;
                    end = to;
                }
                if (end != places) printf("%d places, %d warps: ends at %d\n", places, warps, end), ++bad;
            }
    return bad ? 1 : 0;
}
"""


def test_every_place_is_in_one_part(tmp_path):
    src, exe = tmp_path / "split.cpp", str(tmp_path / "split")
    src.write_text(PROGRAM)
    cuda = os.environ.get("CUDA_HOME") or os.path.dirname(os.path.dirname(shutil.which("nvcc")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(PKG, "csrc"), "-I" + os.path.join(cuda, "include"), str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
