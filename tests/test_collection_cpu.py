"""The order of a GPU session: what fails for want of the reference's build does not
keep the other files from running under -x."""
from __future__ import annotations

import os
import subprocess
import sys

from conftest import REFERENCE_BUILDS, ROOT


def test_tests_without_their_reference_build_come_last():
    r = subprocess.run([sys.executable, "-m", "pytest", "--collect-only", "-q", "-m", "gpu", "-p", "no:cacheprovider", "tests"],
                       cwd=ROOT, capture_output=True, text=True, timeout=300)
    files = [line.split("::")[0] for line in r.stdout.splitlines() if "::" in line]
    names = list(dict.fromkeys(os.path.basename(f) for f in files))
    missing = [n for n, built in REFERENCE_BUILDS.items() if not os.path.exists(built)]
    assert set(names) >= set(REFERENCE_BUILDS), r.stdout[-2000:]
    assert names[len(names) - len(missing):] == missing
    rest = names[:len(names) - len(missing)]
    assert rest == sorted(rest)
