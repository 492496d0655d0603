"""Importing the package loads no compiled code of its own."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

from aicas_b200 import build

REPO = Path(__file__).resolve().parent.parent

SHOW = """
import aicas_b200, aicas_b200.workloads, aicas_b200.paged_decoder
mapped = [line.split()[-1] for line in open("/proc/self/maps") if line.rstrip().endswith(".so")]
print([p for p in mapped if p.startswith({root!r})])
from aicas_b200 import _hostpath
assert _hostpath.fast_append() is None and _hostpath.fast_decode() is None and _hostpath.fast_int4() is None
"""


def test_importing_maps_no_library():
    build.build_hostcalls()
    done = subprocess.run([sys.executable, "-c", SHOW.format(root=str(REPO))], cwd=REPO, capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.strip() == "[]", done.stdout + done.stderr
