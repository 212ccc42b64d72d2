"""Feed-forward calls of an empty batch without a GPU: workspace and acceptance at every width.  Each runs in a process
of its own, so that a call that ends its process fails its test and no other."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
ENODEV = 2

CALLS = """
import sys
from skmetal_amd import _bridge
lib, P = _bridge._lib, 1 << 20
a, k, chosen = map(int, sys.argv[1:])
d, o, chosen = 64, 64, chosen * 9 * P or None
for f, dtype in ((f, dtype) for f in (2048, 4096, 8192, 4100) for dtype in (0, 1, 2)):
    print("workspace", f, dtype, *(lib.skmetal_hip_feed_workspace(dtype, 0, d, f, o, k, a, b) for b in (0, 1)), flush=True)
    if not _bridge.HIP_AVAILABLE:  # an accepted call would write gradients to these addresses
        print("feed", f, dtype, lib.skmetal_hip_feed(dtype, None, d, P, f * d, d, 2 * P, f * d, d, 3 * P, o * f, f, chosen, None, 0, None, 0, None, o, None, 0, d, f, o, k, a,
                                                  4 * P, 1 << 40, None), flush=True)
        print("back", f, dtype, lib.skmetal_hip_feed_backward(dtype, None, o, None, d, P, f * d, d, 2 * P, f * d, d, 3 * P, o * f, f, chosen, None, 0, None, None, 0, None, d,
                                                           5 * P, 6 * P, 7 * P, None, 0, d, f, o, k, a, 4 * P, 1 << 40, None), flush=True)
"""


@pytest.mark.parametrize("a,k,chosen", [(1, 1, 0), (1, 1, 1), (1, 2, 1), (2, 1, 1)])
def test_empty_batch(a, k, chosen):
    """From 4,096 terms on a sum may be cut over blocks (2 f of them in the backward pass), of which no rows have none."""
    r = subprocess.run([sys.executable, "-W", "ignore", "-c", CALLS, *map(str, (a, k, chosen))], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": str(ROOT)})
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
    lines = [ln.split() for ln in r.stdout.splitlines()]
    assert sum(ln[0] == "workspace" for ln in lines) == 12
    for what, _, _, *values in lines:
        if what == "workspace":
            assert all(0 <= int(v) < 1 << 16 for v in values)  # no rows: the sort's tables at most
        else:
            assert int(values[0]) == ENODEV, (what, values)
