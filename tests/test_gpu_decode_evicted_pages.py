"""Pages that a sliding window has left behind may be given back: their table entries are
not used, so the build that reports table entries out of range has nothing to report, also
where a page is smaller than a tile of keys. Each library runs in a child process of its own.
"""

from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
LIB_DIR = ROOT / "flashprefillv2-mlx_b200" / "fpv2" / "_lib"

CHILD = r"""
import json, sys, torch
sys.path[:0] = [sys.argv[1], sys.argv[2]]
import fpv2
from fpv2 import _lib
from tests.test_gpu_decode import problem

got = {"lib": str(_lib.LIB_PATH), "same": [], "clean": [], "reported": []}
for dim, page, new, window, sinks in ((64, 16, 1, 40, 5), (64, 8, 3, 100, 0), (128, 7, 1, 33, 9), (96, 16, 2, 50, 4),
                                      (128, 1, 2, 20, 1)):
    q, k, v, tables, n = problem([700, 90, 5], new, 8, 2, dim, page, torch.float16, seed=dim + page)
    args = dict(scale=0.1, window=window, sinks=sinks)
    want = fpv2.decode_attention(q, k, v, tables, n, **args)
    left = tables.clone()
    for i, length in enumerate(n.tolist()):
        low = max(0, length - new - window + 1)
        for at in range(tables.shape[1]):
            if at * page >= sinks and (at + 1) * page <= low:
                left[i, at] = -1 - at
    assert not torch.equal(left, tables)
    got["same"].append(bool(torch.equal(fpv2.decode_attention(q, k, v, left, n, **args), want)))
    got["clean"].append(_lib.device_status())
    left[0, 699 // page] = -1     # the newest key's own page: that is reported
    fpv2.decode_attention(q, k, v, left, n, **args)
    got["reported"].append(_lib.device_status())
print(json.dumps(got))
"""


def _run(lib: Path) -> dict:
    env = dict(os.environ, FPV2_LIBRARY=str(lib))
    res = subprocess.run([sys.executable, "-c", CHILD, str(ROOT / "flashprefillv2-mlx_b200"), str(ROOT)],
                         env=env, capture_output=True, text=True, timeout=300, cwd=str(ROOT))
    assert res.returncode == 0, res.stderr[-2000:]
    return json.loads(res.stdout.strip().splitlines()[-1])


def test_release_build():
    r = _run(LIB_DIR / "libfpv2_b200.so")
    assert all(r["same"]) and not any(r["clean"]) and not any(r["reported"]), r


@pytest.mark.skipif(not (LIB_DIR / "libfpv2_b200_debug.so").exists(),
                    reason="debug library not built (build.py --debug-bounds)")
def test_reporting_build():
    r = _run(LIB_DIR / "libfpv2_b200_debug.so")
    assert r["lib"].endswith("libfpv2_b200_debug.so"), r
    assert all(r["same"]) and not any(r["clean"]), r
    assert all(s & 8 for s in r["reported"]), r
