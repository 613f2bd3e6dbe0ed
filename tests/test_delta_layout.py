"""Places in the gated delta rule's workspaces (csrc/delta.h), checked by the compiler."""
from __future__ import annotations

import subprocess
from pathlib import Path

from sunnynet_amd import build

ROOT = Path(__file__).resolve().parents[1]


def test_fetches_stay_inside_their_matrix():
    cmd = [build.hipcc(), *build.HIPCC_FLAGS, "--cuda-host-only", "-fsyntax-only", f"-I{build.INCLUDE}", f"-I{build.CSRC}",
           "-x", "hip", str(ROOT / "tests" / "cpp" / "delta_fetch.cpp")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
