"""bench.py where the reference's sources were not there to be built: its arm says so, in one line. CPU only."""
from __future__ import annotations

import json
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.parametrize("mode", ["model", "model-bs64", "moe"])
def test_reference_arm_without_the_reference(mode):
    from oracle import reference_available
    if reference_available():
        pytest.skip("the reference is built here")
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--steps", "2", "--mode", mode], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout)
    assert line["impl"] == "reference" and line["unavailable"]
