"""CPU: the benchmark's reference arm times the reference's own decoders, or says that they are not there."""
from __future__ import annotations

import json
import subprocess
import sys

import pytest

from conftest import ROOT
from oracle import loader


def test_reference_arm_without_the_reference():
    if loader.ref() is not None:
        pytest.skip("the reference's decoders are built here")
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--gpus", "1", "--steps", "1", "--warmup", "3"],
                       cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = r.stdout.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
