"""The cache's attention and page entry points, host code only, under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/sanitize_kv): every call of a grid of shapes, types, alignments and strides
ends in a documented status with a message."""

import os
import shutil
import subprocess
from pathlib import Path

import pytest

SAN = Path(__file__).resolve().parent / "sanitize_kv"


def test_entry_points_are_clean_under_sanitizers():
    for tool in ("/opt/rocm/bin/hipcc", "/opt/rocm/llvm/bin/clang++"):
        if not os.access(tool, os.X_OK):
            pytest.skip(f"{tool} not available")
    if shutil.which("make") is None:
        pytest.skip("make not available")
    r = subprocess.run(["make", "-C", str(SAN), "-j", "5", "run"], capture_output=True, text=True,
                       timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith("calls ")]
    assert len(lines) == 1 and "unexpected 0" in lines[0] and "launch 0;" not in lines[0], out[-4000:]
    assert "Sanitizer" not in out and "runtime error" not in out, out[-4000:]
