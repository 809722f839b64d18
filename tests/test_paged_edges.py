"""The paged-cache operators without a GPU, where bounds and handles decide."""
from __future__ import annotations

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_bounds_cpp_tests():
    exe = os.path.join(ROOT, "tests", "cpp", "paged_bounds_test")
    subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp"), "paged_bounds_test"], check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "paged bounds tests passed" in r.stdout
