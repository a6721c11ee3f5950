"""Runs encoder_gpu_ranges.py in one process in which torch comes before the library (the two have to share one
HIP runtime), all of it whatever fails."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


def test_encoder_ranges():
    args = ["-m", "pytest", os.path.join("tests", "encoder_gpu_ranges.py"), "-m", "gpu", "-q", "--tb=short", "-p", "no:cacheprovider"]
    p = subprocess.run([sys.executable, "-u"] + args, cwd=ROOT, capture_output=True, text=True, timeout=600)
    print(p.stdout[-20000:], flush=True)
    assert p.returncode == 0, "\n".join(l for l in p.stdout.splitlines() if l.startswith(("FAILED", "ERROR"))) or p.stderr[-4000:]
    assert re.search(r"\d+ passed", p.stdout) and "skipped" not in p.stdout
