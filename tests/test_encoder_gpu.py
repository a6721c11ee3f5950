"""Runs encoder_gpu_cases.py in one process in which torch comes before the library (the two have to share one HIP
runtime), apart from the process that runs the other GPU tests."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


def test_encoder_operators():
    args = ["-m", "pytest", os.path.join("tests", "encoder_gpu_cases.py"), "-m", "gpu", "-x", "-q", "--tb=short", "-p", "no:cacheprovider"]
    p = subprocess.run([sys.executable, "-u"] + args, cwd=ROOT, capture_output=True, text=True, timeout=600)
    print(p.stdout[-20000:], flush=True)
    assert p.returncode == 0, p.stdout[-4000:] + p.stderr[-4000:]
    assert re.search(r"\d+ passed", p.stdout) and "skipped" not in p.stdout


def test_the_example_runs():
    """examples/train_text_encoder.py: the operators together, and a search over what they made."""
    args = [os.path.join("examples", "train_text_encoder.py"), "--topics", "50", "--words", "1000", "--steps", "30"]
    p = subprocess.run([sys.executable, "-u"] + args, cwd=ROOT, capture_output=True, text=True, timeout=120)
    print(p.stdout, flush=True)
    assert p.returncode == 0, p.stderr[-4000:]
    assert re.search(r"[0-9.]+ before, [0-9.]+ after", p.stdout) and "nan" not in p.stdout
