"""Runs training_gpu_cases.py and the example, each in one process in which torch comes before the library (the
two have to share one HIP runtime), apart from the process that runs the other GPU tests."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


def _run(args, timeout):
    p = subprocess.run([sys.executable, "-u"] + args, cwd=ROOT, capture_output=True, text=True, timeout=timeout)
    print(p.stdout[-20000:], flush=True)
    assert p.returncode == 0, p.stdout[-4000:] + p.stderr[-4000:]
    return p.stdout


def test_training_operators():
    out = _run(["-m", "pytest", os.path.join("tests", "training_gpu_cases.py"), "-m", "gpu", "-x", "-q", "-p", "no:cacheprovider"], 600)
    passed = re.search(r"(\d+) passed", out)
    assert passed and int(passed.group(1)) >= 400 and "skipped" not in out, out[-500:]


def test_the_example_learns():
    """examples/train_retriever.py: the operators together, and a search over what they trained."""
    out = _run([os.path.join("examples", "train_retriever.py"), "--items", "3000", "--dim", "64", "--steps", "40"], 120)
    losses = [float(x) for x in re.findall(r"loss ([0-9.]+)", out)]
    before, after = re.search(r"([0-9.]+) before, ([0-9.]+) after", out).groups()
    assert losses[-1] < losses[0] / 2 and float(after) > 0.9 and float(before) < 0.1
