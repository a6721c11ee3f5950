"""Runs tests/cpp/test_encoder.cpp: attention, head norms and clipping through the C++ host API.  The binary is built by
vector-rs_amd/Makefile."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "vector-rs_amd")
BIN = os.path.join(PKG, "_build", "test_encoder")


def _run(args, timeout):
    if not os.path.exists(BIN):
        subprocess.run(["make", "-s", "-C", PKG, "_build/test_encoder"], check=True)
    p = subprocess.run([BIN] + args, capture_output=True, text=True, timeout=timeout)
    print(p.stdout)
    fails = [l for l in p.stdout.splitlines() if l.startswith("FAIL")]
    assert p.returncode == 0 and not fails, "\n".join(fails) or p.stderr
    return p.stdout


def test_encoder_refusals_from_cpp():
    assert _run(["--host"], 60).count("PASS") == 4


@pytest.mark.gpu
def test_encoder_operators_from_cpp():
    assert _run([], 110).count("PASS") == 10
