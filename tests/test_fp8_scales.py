"""8-bit weights whose scales are floats, through the traincpp API (tests/cpp/test_fp8_scales.cpp)."""
import subprocess

import pytest

from conftest import ROOT, announce

PROGRAM = str(ROOT / "tests" / "cpp" / "bin" / "test_fp8_scales")


@pytest.mark.gpu
def test_scales_of_floats():
    announce("fp8 scales of floats")
    r = subprocess.run([PROGRAM], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr


def test_activations_have_bytes():
    r = subprocess.run([PROGRAM, "--abort-type"], capture_output=True, text=True, timeout=60)
    assert r.returncode != 0 and "hip_fp8_new" in r.stderr
