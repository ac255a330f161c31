"""Distillation into adapters beside 8-bit weights through the traincpp API: examples/distillation.cpp runs, and
tests/cpp/test_distillation.cpp holds each result of such a step, its gradients among them, to 64 bits and to differences."""
import subprocess

import pytest

from conftest import ROOT, announce

pytestmark = pytest.mark.gpu


def test_step_against_64_bits():
    announce("distillation step")
    r = subprocess.run([str(ROOT / "tests" / "cpp" / "bin" / "test_distillation")], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("steps", ["1", "30"])
def test_example_runs(steps):
    announce(f"distillation example, {steps} steps")
    r = subprocess.run([str(ROOT / "examples" / "bin" / "distillation"), steps], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0 and "ok: one token" in r.stdout, r.stdout + r.stderr
    assert "nan" not in r.stdout
