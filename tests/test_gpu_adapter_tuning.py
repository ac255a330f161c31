"""Adapter tuning through the traincpp API: examples/adapter_tuning.cpp, whose quantized
projection, adapters, preference loss, gradients and AdamW steps run together on the device, and
the optimizer's state by tests/cpp/test_tuning.cpp."""
import subprocess

import pytest

from conftest import ROOT, announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", ["8", "32"])
def test_example_learns(bits):
    announce(f"adapter tuning example, moments in {bits} bits")
    r = subprocess.run([str(ROOT / "examples" / "bin" / "adapter_tuning"), "60", bits], capture_output=True, text=True,
                       timeout=60)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ok: loss" in r.stdout


def test_optimizer_state():
    announce("HipAdamW state")
    r = subprocess.run([str(ROOT / "tests" / "cpp" / "bin" / "test_tuning")], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr
