"""The tuning calls of include/traincpp/trc_hip.h in each of their types, by tests/cpp/test_tuning_types.cpp: HipAdamW's
8-bit step bit for bit, and adapters in F32, F16 and BF16."""
import subprocess

import pytest

from conftest import ROOT, announce

pytestmark = pytest.mark.gpu


def test_every_type(hip):
    announce("tuning calls of every type")
    r = subprocess.run([str(ROOT / "tests" / "cpp" / "bin" / "test_tuning_types")], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr
