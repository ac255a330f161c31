"""Builds the C++ test programs against libtraincpp_hip.so (the backend under test):
tests/cpp/bin/test_hip_backend, the drop-in test, which is checked by oracle/liboracle.so,
tests/cpp/bin/test_tuning and tests/cpp/bin/test_tuning_types."""
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent.parent


def build(name: str, oracle: bool) -> None:
    out = HERE / "bin" / name
    out.parent.mkdir(exist_ok=True)
    cmd = ["g++", "-std=c++20", "-O2", "-Wall", "-Wextra", "-Wno-unused-parameter",
           f"-I{ROOT / 'include'}", f"-I{ROOT / 'oracle'}", str(HERE / f"{name}.cpp"),
           f"-L{ROOT / 'train.cpp_amd' / 'lib'}", "-ltraincpp_hip", "-ltrc_hip",
           *([f"-L{ROOT / 'oracle'}", "-l:liboracle.so"] if oracle else []),
           "-Wl,-rpath,$ORIGIN/../../../train.cpp_amd/lib", "-Wl,-rpath,$ORIGIN/../../../oracle",
           "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise SystemExit(r.returncode)


def main() -> None:
    build("test_hip_backend", oracle=True)
    build("test_tuning", oracle=False)
    build("test_tuning_types", oracle=False)


if __name__ == "__main__":
    main()
