"""Runs the program of the C++ launchers of the 8-bit cache (tests/cpp/test_kv8.cpp): their
refusals on the CPU, and on the GPU inputs whose results are known."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
EXE = ROOT / "tests" / "cpp" / "test_kv8"


def _run(*args):
    if not EXE.exists():
        subprocess.run(["make", "-j8", "-C", str(ROOT / "mini-infer_amd")], check=True, capture_output=True)
        subprocess.run(["make", "-C", str(ROOT / "tests" / "cpp"), "test_kv8"], check=True, capture_output=True)
    r = subprocess.run([str(EXE), *args], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0 and "ALL OK" in r.stdout, r.stdout + r.stderr


def test_refusals():
    _run("--cpu")


@pytest.mark.gpu
def test_known_results(dev):
    print("[case] C++ launchers of the 8-bit cache", flush=True)
    _run()
