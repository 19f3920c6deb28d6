"""Growth of scratch that a call can do without: tests/host_plan/scratch_check.cpp is compiled with the library's own header."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_scratch_grows_up_to_its_limit_and_does_not_ask_twice(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp_path / "scratch_check"
    done = subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}", f"-I{ROOT / 'psi-dec_b200' / 'csrc'}",
                           str(ROOT / "tests" / "host_plan" / "scratch_check.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "scratch ok" in done.stdout, done.stdout + done.stderr
