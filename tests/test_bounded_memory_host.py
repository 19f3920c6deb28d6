"""Key weights, eviction and linear attention as C and C++ callers see them, and the parts that need no GPU."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

import hostapi as H
from test_cpp_host import _cuda_include

pkg = H.pkg
ROOT = Path(__file__).resolve().parent.parent


def build(compiler, flags, source, exe, libs=()):
    found = shutil.which(compiler)
    if found is None:
        pytest.skip(f"no {compiler}")
    lib = pkg.library_path().parent
    cmd = [found, *flags, "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}", str(source), "-o", str(exe), f"-L{lib}", "-lpsi_cuda",
           f"-Wl,-rpath,{lib}", *libs]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    return exe


def test_the_header_from_c_and_what_null_handles_answer(tmp_path):
    exe = build("gcc", ["-std=c11", "-pedantic"], ROOT / "tests" / "c_abi" / "bounded_memory.c", tmp_path / "c")
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.endswith("null ok\n"), (done.returncode, done.stdout)
    rows = [line.split() for line in done.stdout.splitlines()[:-1]]
    assert int(rows[0][2]) == C.sizeof(pkg.LinearConfig)
    names = [name for name, _ in pkg.LinearConfig._fields_]
    assert len(rows) - 1 == len(names)
    for row, name in zip(rows[1:], names):
        field = getattr(pkg.LinearConfig, name)
        assert (int(row[1]), int(row[2])) == (field.offset, field.size), (row, name)


@pytest.fixture(scope="module")
def cpp(tmp_path_factory):
    cuda = _cuda_include()
    libs = [f"-L{cuda.parent / 'lib64'}", "-lcudart", f"-Wl,-rpath,{cuda.parent / 'lib64'}"]
    return build("g++", ["-std=c++17", f"-isystem{cuda}"], ROOT / "tests" / "cpp_host" / "bounded_memory.cpp",
                 tmp_path_factory.mktemp("cpp") / "cpp", libs)


def test_the_component_types_compile_for_a_host(cpp):
    assert subprocess.run([str(cpp)]).returncode == 0


@pytest.mark.gpu
def test_a_host_program_runs_the_three_operators(cpp):
    done = subprocess.run([str(cpp), "step"], capture_output=True, text=True)
    assert done.returncode == 0 and "step ok" in done.stdout, (done.returncode, done.stdout, done.stderr)
