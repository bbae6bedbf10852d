"""The library's host code around its launches, without a GPU: the program
tests/cpp/host_calls_check.cpp stands in for the HIP runtime, refuses and counts
allocations and records the launches."""
import os
import shutil
import subprocess

import pytest

from molot_amd import lib as _lib

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="session")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    if cxx is None or not os.path.exists(os.path.join(rocm, "include/hip/hip_runtime.h")):
        pytest.skip("no C++ compiler, or no HIP headers")
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("native library not built")
    exe = str(tmp_path_factory.mktemp("host") / "host_calls_check")
    libdir = os.path.dirname(_lib.LIB_PATH)
    subprocess.run([cxx, "-O1", "-std=c++17", "-pthread", "-D__HIP_PLATFORM_AMD__",
                    "-isystem", os.path.join(rocm, "include"), "-I" + os.path.join(ROOT, "include"),
                    os.path.join(HERE, "cpp", "host_calls_check.cpp"), "-o", exe,
                    "-L" + libdir, "-lmolot_amd", "-Wl,-rpath," + libdir,
                    "-Wl,-rpath-link," + os.path.join(rocm, "lib")], check=True)
    return exe


@pytest.mark.parametrize("case", ["threads", "growth", "no_memory", "track", "table"])
def test_host_calls(program, case):
    r = subprocess.run([program, case], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "PASSED" in r.stdout, r.stdout[-4000:] + r.stderr
