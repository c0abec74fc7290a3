"""The C++ layer's calls for serving in fewer bits (include/irontensor_b200.hpp): they compile and link everywhere, and their test
program (tests/cpp/quantized_test.cpp) passes on a GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "irontensor_b200")


def build(out, source="quantized_test.cpp"):
    from irontensor_b200 import _lib
    _lib.load()   # makes sure the shared library exists
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", source),
                    "-L", LIBDIR, "-lirontensor_b200", f"-Wl,-rpath,{LIBDIR}", "-o", out], check=True)


def test_compiles_and_links(tmp_path):
    build(str(tmp_path / "quantized_test"))


def test_members_that_do_not_fit_together_are_refused(tmp_path):
    exe = str(tmp_path / "quantized_refusals_test")
    build(exe, "quantized_refusals_test.cpp")
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "all checks passed" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_runs(tmp_path):
    exe = str(tmp_path / "quantized_test")
    build(exe)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "all checks passed" in out.stdout
