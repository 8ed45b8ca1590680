"""Which operands of rocket_serve.h's calls are used in place, on the CPU: tests/native/serve_check.cpp links the
library's objects with a HIP runtime that has no device and counts what the calls allocate, wait for and launch."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "rocket-userspace_amd")


def test_operands_in_place(tmp_path):
    lib = os.path.join(PKG, "librocketnpu.a")
    src = os.path.join(REPO, "tests", "native", "serve_check.cpp")
    cxx = "/opt/rocm/llvm/bin/clang++"
    if not os.path.exists(cxx) or not os.path.exists(lib) or not os.path.exists(src):
        pytest.skip("needs clang++ and the static library")
    exe = str(tmp_path / "serve_check")
    b = subprocess.run([cxx, "-std=c++17", "-O1", "-I", os.path.join(REPO, "include"), "-I", os.path.join(PKG, "csrc"),
                        "-I/opt/rocm/include", src, lib, "-o", exe,
                        "-lm", "-lpthread"], capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stdout[-3000:] + b.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
