"""What the calls of rocket_fp8.h and rocket_layer.h launch, stage and take of a handle's scratch, captured and not, on the CPU:
tests/native/layer_check.cpp links the library's objects with a HIP runtime that has no device."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "rocket-userspace_amd")


def test_launches_and_staging(tmp_path):
    lib, src, cxx = os.path.join(PKG, "librocketnpu.a"), os.path.join(REPO, "tests", "native", "layer_check.cpp"), "/opt/rocm/llvm/bin/clang++"
    if not os.path.exists(cxx) or not os.path.exists(lib):
        pytest.skip("needs clang++ and the static library")
    exe = str(tmp_path / "layer_check")
    b = subprocess.run([cxx, "-std=c++17", "-O1", "-I", os.path.join(REPO, "include"), "-I", os.path.join(PKG, "csrc"), "-I/opt/rocm/include", src, lib, "-o", exe,
                        "-lm", "-lpthread"], capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stdout[-3000:] + b.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
