"""Which kernels the products of rocket_fp8.h launch, without a GPU: tests/native/layer_tiles.cpp links the library's objects with a HIP runtime
that has no device and prints their names."""
import os
import re
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "rocket-userspace_amd")
CXX = "/opt/rocm/llvm/bin/clang++"
LIB = os.path.join(PKG, "librocketnpu.a")


def available():
    return os.path.exists(CXX) and os.path.exists(LIB)


def build(folder):
    exe, src = os.path.join(str(folder), "layer_tiles"), os.path.join(REPO, "tests", "native", "layer_tiles.cpp")
    b = subprocess.run([CXX, "-std=c++17", "-O1", "-I", os.path.join(REPO, "include"), "-I/opt/rocm/include", src, LIB, "-o", exe, "-lm", "-lpthread"],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stdout[-3000:] + b.stderr[-3000:]
    return exe


def call(f16, M, K, N, E=0, gathered=False):
    """A product as the program reads it; E 0: dense."""
    return int(f16), int(E > 0), int(gathered), E or 1, M, K, N


def forms(exe, calls):
    """Of each call (tile, result, slices, rows): "128x128/4" (rows, columns, slots of LDS) or "rows 4/6" (blocks of 16 weight rows, waves),
    "fp16" or "fp32", "sliced" or "whole", "dense", "experts" or "gathered"."""
    r = subprocess.run([exe], input="".join("%d %d %d %d %d %d %d\n" % c for c in calls), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    lines = r.stdout.splitlines()
    assert len(lines) == len(calls)
    out = []
    for (f16, grouped, gathered, *_), line in zip(calls, lines):
        *names, threads = line.split(";")
        t = re.search(r"k_gemm_fp8<.*Cfg<(\d+), (\d+), \d+, \d+, (\d+), .*>, (true|false), (true|false)>", names[0])
        w = re.search(r"k_rows_fp8<(\d+), (true|false)>", names[0])
        assert (t or w) and len(names) <= 2 and all("k_join_fp8" in n for n in names[1:]), line
        assert (t.group(5) if t else w.group(2)) == ("true" if f16 else "false") and (not t or t.group(4) != t.group(5)), line
        out.append(("%sx%s/%s" % t.group(1, 2, 3) if t else "rows %s/%d" % (w.group(1), int(threads) // 64), "fp16" if f16 else "fp32", "sliced" if names[1:] else "whole",
                    "gathered" if gathered else "experts" if grouped else "dense"))
    return out
