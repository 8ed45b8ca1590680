"""Which kernels the products of rocket_fp8.h take by their sizes: each case of test_gpu_layer_tiles.py the one that it stands for, and no call of
any size one that has no case there. Without a GPU (layertiles.py)."""
import math
import random

import pytest

import layertiles as T
from test_gpu_layer_tiles import CASES


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if not T.available():
        pytest.skip("needs clang++ and the static library")
    return T.build(tmp_path_factory.mktemp("layer_tiles"))


def test_cases_take_their_kernels(exe):
    for form, cases in CASES.items():
        calls = [T.call("fp16" in form, *c, gathered="gathered" in form) for c in cases]
        got = [" ".join(f) for f in T.forms(exe, calls)]
        assert got == [form] * len(cases), (form, cases, got)


def test_no_other_kernels(exe):
    rng = random.Random(5)
    size = lambda lo, hi, step=1: max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step  # noqa: E731
    calls = []
    while len(calls) < 60000:
        f16, M, K, N, kind = rng.randrange(2), size(1, 20000), size(16, 65536, 16), size(1, 20000), rng.randrange(4)
        if kind == 0:
            calls.append(T.call(f16, M, K, N))
        elif kind == 1:   # few rows, many columns
            calls.append(T.call(f16, size(1, 40), K, size(3000, 1 << 22)))
        elif M * K < 1 << 31:
            calls.append(T.call(f16, M, K, N, rng.choice([1, 2, 8, size(1, 1024)]), kind == 3))
    forms = {" ".join(f) for f in T.forms(exe, calls)}
    assert forms <= set(CASES), forms - set(CASES)
    # (what only few sizes take may not be drawn: all but these forms are)
    assert len(set(CASES) - forms) <= 4, set(CASES) - forms
