"""test_layer_range.py's rows on the GPU, and products whose rows hold infinite groups or scales at the ends of their range."""
import math

import pytest
import torch

import layerforms as F
from test_gpu_layer import DEV, F32, H16, dev, full, gen
from test_layer import operands, p, quant
from test_layer_range import EPS, infinite_rows, run_ends, run_none, run_past

pytestmark = pytest.mark.gpu


def put(v):
    v = dev(v)
    torch.cuda.synchronize()
    return v


@pytest.mark.parametrize("eps", EPS)
@pytest.mark.parametrize("where", ["h", "y", "experts"])
@pytest.mark.parametrize("H", [72, 1032, 8200])
def test_norm_ends(lib, fd, H, where, eps):
    print("ends", H, where, eps, flush=True)
    run_ends(lib, fd, put, H, where, eps)


@pytest.mark.parametrize("dtype", [H16, F32])
def test_norm_of_nothing(lib, fd, dtype):
    run_none(lib, fd, put, dtype)


@pytest.mark.parametrize("dtype", [H16, F32])
def test_norm_past_fp16(lib, fd, dtype):
    run_past(lib, fd, put, dtype)


@pytest.mark.parametrize("dtype", [H16, F32])
def test_quantise_infinities(lib, fd, dtype):
    """An infinity makes its group NaN in every product, and no other row."""
    x = infinite_rows(dtype)
    wq, ws = F.quantise(x.float())
    d = put(x)
    q, s = full((5, 400), 7, torch.uint8), full((5, 4), 7.0, F32)
    fn = lib.rocket_quantize_rows_fp8 if dtype == F32 else lib.rocket_quantize_rows_fp8_fp16
    assert fn(fd, 5, 400, p(d), 400, p(q), p(s)) == 0
    assert torch.equal(s.cpu(), ws) and F.same_codes(q.cpu(), wq)
    for rows in (5, 100):
        at = torch.arange(rows) % 5
        A, sa = put(q[at.to(DEV)].contiguous()), put(s[at.to(DEV)].contiguous())
        _, _, B, sb = (put(t) for t in operands(gen(70), 1, 400, 72))
        for t, fn in ((F32, lib.rocket_matmul_fp8_block), (H16, lib.rocket_matmul_fp8_block_f16out)):
            out = full((rows, 72), 7, t)
            assert fn(fd, rows, 400, 72, p(A), p(sa), p(B), p(sb), p(out)) == 0
            assert torch.equal(out.isnan(), (at < 4)[:, None].expand(rows, 72).to(DEV))
