"""test_layer_range.py's rows on the GPU, and products whose rows hold infinite groups or scales at the ends of their range."""
import pytest
import torch

import layerforms as F
from test_gpu_layer import DEV, F32, H16, dev, full, gen
from test_layer import operands, p
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


@pytest.mark.parametrize("M,K,N", [(3, 272, 40), (70, 1392, 114), (255, 1184, 313), (2203, 1184, 955)])
@pytest.mark.parametrize("experts", [False, True])
def test_scales_at_their_ends(lib, fd, M, K, N, experts):
    """Products of scales of 2^-126 and of 2^127 give exact sums (whole numbers; steps of e4m3's smallest), and rows of zero codes give zeros."""
    g = gen(71)
    scale = lambda e, *s: torch.full(s, 2.0 ** e)  # noqa: E731
    for ea, eb, step in ((-70, -56, 1.0), (-20, -106, 1.0), (63, 64, 2.0 ** -9), (120, 7, 2.0 ** -9)):
        A, B = (F.encode(torch.randint(-3, 4, s, generator=g).float() * step) for s in ((M, K), (N, K)))
        A[1] = 0
        want = (F.decode(A).to(DEV) @ F.decode(B).to(DEV).t()) * 2.0 ** (ea + eb)
        A, B, sa, sb = put(A), put(B), put(scale(ea, M, F.blocks(K))), put(scale(eb, F.blocks(N), F.blocks(K)))
        out = full((M, N), 7, F32)
        if experts:
            off = put(torch.tensor([0, M], dtype=torch.int32))
            assert lib.rocket_matmul_fp8_block_grouped(fd, 1, M, M, K, N, p(A), p(sa), None, p(off), p(B), p(sb), p(out)) == 0
        else:
            assert lib.rocket_matmul_fp8_block(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
        assert torch.equal(out.double(), want) and (out[1] == 0).all()
