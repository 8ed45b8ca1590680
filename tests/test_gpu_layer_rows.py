"""Rows of an experts' product that have no source: zeros, whatever the expert's weights hold."""
import math

import pytest
import torch

import layerforms as F
from test_gpu_layer import DEV, F32, H16, dev, full, gen
from test_layer import operands, p, within

pytestmark = pytest.mark.gpu

# experts, rows, rows of A, K, N: the kernel of few rows, tiles of every size (results of 16 and of 32 bits), odd columns, K inside a block
SOURCES = [(8, 24, 5, 272, 40), (40, 200, 60, 2064, 515), (32, 640, 300, 1024, 1024), (60, 1200, 300, 2064, 515), (9, 3000, 800, 160, 2560), (3, 3000, 700, 816, 770),
           (3, 3001, 900, 1136, 4099)]


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("E,rows,a_rows,K,N", SOURCES)
def test_no_source_is_zeros(lib, fd, E, rows, a_rows, K, N, dtype):
    """Weights with NaN codes in one column and, for another expert, an infinite scale reach every row that has a source, and no other."""
    print("sources", E, rows, a_rows, K, N, dtype, flush=True)
    g = gen(50)
    A, sa, B, sb = operands(g, a_rows, K, N, E)
    if dtype == H16:
        sa = sa * min(1.0, 300.0 / K)   # (sums stay inside fp16)
    B[:, 3, K - 1] = 0x7f
    sb[1, :, 0] = math.inf
    off = (torch.arange(E + 1) * rows // E).to(torch.int32)
    src = torch.randint(0, a_rows, (rows,), generator=g, dtype=torch.int32)
    none = torch.rand(rows, generator=g) < 0.4
    src[none] = torch.where(torch.rand(int(none.sum()), generator=g) < 0.5, -1, a_rows).to(torch.int32)
    A, sa, B, sb, src, none, doff = (dev(t) for t in (A, sa, B, sb, src, none, off))
    out = full((rows, N), 7, dtype)
    fn = lib.rocket_matmul_fp8_block_grouped_f16out if dtype == H16 else lib.rocket_matmul_fp8_block_grouped
    assert fn(fd, E, rows, a_rows, K, N, p(A), p(sa), p(src), p(doff), p(B), p(sb), p(out)) == 0
    assert (out[none] == 0).all()
    want, tol = F.grouped(A, sa, src, off, B, sb, rows, dtype)
    fine = ~none[:, None] & want.isfinite()
    assert torch.equal(out.isfinite(), fine | none[:, None])
    within(out[fine], want[fine], tol[fine])
