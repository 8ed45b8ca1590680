"""Every kernel that a product of rocket_fp8.h can launch, on sums that are exact: codes of small whole numbers and scales of powers of two, so that
every element has to be right to the bit, whatever the order of the sums. test_layer_tiles.py checks without a GPU that each case takes the
kernel that it stands under, and that there are no others."""
import pytest
import torch

import layerforms as F
from test_gpu_layer import DEV, F32, H16, dev, full, gen, split
from test_layer import p

pytestmark = pytest.mark.gpu

# The form as layertiles.py names it, and two calls (rows, K, N, and how many experts): K ends inside a block and rows of C are
# not aligned to four; and rows of C in whole stores.
CASES = {
    "128x128/2 fp16 sliced dense": [(5480, 9776, 90), (2845, 17424, 136)],
    "128x128/2 fp16 whole dense": [(8944, 1120, 430), (3076, 400, 1328)],
    "128x128/2 fp16 whole experts": [(4821, 1216, 782, 2), (3511, 400, 1168, 1)],
    "128x128/2 fp16 whole gathered": [(2445, 1104, 1930, 1), (5333, 416, 664, 8)],
    "128x128/2 fp32 sliced dense": [(4404, 2736, 502), (2993, 2592, 712)],
    "128x128/2 fp32 whole dense": [(2203, 1184, 955), (1785, 400, 1344)],
    "128x128/2 fp32 whole experts": [(537, 1360, 3830, 1), (2742, 416, 824, 1)],
    "128x128/2 fp32 whole gathered": [(5800, 1120, 323, 2), (1011, 416, 2288, 1)],
    "128x128/4 fp16 sliced dense": [(782, 9200, 827), (1872, 9664, 272)],
    "128x128/4 fp16 whole dense": [(2001, 1136, 1591), (7139, 944, 400)],
    "128x128/4 fp16 whole experts": [(9780, 1104, 265, 3), (15150, 784, 176, 2)],
    "128x128/4 fp16 whole gathered": [(8388, 1184, 369, 3), (14117, 928, 136, 3)],
    "256x256/2 fp16 sliced dense": [(10534, 17552, 129), (9046, 25104, 152)],
    "256x256/2 fp16 whole dense": [(1612, 1120, 5814), (1102, 432, 7672)],
    "256x256/2 fp16 whole experts": [(7224, 1136, 991, 16), (2378, 416, 3944, 1)],
    "256x256/2 fp16 whole gathered": [(7826, 1216, 1191, 3), (6775, 432, 1272, 6)],
    "32x64/4 fp16 sliced dense": [(86, 2000, 94), (67, 1808, 112)],
    "32x64/4 fp16 whole dense": [(50, 1120, 93), (59, 480, 96)],
    "32x64/4 fp16 whole experts": [(80, 1168, 141, 1), (80, 480, 104, 2)],
    "32x64/4 fp16 whole gathered": [(50, 1120, 109, 1), (52, 544, 96, 1)],
    "32x64/4 fp32 sliced dense": [(69, 9792, 99), (67, 9488, 96)],
    "32x64/4 fp32 whole dense": [(255, 1184, 313), (476, 1184, 128)],
    "32x64/4 fp32 whole experts": [(92, 1296, 95, 2), (50, 1168, 104, 1)],
    "32x64/4 fp32 whole gathered": [(67, 1392, 114, 1), (69, 1696, 96, 2)],
    "64x128/2 fp16 sliced dense": [(131, 12944, 5661), (2668, 7872, 72)],
    "64x128/2 fp16 whole dense": [(1975, 1104, 945), (782, 432, 1840)],
    "64x128/2 fp16 whole experts": [(5001, 1136, 283, 8), (6202, 416, 208, 3)],
    "64x128/2 fp16 whole gathered": [(5166, 1248, 343, 5), (490, 432, 3224, 1)],
    "64x128/4 fp16 sliced dense": [(1055, 8080, 194), (331, 12880, 456)],
    "64x128/4 fp16 whole dense": [(345, 1360, 3593), (389, 688, 3352)],
    "64x128/4 fp16 whole experts": [(6314, 1328, 201, 3), (2821, 736, 464, 3)],
    "64x128/4 fp16 whole gathered": [(2506, 1120, 526, 2), (1430, 992, 984, 1)],
    "64x64/4 fp16 sliced dense": [(539, 4624, 145), (567, 6032, 152)],
    "64x64/4 fp16 whole dense": [(2702, 1184, 213), (1588, 400, 520)],
    "64x64/4 fp16 whole experts": [(715, 1104, 861, 3), (3132, 464, 208, 3)],
    "64x64/4 fp16 whole gathered": [(587, 1136, 1067, 2), (3000, 416, 224, 1)],
    "64x64/4 fp32 sliced dense": [(98, 1248, 119), (112, 1088, 104)],
    "64x64/4 fp32 whole dense": [(592, 1104, 127), (114, 416, 96)],
    "64x64/4 fp32 whole experts": [(792, 1104, 105, 5), (115, 416, 96, 1)],
    "64x64/4 fp32 whole gathered": [(338, 1136, 153, 1), (116, 432, 104, 2)],
    "rows 1/4 fp16 whole dense": [(5, 1120, 8794), (5, 448, 8840)],
    "rows 1/4 fp16 whole experts": [(72, 1488, 478, 5), (251, 528, 144, 16)],
    "rows 1/4 fp16 whole gathered": [(224, 1936, 139, 16), (40, 448, 976, 3)],
    "rows 1/4 fp32 whole dense": [(2, 1376, 8257), (3, 400, 8336)],
    "rows 1/4 fp32 whole experts": [(88, 1616, 307, 8), (281, 448, 96, 28)],
    "rows 1/4 fp32 whole gathered": [(124, 1584, 229, 16), (241, 464, 152, 16)],
    "rows 1/6 fp16 whole dense": [(3, 1520, 90), (3, 400, 96)],
    "rows 1/6 fp16 whole experts": [(32, 1312, 197, 2), (32, 544, 128, 2)],
    "rows 1/6 fp16 whole gathered": [(29, 1104, 141, 3), (28, 464, 104, 5)],
    "rows 1/6 fp32 whole dense": [(4, 1184, 94), (1, 432, 96)],
    "rows 1/6 fp32 whole experts": [(24, 1680, 122, 2), (30, 400, 104, 3)],
    "rows 1/6 fp32 whole gathered": [(42, 1232, 95, 3), (26, 704, 120, 2)],
    "rows 2/4 fp16 whole dense": [(9, 1216, 17806), (13, 416, 19040)],
    "rows 2/4 fp16 whole experts": [(78, 1520, 737, 8), (116, 416, 368, 16)],
    "rows 2/4 fp16 whole gathered": [(34, 1856, 1374, 5), (57, 416, 1224, 5)],
    "rows 2/4 fp32 whole dense": [(9, 2016, 16477), (13, 400, 16744)],
    "rows 2/4 fp32 whole experts": [(253, 1856, 266, 16), (240, 448, 304, 16)],
    "rows 2/4 fp32 whole gathered": [(82, 1376, 442, 16), (229, 400, 320, 16)],
    "rows 2/6 fp16 whole dense": [(2, 1440, 4290), (5, 416, 4104)],
    "rows 2/6 fp16 whole experts": [(190, 1392, 218, 16), (24, 416, 1808, 2)],
    "rows 2/6 fp16 whole gathered": [(82, 1264, 485, 8), (107, 496, 400, 8)],
    "rows 2/6 fp32 whole dense": [(5, 1104, 4257), (2, 400, 4520)],
    "rows 2/6 fp32 whole experts": [(28, 1104, 1030, 5), (72, 416, 712, 5)],
    "rows 2/6 fp32 whole gathered": [(33, 1184, 1214, 3), (27, 400, 1952, 2)],
    "rows 4/4 fp16 whole experts": [(236, 1360, 583, 16), (213, 544, 640, 16)],
    "rows 4/4 fp16 whole gathered": [(78, 1424, 1422, 8), (723, 784, 136, 51)],
    "rows 4/4 fp16 whole dense": [(13, 1104, 25003), (9, 432, 25600)],
    "rows 4/4 fp32 whole dense": [(11, 1104, 25003), (16, 432, 25600)],
    "rows 4/4 fp32 whole experts": [(49, 1552, 2394, 5), (53, 448, 2248, 5)],
    "rows 4/4 fp32 whole gathered": [(212, 1104, 622, 16), (97, 432, 1328, 8)],
    "rows 4/6 fp16 whole dense": [(14, 1248, 8209), (12, 528, 8224)],
    "rows 4/6 fp16 whole experts": [(107, 1104, 770, 8), (200, 432, 416, 16)],
    "rows 4/6 fp16 whole gathered": [(42, 1120, 2409, 3), (25, 448, 3608, 2)],
    "rows 4/6 fp32 whole dense": [(15, 1168, 10335), (9, 400, 10352)],
    "rows 4/6 fp32 whole experts": [(56, 1392, 1427, 5), (199, 432, 424, 16)],
    "rows 4/6 fp32 whole gathered": [(481, 1120, 243, 32), (70, 496, 1208, 5)],
}


@pytest.mark.parametrize("form,case", [(f, c) for f, cases in CASES.items() for c in cases])
def test_exact(lib, fd, form, case):
    print(form, case, flush=True)
    M, K, N, *E = case
    dtype, gathered = H16 if "fp16" in form else F32, "gathered" in form
    g = gen(60)
    whole = lambda *s: F.encode(torch.randint(-3, 4, s, generator=g).float())  # noqa: E731
    two = lambda *s: 2.0 ** torch.randint(-1, 2, s, generator=g).float()  # noqa: E731
    A, sa, B, sb = (dev(t) for t in (whole(M, K), two(M, F.blocks(K)), whole(*E, N, K), two(*E, F.blocks(N), F.blocks(K))))
    out = full((M + 1, N), 7, dtype)
    if E:
        off = split(g, M, E[0], 0.2)
        src = torch.randint(-1, M + 1, (M,), generator=g, dtype=torch.int32) if gathered else None   # (both ends are no row)
        fn = lib.rocket_matmul_fp8_block_grouped_f16out if dtype == H16 else lib.rocket_matmul_fp8_block_grouped
        doff, dsrc = dev(off), dev(src)
        assert fn(fd, E[0], M, M, K, N, p(A), p(sa), p(dsrc), p(doff), p(B), p(sb), p(out)) == 0
        want, n = F.grouped(A, sa, dsrc, off, B, sb, M, F32)[0], int(off[-1])
    else:
        fn = lib.rocket_matmul_fp8_block_f16out if dtype == H16 else lib.rocket_matmul_fp8_block
        assert fn(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
        want, n = F.product(A, sa, B, sb, F32)[0], M
    assert 36 * K < 2 ** 22   # (products up to 9 and factors up to 4, in steps of 1/4: no sum in any order takes more than 24 bits)
    assert torch.equal(out[:n], want[:n].to(dtype))
    assert (out[n:] == 7).all()
