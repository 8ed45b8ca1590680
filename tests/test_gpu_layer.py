"""rocket_fp8.h and rocket_layer.h on the GPU against layerforms.py (64 bits, which derives each bound): one row to many, sizes
around every tile, odd columns, the last part of a block, NaN codes, experts without rows and rows without experts,
strides, results that stay as they were, streams, captured calls that are replayed, and a layer of experts in a row."""
import ctypes as C
import math

import pytest
import torch

import layerforms as F
import rocketnpu as R
from test_layer import (EDGES, NORMS, ROUTES, codes, logits_of, norm_call, norm_check, norm_inputs, odd_rows, operands, p, quant, route_call, route_check, within)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H16, F32 = torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(0x52434F00 + seed)


def dev(x):
    return {n: dev(v) for n, v in x.items()} if isinstance(x, dict) else x.to(DEV) if torch.is_tensor(x) else x


def full(shape, value, dtype):
    t = torch.full(shape, value, dtype=dtype, device=DEV)
    torch.cuda.synchronize()
    return t


# ---- quantisation ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M,K,spare", [(1, 8, 0), (5, 128, 8), (17, 136, 0), (9, 1408, 24), (33, 3840, 0), (4, 65536, 0), (700, 264, 8)])
def test_quantise(lib, fd, M, K, spare, dtype):
    print("quantise", M, K, spare, dtype, flush=True)
    x = odd_rows(gen(1), M, K + spare, dtype)
    d = dev(x)
    q, s = full((M + 1, K), 7, torch.uint8), full((M + 1, F.blocks(K)), 7.0, F32)
    fn = lib.rocket_quantize_rows_fp8 if dtype == F32 else lib.rocket_quantize_rows_fp8_fp16
    assert fn(fd, M, K, p(d), d.stride(0), p(q), p(s)) == 0
    wq, ws = F.quantise(x[:, :K].float())
    assert torch.equal(s[:M].cpu(), ws) and F.same_codes(q[:M].cpu(), wq)
    assert (q[M] == 7).all() and (s[M] == 7).all()
    rc, hq, hs = quant(lib, fd, x, K)        # host operands
    assert rc == 0 and torch.equal(hs, ws) and F.same_codes(hq, wq)


def test_quantise_every_step(lib, fd):
    """Values at and next to every half between two codes, at scales of many exponents."""
    v = F.VALUES[:127]
    half = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, half, half * (1 + 2.0 ** -20), half * (1 - 2.0 ** -20)]).float()
    x = torch.nn.functional.pad(x, (0, -x.numel() % 127)).view(-1, 127)
    x = torch.cat([torch.full((x.shape[0], 1), 448.0), x], 1) * torch.tensor([1.0, -1.0]).repeat(64)
    x = torch.cat([x * 2.0 ** e for e in range(-90, 100, 7)])
    d, (M, K) = dev(x), x.shape
    q, s = full((M, K), 7, torch.uint8), full((M, 1), 7.0, F32)
    assert lib.rocket_quantize_rows_fp8(fd, M, K, p(d), K, p(q), p(s)) == 0
    wq, ws = F.quantise(x)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,n", [(1, 8, None), (37, 1408, 29), (5, 200, 0), (6, 256, 1 << 30)])
def test_quantise_gated(lib, fd, M, K, n, act, dtype):
    print("gated", M, K, n, act, dtype, flush=True)
    x = dev((torch.randn((M, 2 * K + 8), generator=gen(2)) * 4).to(dtype))
    up = x.data_ptr() + K * x.element_size()
    count = None if n is None else dev(torch.tensor([5, n], dtype=torch.int32))[1:]   # (4-byte aligned)
    q, s = full((M, K), 7, torch.uint8), full((M, F.blocks(K)), 7.0, F32)
    fn = lib.rocket_quantize_glu_fp8 if dtype == F32 else lib.rocket_quantize_glu_fp8_fp16
    code = dict(silu=R.ROCKET_ACTIVATION_SILU, gelu=R.ROCKET_ACTIVATION_GELU)[act]
    assert fn(fd, M, K, p(x), C.c_void_p(up), x.stride(0), code, p(count), p(q), p(s)) == 0
    done = M if n is None else min(M, n)
    want, tol = F.gated(act, x[:done, :K], x[:done, K:2 * K])
    if done:
        assert F.near_codes(q[:done], s[:done], want, tol + F.e32 * want.abs())
    assert (q[done:] == 7).all() and (s[done:] == 7).all()


# ---- products --------------------------------------------------------------------------

PRODUCTS = [(1, 16, 1), (1, 3840, 640), (2, 144, 7), (7, 4096, 130), (15, 272, 257), (16, 128, 128), (17, 1024, 100), (32, 640, 384), (33, 2080, 1000), (64, 16, 640),
            (65, 512, 129), (77, 2080, 1001), (128, 1152, 512), (129, 384, 255), (200, 4096, 256), (256, 256, 320), (257, 1040, 770), (300, 128, 2050), (512, 2048, 512),
            (1030, 528, 516), (5, 65536, 33), (130, 65536, 17),
            # the larger tiles and their slices of K, with rows and columns left over
            (1030, 192, 4100), (2050, 384, 1000), (2050, 1232, 257), (1500, 656, 1000), (3000, 944, 770), (3000, 1120, 4100), (2900, 1136, 4099), (3000, 464, 1030),
            (2050, 6832, 1000), (2050, 7520, 516), (1000, 7216, 513), (1500, 8608, 516), (2050, 3552, 257), (1000, 5152, 100), (17, 2432, 99), (700, 6960, 104), (200, 3088, 256), (24, 3088, 100),
            (512, 15360, 640), (300, 16384, 1024), (3000, 928, 1030), (3000, 9360, 257), (2050, 7952, 260), (2050, 8672, 1000), (70, 9136, 2560), (16, 1024, 9000),
            (13, 400, 40000)]


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_product(lib, fd, M, K, N, dtype):
    print("product", M, K, N, dtype, flush=True)
    A, sa, B, sb = dev(operands(gen(3), M, K, N)[0]), *(dev(t) for t in operands(gen(3), M, K, N)[1:])
    if dtype == H16:
        sa = sa * min(1.0, 300.0 / K)   # (sums stay inside fp16)
    out = full((M + 1, N), 7, dtype)
    fn = lib.rocket_matmul_fp8_block_f16out if dtype == H16 else lib.rocket_matmul_fp8_block
    assert fn(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
    want, tol = F.product(A, sa, B, sb, dtype)
    within(out[:M], want, tol)
    assert (out[M] == 7).all()


def test_product_is_exact_on_whole_numbers(lib, fd):
    """Codes of small whole numbers and scales of powers of two: every sum is exact, so every element has to be."""
    for M, K, N in ((3, 256, 40), (40, 400, 72), (300, 1024, 264)):
        g = gen(4)
        A, B = (F.encode(torch.randint(-3, 4, s, generator=g).float()) for s in ((M, K), (N, K)))
        sa, sb = (2.0 ** torch.randint(-2, 3, s, generator=g).float() for s in ((M, F.blocks(K)), (F.blocks(N), F.blocks(K))))
        A, B, sa, sb = dev(A), dev(B), dev(sa), dev(sb)
        want = F.product(A, sa, B, sb, F32)[0]
        out, half = full((M, N), 7, F32), full((M, N), 7, H16)
        assert lib.rocket_matmul_fp8_block(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
        assert lib.rocket_matmul_fp8_block_f16out(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(half)) == 0
        assert torch.equal(out.double(), want) and torch.equal(half, want.half())


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M", [2, 24, 140, 600])
def test_product_nan_and_overflow(lib, fd, M, dtype):
    """A NaN code reaches its row or column and nothing else, behind a last part of a block too; fp16 sums past fp16 are infinite."""
    K, N = 336, 136
    A, sa, B, sb = operands(gen(5), M, K, N)
    A[M - 1, 5], B[3, K - 1], sa[0] = 0x7f, 0xff, 1e5
    A, sa, B, sb = dev(A), dev(sa), dev(B), dev(sb)
    out = full((M, N), 7, dtype)
    fn = lib.rocket_matmul_fp8_block_f16out if dtype == H16 else lib.rocket_matmul_fp8_block
    assert fn(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[M - 1], bad[:, 3] = True, True
    want, tol = F.product(A, sa, B, sb, dtype)
    assert torch.equal(out.isnan(), bad)
    big = want.abs() > 65536 if dtype == H16 else torch.zeros_like(bad)
    ok = ~bad & ~big & (want.abs() < 65504 - tol if dtype == H16 else ~bad)
    within(out[ok], want[ok], tol[ok])
    assert out[big & ~bad & (want.abs() > 65536 + tol)].isinf().all()


def split(g, rows, E, empty=0.3):
    """Offsets of E experts over the rows, some without any."""
    w = torch.rand(E, generator=g) ** 3 * (torch.rand(E, generator=g) > empty)
    w[int(torch.randint(0, E, (1,), generator=g))] += 0.5
    n = torch.floor(w / w.sum() * rows).long()
    return torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]).to(torch.int32)


GROUPED = [  # experts, rows, rows of A (None: in order), K, N
    (1, 1, None, 128, 16), (8, 3, 2, 272, 40), (64, 96, 16, 512, 384), (64, 96, None, 400, 130), (5, 300, 70, 1024, 257), (16, 700, None, 144, 264),
    (1024, 64, 40, 128, 36), (130, 2000, 500, 256, 128), (3, 1500, 1500, 640, 516), (200, 40, 40, 2064, 64),
    (3, 3000, None, 1056, 4100), (3, 3001, 900, 1136, 4099), (3, 2050, None, 176, 2050), (3, 3000, 700, 816, 770), (3, 2050, None, 352, 1030), (3, 3000, 2000, 944, 516),
    (3, 2050, 300, 1296, 257), (3, 3000, 1500, 928, 1030), (3, 3000, None, 1264, 516), (9, 3000, 800, 160, 2560), (9, 129, 50, 80, 1000), (40, 200, None, 112, 2050),
]


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("case", GROUPED)
def test_grouped(lib, fd, case, dtype):
    E, rows, a_rows, K, N = case
    print("grouped", case, dtype, flush=True)
    g = gen(6)
    A, sa, B, sb = (dev(t) for t in operands(g, a_rows or rows, K, N, E))
    if dtype == H16:
        sa = sa * min(1.0, 300.0 / K)
    off = split(g, rows, E)
    src = None if a_rows is None else torch.randint(-1, a_rows + 1, (rows,), generator=g, dtype=torch.int32)   # (both ends are no row)
    out = full((rows + 1, N), math.nan, dtype)
    fn = lib.rocket_matmul_fp8_block_grouped_f16out if dtype == H16 else lib.rocket_matmul_fp8_block_grouped
    doff, dsrc = dev(off), dev(src)
    assert fn(fd, E, rows, A.shape[0], K, N, p(A), p(sa), p(dsrc), p(doff), p(B), p(sb), p(out)) == 0
    want, tol = F.grouped(A, sa, dsrc, off, B, sb, rows, dtype)
    n = int(off[-1])
    within(out[:n], want[:n], tol[:n])
    assert out[n:].isnan().all()


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("E,rows,K,N", [(64, 500, 512, 96), (8, 1500, 640, 516), (9, 3000, 160, 2560)])
def test_grouped_one_expert(lib, fd, E, rows, K, N, dtype):
    """All rows are one expert's, the same row of A again and again; sizes where an even share would be a few rows, and many."""
    g = gen(34)
    A, sa, B, sb = (dev(t) for t in operands(g, 3, K, N, E))
    if dtype == H16:
        sa = sa * min(1.0, 300.0 / K)
    for e in (0, E - 1):
        off = torch.tensor([0] * (e + 1) + [rows - 1] * (E - e), dtype=torch.int32)
        src = torch.full((rows,), 1, dtype=torch.int32)
        out = full((rows, N), math.nan, dtype)
        fn = lib.rocket_matmul_fp8_block_grouped_f16out if dtype == H16 else lib.rocket_matmul_fp8_block_grouped
        doff, dsrc = dev(off), dev(src)
        assert fn(fd, E, rows, 3, K, N, p(A), p(sa), p(dsrc), p(doff), p(B), p(sb), p(out)) == 0
        want, tol = F.product(A[1:2], sa[1:2], B[e], sb[e], dtype)
        within(out[:rows - 1], want.expand(rows - 1, N), tol.expand(rows - 1, N))
        assert out[rows - 1].isnan().all() and torch.equal(out[0].expand(rows - 1, N), out[:rows - 1])


def test_grouped_offsets_out_of_range(lib, fd):
    """Offsets far outside, and descending ones, write nothing outside of C; host results keep the rows that nothing computes."""
    E, rows, K, N = 6, 40, 128, 24
    A, sa, B, sb = (dev(t) for t in operands(gen(7), rows, K, N, E))
    for off in ([0, 2 ** 31 - 1, -2 ** 31, 5, 3, 70, 70], [-5, -4, 100, 100, 100, 100, 100], [40] * 7, [0] * 7, [7, 1, 9, 2, 30, 5, 2 ** 31 - 1]):
        mem, d = full((rows + 16, N), 7, F32), dev(torch.tensor(off, dtype=torch.int32))
        assert lib.rocket_matmul_fp8_block_grouped(fd, E, rows, rows, K, N, p(A), p(sa), None, p(d), p(B), p(sb), p(mem[8:])) == 0
        assert (mem[:8] == 7).all() and (mem[8 + rows:] == 7).all()
    host, off = torch.full((rows, N), 7.0), torch.tensor([0, 0, 3, 3, 3, 9, 11], dtype=torch.int32)
    assert lib.rocket_matmul_fp8_block_grouped(fd, E, rows, rows, K, N, p(A), p(sa), None, p(off), p(B), p(sb), p(host)) == 0
    want, tol = F.grouped(A, sa, None, off, B, sb, rows, F32)
    within(host[:11], want[:11].cpu(), tol[:11].cpu())
    assert (host[11:] == 7).all()


def shifted(t, by):
    """The tensor `by` bytes behind an aligned start, between guards."""
    n = t.numel() * t.element_size()
    mem = torch.full((by + n + 64,), 7, dtype=torch.uint8, device=DEV)
    view = torch.as_strided(mem[by:by + n].view(t.dtype), t.shape, t.contiguous().stride())
    view.copy_(t)
    return mem, view


@pytest.mark.parametrize("by", [4, 8, 12])
def test_unaligned_device_memory(lib, fd, by):
    """Operands and results in device memory at every multiple of four bytes, with nothing around a result touched."""
    M, K, N = 40, 400, 72
    A, sa, B, sb = operands(gen(30), M, K, N)
    keep = [shifted(dev(t), by) for t in (A, sa, B, sb)]
    A, sa, B, sb = (v for _, v in keep)
    for dtype, fn in ((F32, lib.rocket_matmul_fp8_block), (H16, lib.rocket_matmul_fp8_block_f16out)):
        mem, out = shifted(full((M, N), 0, dtype), by)
        torch.cuda.synchronize()
        assert fn(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(out)) == 0
        within(out, *F.product(A, sa, B, sb, dtype))
        assert (mem[:by] == 7).all() and (mem[-64:] == 7).all()
    x = odd_rows(gen(31), M, K, F32)
    _, d = shifted(dev(x), by)
    (mq, q), (ms, s) = shifted(full((M, K), 0, torch.uint8), by), shifted(full((M, F.blocks(K)), 0, F32), by)
    torch.cuda.synchronize()
    assert lib.rocket_quantize_rows_fp8(fd, M, K, p(d), K, p(q), p(s)) == 0
    wq, ws = F.quantise(x)
    assert torch.equal(s.cpu(), ws) and F.same_codes(q.cpu(), wq)
    assert all((m[:by] == 7).all() and (m[-64:] == 7).all() for m in (mq, ms))


@pytest.mark.parametrize("M,K,N", [(200, 4096, 256), (700, 6960, 104), (300, 16384, 1024)])
def test_product_captured(lib, M, K, N):
    """Products in slices of K: captured on a handle without scratch, then on one that has it, both replayed between eager calls."""
    fd, stream = lib.rocket_open(), torch.cuda.Stream()
    assert lib.rocket_hip_set_stream(fd, C.c_void_p(stream.cuda_stream)) == 0 and lib.rocket_hip_set_mode(fd, R.ROCKET_HIP_ASYNC | R.ROCKET_HIP_DEVICE_OPERANDS) == 0
    try:
        A, sa, B, sb = (dev(t) for t in operands(gen(32), M, K, N))
        sa = sa * min(1.0, 300.0 / K)
        outs = [full((M, N), 7, H16) for _ in range(3)]
        call = lambda o: lib.rocket_matmul_fp8_block_f16out(fd, M, K, N, p(A), p(sa), p(B), p(sb), p(o))  # noqa: E731
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                assert call(outs[i]) == 0
            graphs.append(g)
            assert call(outs[2]) == 0    # (eager: the handle's scratch from here on)
            stream.synchronize()
        want, tol = F.product(A, sa, B, sb, H16)
        for _ in range(3):
            for o in outs:
                o.fill_(7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for g in graphs:
                    g.replay()
            assert call(outs[2]) == 0
            stream.synchronize()
            for o in outs:
                within(o, want, tol)
            assert torch.equal(outs[1], outs[2])
        del graphs, g
    finally:
        lib.rocket_close(fd)


def test_weights_past_4_gib(lib, fd):
    """Experts whose weights lie past 2^32 bytes."""
    E, K, N, rows = 17, 16384, 16384, 6     # 4.25 GiB
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB")
    g = gen(8)
    A, sa = (dev(t) for t in operands(g, rows, K, 16)[:2])
    B = torch.zeros((E, N, K), dtype=torch.uint8, device=DEV)
    B[16] = dev(codes(g, N, K))
    sb = torch.ones((E, N // 128, K // 128), device=DEV) * 0.01
    off = dev(torch.tensor([0] * 10 + [2] * 7 + [6], dtype=torch.int32))
    out = full((rows, N), 7, F32)
    assert lib.rocket_matmul_fp8_block_grouped(fd, E, rows, rows, K, N, p(A), p(sa), None, p(off), p(B), p(sb), p(out)) == 0
    assert (out[:2] == 0).all()
    within(out[2:], *F.product(A[2:], sa[2:], B[16], sb[16], F32))


# ---- norms -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("case", NORMS + [(37, 3840, True, True, 10, (1e-6, 1e-6), True, ("h", "x", "q")), (3, 16384, True, True, 1, (1e-6, 1e-6), True, ("h", "x", "q")),
                                          (2, 8200, False, True, 0, (1e-6, 1e-6), True, ("h", "q")), (700, 520, True, True, 100, (1e-6, 1e-6), True, ("x", "q")),
                                          (5, 8192, False, True, 0, (-1.0, 1e-6), False, ("q",))])
def test_norm(lib, fd, case, dtype):
    M, H, post, pre, every, eps, y, outs = case
    print("norm", case, dtype, flush=True)
    t = dev(norm_inputs(gen(9), M, H, dtype, post, pre, every))
    wide = torch.cat([t["y"], torch.full((M, 16), math.nan, dtype=dtype, device=DEV)], 1)[:, :H]   # columns of wider rows
    rc, o = norm_call(lib, fd, dict(t, y=wide), every, eps, outs, y)
    assert rc == 0
    norm_check(t, o, every, eps, outs, y)
    h = t["h"].clone()
    if "h" in outs:   # in place: the same bits
        rc, o2 = norm_call(lib, fd, t, every, eps, outs, y, over_h=True)
        assert rc == 0 and all(torch.equal(o[n], o2[n]) for n in o)
        t["h"].copy_(h)


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M,H,k,shared", [(1, 8, 1, False), (16, 2048, 6, True), (5, 200, 32, False), (300, 1408, 8, True), (3, 16384, 2, True)])
def test_moe_norm(lib, fd, M, H, k, shared, dtype):
    print("moe norm", M, H, k, shared, dtype, flush=True)
    t = dev(norm_inputs(gen(10), M, H, dtype, True, True, 3, k, shared))
    rc, o = norm_call(lib, fd, t, 3, (1e-6, 1e-6))
    assert rc == 0
    norm_check(t, o, 3, (1e-6, 1e-6))


# ---- routing ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("case", ROUTES + [(64, 64, 6, dict()), (65, 60, 6, dict()), (257, 256, 8, dict(groups=8, best=2, top_groups=4, sigmoid=True, bias=True)), (100, 1024, 4, dict()),
                                           (1000, 3, 3, dict(renorm=False)), (33, 512, 10, dict(groups=16, best=1, top_groups=3))])
def test_route(lib, fd, case, dtype):
    M, n, k, kw = case
    print("route", case, dtype, flush=True)
    g = gen(11)
    x = dev(logits_of(g, M, n, dtype, 0.3 if n % 2 == 0 else 0.0))
    if dtype == H16:
        kw = dict(kw, active=dev((torch.arange(M) % 3 != 1).to(torch.uint8)))
    if kw.get("bias"):
        kw = dict(kw, bias=dev(torch.randn(n, generator=g) * 0.1))
    rc, o = route_call(lib, fd, x, k, **kw)
    assert rc == 0
    route_check(o, x, k, **kw)
    rc, o = route_call(lib, fd, x, k, plan=False, **kw)
    assert rc == 0
    route_check(o, x, k, plan=False, **kw)


@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 70])
@pytest.mark.parametrize("n", [1, 2, 16, 17, 64, 65, 128, 129, 250, 256, 257, 512, 513, 1024])
def test_route_sizes(lib, fd, n, M):
    """Every form of a token (rows of lanes, waves) at its smallest and largest count, results 4-byte aligned."""
    print("route sizes", M, n, flush=True)
    g, k = gen(33 + n), min(n, 7)
    x = dev(logits_of(g, M, n, F32, 0.2))
    groups = next(d for d in (8, 5, 3, 2, 1) if n % d == 0)
    kw = dict(sigmoid=M % 2 == 0, bias=dev(torch.randn(n, generator=g) * 0.1), groups=groups, best=1 + (n > 2 * groups), top_groups=(groups + 1) // 2)
    new = lambda *s, dtype: torch.full((math.prod(s) + 1,), 77, dtype=dtype, device=DEV)[1:].view(s)  # noqa: E731
    o = dict(ids=new(M, k, dtype=torch.int32), weight=new(M, k, dtype=F32), off=new(n + 1, dtype=torch.int32), src=new(M * k, dtype=torch.int32), slot=new(M, k, dtype=torch.int32))
    torch.cuda.synchronize()
    assert lib.rocket_moe_route_f32(fd, M, n, p(x), x.stride(0), R.ROCKET_ROUTE_SIGMOID if kw["sigmoid"] else R.ROCKET_ROUTE_SOFTMAX, p(kw["bias"]), groups, kw["best"], kw["top_groups"], k, 1,
                                    1.0, None, p(o["ids"]), p(o["weight"]), p(o["off"]), p(o["src"]), p(o["slot"])) == 0
    route_check(o, x, k, **kw)


@pytest.mark.parametrize("many", [1, 13])
@pytest.mark.parametrize("kw", [dict(), dict(sigmoid=True), dict(sigmoid=True, bias=True), dict(bias=True), dict(groups=4, best=2, top_groups=2),
                                dict(groups=2, best=1, top_groups=1, sigmoid=True, bias=True, renorm=False), dict(bias=math.nan), dict(bias=math.inf), dict(bias=-math.inf),
                                dict(groups=4, best=2, top_groups=2, sigmoid=True, bias=-math.inf)])
def test_route_edges(lib, fd, kw, many):
    x = dev(torch.tensor(EDGES).repeat(many, 1))
    if "bias" in kw:
        bias = torch.tensor([0.0, 0, 0.5, 0, -1, 0, 0, 0.25])
        bias[3] = bias[3] if kw["bias"] is True else kw["bias"]
        kw = dict(kw, bias=dev(bias))
    rc, o = route_call(lib, fd, x, 3, **kw)
    assert rc == 0
    route_check(o, x, 3, **kw)


def test_route_host_operands(lib, fd):
    x = logits_of(gen(12), 70, 40, F32, 0.2)
    kw = dict(active=(torch.arange(70) % 2).to(torch.uint8))
    rc, o = route_call(lib, fd, x, 4, **kw)
    assert rc == 0
    route_check(o, x, 4, **kw)


# ---- together --------------------------------------------------------------------------

class Layer:
    """A layer of experts as a program calls it, all on the device: norm, router product, routing, the gathered gate and up products,
    gated rows, the down products, and the weighted sum with the next norm."""

    def __init__(self, M, H, I, E, k, seed):
        g = gen(seed)
        self.M, self.H, self.I, self.E, self.k = M, H, I, E, k
        self.wr = dev((torch.randn((E, H), generator=g) * 0.05).half())
        q = lambda *s: F.quantise_weights(torch.randn(s, generator=g) * 0.05)  # noqa: E731
        (self.B1, self.s1), (self.B2, self.s2) = ((dev(t) for t in q(E, 2 * I, H)), (dev(t) for t in q(E, H, I)))
        self.w = dev((1 + 0.2 * torch.randn((2, H), generator=g)).half())
        new = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
        rows = M * k
        self.h, self.y, self.active = new(M, H, dtype=H16), new(M, H, dtype=H16), new(M, dtype=torch.uint8)
        self.h1, self.x, self.xq, self.xs = new(M, H, dtype=H16), new(M, H, dtype=H16), new(M, H, dtype=torch.uint8), new(M, F.blocks(H), dtype=F32)
        self.logits = new(M, E, dtype=F32)
        self.ids, self.weight, self.slot = new(M, k, dtype=torch.int32), new(M, k, dtype=F32), new(M, k, dtype=torch.int32)
        self.off, self.src = new(E + 1, dtype=torch.int32), new(rows, dtype=torch.int32)
        self.gu, self.aq, self.as_ = new(rows, 2 * I, dtype=H16), new(rows, I, dtype=torch.uint8), new(rows, F.blocks(I), dtype=F32)
        self.out, self.h2, self.x2 = new(rows, H, dtype=H16), new(M, H, dtype=H16), new(M, H, dtype=H16)
        torch.cuda.synchronize()

    def inputs(self, seed):
        g = gen(seed)
        self.h.copy_((torch.randn((self.M, self.H), generator=g) * 2).half())
        self.y.copy_(torch.randn((self.M, self.H), generator=g).half())
        self.active.copy_((torch.rand(self.M, generator=g) > 0.2).to(torch.uint8))
        torch.cuda.synchronize()

    def call(self, lib, fd):
        M, H, I, E, k, rows = self.M, self.H, self.I, self.E, self.k, self.M * self.k
        a = self
        calls = [
            lib.rocket_add_norm_fp16(fd, M, H, p(a.h), p(a.y), H, p(a.w[0]), 1e-6, None, 1, 1.0, p(a.w[1]), 1e-6, p(a.h1), p(a.x), p(a.xq), p(a.xs)),
            lib.rocket_matmul_fp16_f32out(fd, M, H, E, p(a.x), p(a.wr), p(a.logits)),
            lib.rocket_moe_route_f32(fd, M, E, p(a.logits), E, R.ROCKET_ROUTE_SOFTMAX, None, 1, 1, 1, k, 1, 1.0, p(a.active), p(a.ids), p(a.weight), p(a.off), p(a.src), p(a.slot)),
            lib.rocket_matmul_fp8_block_grouped_f16out(fd, E, rows, M, H, 2 * I, p(a.xq), p(a.xs), p(a.src), p(a.off), p(a.B1), p(a.s1), p(a.gu)),
            lib.rocket_quantize_glu_fp8_fp16(fd, rows, I, p(a.gu), C.c_void_p(a.gu.data_ptr() + 2 * I), 2 * I, R.ROCKET_ACTIVATION_SILU, C.c_void_p(a.off.data_ptr() + 4 * E), p(a.aq),
                                             p(a.as_)),
            lib.rocket_matmul_fp8_block_grouped_f16out(fd, E, rows, rows, I, H, p(a.aq), p(a.as_), None, p(a.off), p(a.B2), p(a.s2), p(a.out)),
            lib.rocket_moe_add_norm_fp16(fd, M, H, p(a.h1), rows, k, p(a.out), p(a.slot), p(a.weight), None, None, -1.0, None, 1, 1.0, p(a.w[0]), 1e-6, p(a.h2), p(a.x2), None, None),
        ]
        assert not any(calls), calls

    def check(self):
        """Each step against 64 bits on the step's own inputs."""
        a = self
        h, eh, x, ex = F.add_norm(a.h, a.y, a.w[0], 1e-6, None, 1, 1.0, a.w[1], 1e-6)
        within(a.h1, h, F.rounded(h, eh, H16))
        within(a.x, x, F.rounded(x, ex, H16))
        assert F.near_codes(a.xq, a.xs, x, ex)
        o = dict(ids=a.ids, weight=a.weight, off=a.off, src=a.src.clone(), slot=a.slot)
        n = int(a.off[-1])
        o["src"][n:] = 77
        route_check(o, a.logits, a.k, active=a.active)
        for out, (A, sa, src, B, s) in ((a.gu, (a.xq, a.xs, a.src, a.B1, a.s1)), (a.out, (a.aq, a.as_, None, a.B2, a.s2))):
            want, tol = F.grouped(A, sa, src, a.off, B, s, a.M * a.k, H16)
            within(out[:n], want[:n], tol[:n])
        want, tol = F.gated("silu", a.gu[:n, :a.I], a.gu[:n, a.I:])
        assert F.near_codes(a.aq[:n], a.as_[:n], want, tol + F.e32 * want.abs())
        h, eh, x, ex = F.add_norm(a.h1, a.out, None, -1.0, None, 1, 1.0, a.w[0], 1e-6, a.slot, a.weight)
        within(a.h2, h, F.rounded(h, eh, H16))
        within(a.x2, x, F.rounded(x, ex, H16))


@pytest.mark.parametrize("M", [4, 16, 72, 260])
def test_layer_of_experts(lib, fd, M):
    a = Layer(M, 512, 192, 16, 4, 13)
    a.inputs(14)
    a.call(lib, fd)
    a.check()
    first = a.x2.clone()
    a.call(lib, fd)                      # no order of anything changes a bit
    assert torch.equal(first, a.x2)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_dense_layer(lib, fd, M):
    """A layer without experts: norm to codes, gate and up, gated rows, down, and the norm behind in place; device and host memory."""
    K, I, H, g = 496, 384, 520, gen(35)
    (B1, s1), (B2, s2) = (F.quantise_weights(torch.randn(s, generator=g) * 0.05) for s in ((2 * I, K), (H, I)))
    w = (1 + 0.2 * torch.randn(K, generator=g)).half()
    h0, back = (torch.randn((M, K), generator=g) * 2).half(), torch.randn((M, H), generator=g).half()
    for put in (dev, lambda t: t.clone()):
        new = lambda *s, dtype: put(torch.zeros(s, dtype=dtype))  # noqa: E731
        b1, t1, b2, t2, wd, h, hb = (put(t) for t in (B1, s1, B2, s2, w, h0, back))
        xq, xs, gu = new(M, K, dtype=torch.uint8), new(M, F.blocks(K), dtype=F32), new(M, 2 * I, dtype=H16)
        aq, as_, y, x2 = new(M, I, dtype=torch.uint8), new(M, F.blocks(I), dtype=F32), new(M, H, dtype=H16), new(M, H, dtype=H16)
        torch.cuda.synchronize()
        up = C.c_void_p(gu.data_ptr() + 2 * I)
        assert lib.rocket_add_norm_fp16(fd, M, K, p(h), None, K, None, -1.0, None, 1, 1.0, p(wd), 1e-6, None, None, p(xq), p(xs)) == 0
        assert lib.rocket_matmul_fp8_block_f16out(fd, M, K, 2 * I, p(xq), p(xs), p(b1), p(t1), p(gu)) == 0
        assert lib.rocket_quantize_glu_fp8_fp16(fd, M, I, p(gu), up, 2 * I, R.ROCKET_ACTIVATION_GELU, None, p(aq), p(as_)) == 0
        assert lib.rocket_matmul_fp8_block_f16out(fd, M, I, H, p(aq), p(as_), p(b2), p(t2), p(y)) == 0
        assert lib.rocket_add_norm_fp16(fd, M, H, p(hb), p(y), H, None, -1.0, None, 1, 0.5, None, 1e-5, p(hb), p(x2), None, None) == 0
        xq, xs, gu, aq, as_, y, hb, x2 = (dev(t) for t in (xq, xs, gu, aq, as_, y, hb, x2))
        _, _, x, ex = F.add_norm(dev(h0), None, None, -1.0, None, 1, 1.0, dev(w), 1e-6)
        assert F.near_codes(xq, xs, x, ex)
        within(gu, *F.product(xq, xs, dev(B1), dev(s1), H16))
        want, tol = F.gated("gelu", gu[:, :I], gu[:, I:])
        assert F.near_codes(aq, as_, want, tol + F.e32 * want.abs())
        within(y, *F.product(aq, as_, dev(B2), dev(s2), H16))
        hn, eh, x, ex = F.add_norm(dev(back), y, None, -1.0, None, 1, 0.5, None, 1e-5)
        within(hb, hn, F.rounded(hn, eh, H16))
        within(x2, x, F.rounded(x, ex, H16))


@pytest.mark.parametrize("M", [8, 128])
def test_layer_captured(lib, M):
    """The layer as one graph, replayed with other inputs between eager calls of another layer on the same handle's stream."""
    fd = lib.rocket_open()
    stream = torch.cuda.Stream()
    assert lib.rocket_hip_set_stream(fd, C.c_void_p(stream.cuda_stream)) == 0 and lib.rocket_hip_set_mode(fd, R.ROCKET_HIP_ASYNC | R.ROCKET_HIP_DEVICE_OPERANDS) == 0
    try:
        a, other = Layer(M, 512, 192, 16, 4, 15), Layer(M + 72, 256, 128, 32, 2, 16)
        a.inputs(17)
        other.inputs(18)
        a.call(lib, fd)                  # (an eager call first: attributes and scratch)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a.call(lib, fd)
        for seed in (19, 20, 21, 22):
            a.inputs(seed)
            for t in (a.x, a.gu, a.out, a.h2, a.x2, a.ids):
                t.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            a.check()
            other.call(lib, fd)
            stream.synchronize()
            other.check()
        del graph
    finally:
        lib.rocket_close(fd)


def test_two_handles_at_once(lib):
    """Two handles on streams of their own, their calls interleaved without waits."""
    fds, streams = [lib.rocket_open() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    layers = [Layer(132, 512, 192, 16, 4, 23), Layer(132, 512, 192, 16, 4, 24)]
    try:
        for i in range(2):
            layers[i].inputs(25 + i)
            assert lib.rocket_hip_set_stream(fds[i], C.c_void_p(streams[i].cuda_stream)) == 0
            assert lib.rocket_hip_set_mode(fds[i], R.ROCKET_HIP_ASYNC | R.ROCKET_HIP_DEVICE_OPERANDS) == 0
        for _ in range(5):
            for i in range(2):
                layers[i].call(lib, fds[i])
        torch.cuda.synchronize()
        for a in layers:
            a.check()
    finally:
        for f in fds:
            lib.rocket_close(f)
