"""rocket_fp8.h and rocket_layer.h on the CPU: what each entry refuses, before any device call, and the host paths
(fd < 0) against layerforms.py: codes, choices and rows exactly, the rest within the rounding of the result."""
import math

import pytest
import torch

import layerforms as F
import rocketnpu as R

S = R.ROCKET_E_SHAPE
H16, F32 = torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(0x52434E00 + seed)


def within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3], want[bad][:3], tol[bad][:3])


def p(x):
    return None if x is None else R.ptr(x)


# ---- quantisation ----------------------------------------------------------------------

def quant(lib, fd, x, K, act=None, up=None, n_rows=None, fill=7):
    M = x.shape[0]
    q, s = torch.full((M, K), fill, dtype=torch.uint8), torch.full((M, F.blocks(K)), 7.0)
    f32 = x.dtype == F32
    if act is None:
        rc = (lib.rocket_quantize_rows_fp8 if f32 else lib.rocket_quantize_rows_fp8_fp16)(fd, M, K, p(x), x.stride(0), p(q), p(s))
    else:
        rc = (lib.rocket_quantize_glu_fp8 if f32 else lib.rocket_quantize_glu_fp8_fp16)(fd, M, K, p(x), p(up), x.stride(0), act, p(n_rows), p(q), p(s))
    return rc, q, s


def odd_rows(g, M, K, dtype):
    """Rows with groups of zeros, of subnormal and of the largest values, a NaN, and values at the halves between codes."""
    x = torch.randn((M, K), generator=g) * torch.exp(3 * torch.randn((M, 1), generator=g))
    x[0, :min(K, 128)] = 0.0
    if M > 1:
        x[1] = (torch.arange(K) % 61 - 30) * 28.0 / 2 ** (torch.arange(K) % 11)   # a maximum of 840, quotients on halves
        x[1, ::128] = 448.0
        x[1] = x[1].clamp(-448, 448)
    if M > 2:
        x[2] *= 2.0 ** -30 if dtype == H16 else 2.0 ** -130
    if M > 3:
        x[3, -1] = math.nan
        x[3, 0] = 65504.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M,K", [(1, 8), (5, 128), (4, 136), (7, 392)])
def test_quantise_host(lib, M, K, dtype):
    x = odd_rows(gen(1), M, K + 8, dtype)
    rc, q, s = quant(lib, -1, x, K)
    wq, ws = F.quantise(x[:, :K].float())
    assert rc == 0 and torch.equal(s, ws) and F.same_codes(q, wq)


def test_encode_is_nearest_even():
    """(the oracle's own rounding, against torch's conversion)"""
    v = torch.cat([torch.linspace(-448, 448, 40001), F.VALUES.nan_to_num(0).float(), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, -0.0, math.nan])])
    assert F.same_codes(F.encode(v), v.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_quantise_gated_host(lib, act):
    x = torch.randn((6, 2 * 200), generator=gen(2)) * 3
    code = dict(silu=R.ROCKET_ACTIVATION_SILU, gelu=R.ROCKET_ACTIVATION_GELU)[act]
    n = torch.tensor([4], dtype=torch.int32)
    rc, q, s = quant(lib, -1, x, 200, act=code, up=x.data_ptr() + 200 * 4, n_rows=n)
    want, tol = F.gated(act, x[:4, :200], x[:4, 200:])
    assert rc == 0 and F.near_codes(q[:4], s[:4], want, tol + F.e32 * want.abs())
    assert (q[4:] == 7).all() and (s[4:] == 7).all()
    n[0] = -5
    rc, q, s = quant(lib, -1, x, 200, act=code, up=x.data_ptr() + 200 * 4, n_rows=n)
    assert rc == 0 and (q == 7).all() and (s == 7).all()


def test_quantise_refusals(lib):
    x, q, s, n = torch.ones(4096), torch.full((4096,), 7, dtype=torch.uint8), torch.full((64,), 7.0), torch.ones(1, dtype=torch.int32)
    base = dict(fd=-1, M=2, K=256, a=x, rs=256, q=q, s=s)
    for kw in (dict(M=0), dict(M=1 << 25), dict(K=0), dict(K=4), dict(K=12), dict(K=65544, rs=65544), dict(rs=248), dict(rs=260), dict(rs=(1 << 39) + 8), dict(rs=-256), dict(M=1 << 20, rs=1 << 40),
               dict(a=None), dict(q=None), dict(s=None), dict(M=1 << 24, K=65536, rs=65536)):
        a = dict(base, **kw)
        for fn in (lib.rocket_quantize_rows_fp8, lib.rocket_quantize_rows_fp8_fp16):
            assert fn(a["fd"], a["M"], a["K"], p(a["a"]), a["rs"], p(a["q"]), p(a["s"])) == S, kw
        for fn in (lib.rocket_quantize_glu_fp8, lib.rocket_quantize_glu_fp8_fp16):
            assert fn(a["fd"], a["M"], a["K"], p(a["a"]), p(x), a["rs"], 3, p(n), p(a["q"]), p(a["s"])) == S, kw
    glu = lib.rocket_quantize_glu_fp8
    assert glu(-1, 2, 256, p(x), p(x), 256, 0, None, p(q), p(s)) == S and glu(-1, 2, 256, p(x), None, 256, 3, None, p(q), p(s)) == S
    for over in (dict(q=x), dict(s=x), dict(q=s)):
        a = dict(base, **over)
        assert lib.rocket_quantize_rows_fp8(-1, 2, 256, p(a["a"]), 256, p(a["q"]), p(a["s"])) == S
    assert glu(-1, 2, 256, p(x), p(x), 256, 3, p(s), p(q), p(s)) == S
    assert (q == 7).all() and (s == 7).all()
    assert lib.rocket_quantize_rows_fp8(999, 2, 256, p(x), 256, p(q), p(s)) == R.ROCKET_E_DEVICE


# ---- products --------------------------------------------------------------------------

def codes(g, *shape):
    """Codes of every exponent, no NaN."""
    q = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    return torch.where((q & 127) == 127, torch.zeros_like(q), q)


def operands(g, M, K, N, E=None):
    lots = () if E is None else (E,)
    scale = lambda *sh: torch.exp(torch.randn(sh, generator=g)) * 0.01  # noqa: E731
    return codes(g, M, K), scale(M, F.blocks(K)), codes(g, *lots, N, K), scale(*lots, F.blocks(N), F.blocks(K))


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (3, 144, 130), (5, 256, 257)])
def test_product_host(lib, M, K, N, dtype):
    A, sa, B, sb = operands(gen(3), M, K, N)
    C = torch.full((M, N), 7, dtype=dtype)
    fn = lib.rocket_matmul_fp8_block_f16out if dtype == H16 else lib.rocket_matmul_fp8_block
    assert fn(-1, M, K, N, p(A), p(sa), p(B), p(sb), p(C)) == 0
    within(C, *F.product(A, sa, B, sb, dtype))


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_host(lib, gather):
    g = gen(4)
    E, rows, K, N = 5, 11, 160, 40
    A, sa, B, sb = operands(g, 4 if gather else rows, K, N, E)
    off = torch.tensor([0, 3, 3, 4, 9, 9], dtype=torch.int32)
    src = torch.tensor([0, 3, 1, 2, -1, 4, 1, 1, 0, 99, 0], dtype=torch.int32) if gather else None
    C = torch.full((rows, N), math.nan)
    assert lib.rocket_matmul_fp8_block_grouped(-1, E, rows, A.shape[0], K, N, p(A), p(sa), p(src), p(off), p(B), p(sb), p(C)) == 0
    want, tol = F.grouped(A, sa, src, off, B, sb, rows, F32)
    assert C[9:].isnan().all()
    within(C[:9], want[:9], tol[:9])
    # offsets past the rows, and descending ones: nothing outside of C is written
    off[3:] = torch.tensor([50, -7, 2 ** 31 - 1])
    mem = torch.full((rows + 8, N), 7.0)
    assert lib.rocket_matmul_fp8_block_grouped(-1, E, rows, A.shape[0], K, N, p(A), p(sa), p(src), p(off), p(B), p(sb), p(mem)) == 0
    assert (mem[rows:] == 7).all()


def test_product_refusals(lib):
    x, o = torch.ones(1 << 14, dtype=torch.uint8), torch.full((4096,), 7.0)
    s, off = torch.ones(512), torch.zeros(16, dtype=torch.int32)
    base = dict(M=4, K=128, N=16, A=x, sa=s, B=x, sb=s, C=o)
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(K=8), dict(K=136), dict(K=65552), dict(M=1 << 25), dict(N=1 << 25), dict(A=None), dict(sa=None),
               dict(B=None), dict(sb=None), dict(C=None), dict(C=x), dict(C=s)):
        a = dict(base, **kw)
        for fn in (lib.rocket_matmul_fp8_block, lib.rocket_matmul_fp8_block_f16out):
            assert fn(-1, a["M"], a["K"], a["N"], p(a["A"]), p(a["sa"]), p(a["B"]), p(a["sb"]), p(a["C"])) == S, kw
        for fn in (lib.rocket_matmul_fp8_block_grouped, lib.rocket_matmul_fp8_block_grouped_f16out):
            assert fn(-1, 2, a["M"], max(a["M"], 1), a["K"], a["N"], p(a["A"]), p(a["sa"]), None, p(off), p(a["B"]), p(a["sb"]), p(a["C"])) == S, kw
    call = lambda E=2, rows=4, a_rows=4, src=None, o_=off: lib.rocket_matmul_fp8_block_grouped(  # noqa: E731
        -1, E, rows, a_rows, 128, 16, p(x), p(s), p(src), p(o_), p(x), p(s), p(o))
    assert call(E=0) == S and call(E=1025) == S and call(a_rows=3) == S and call(a_rows=0, src=off) == S and call(o_=None) == S
    assert call(a_rows=1 << 24) == S and call(o_=o) == S and call(src=o) == S
    assert (o == 7).all()
    assert lib.rocket_matmul_fp8_block(999, 4, 128, 16, p(x), p(s), p(x), p(s), p(o)) == R.ROCKET_E_DEVICE


# ---- norms -----------------------------------------------------------------------------

def norm_inputs(g, M, H, dtype, post, pre, every, k=0, shared=False):
    r = lambda *sh: torch.randn(sh, generator=g)  # noqa: E731
    t = dict(h=(r(M, H) * 3).to(dtype), y=(r(max(1, 2 * M if k else M), H)).to(dtype), w_post=(1 + 0.3 * r(H)).to(H16) if post else None,
             w_pre=(1 + 0.3 * r(H)).to(H16) if pre else None, gate=r(-(-M // every), H).to(H16) if every else None)
    if k:
        t["slot"] = torch.randint(-1, 2 * M + 1, (M, k), generator=g, dtype=torch.int32)   # (both ends are no row)
        t["slot"][-1] = -1
        t["weight"] = torch.rand((M, k), generator=g)
        t["weight"][t["slot"] < 0] = math.nan                                            # what is left out has no effect
        t["shared"] = r(M, H).to(dtype) if shared else None
    return t


def norm_call(lib, fd, t, every, eps, outs=("h", "x", "q"), y=True, alpha=0.75, over_h=False, new=torch.full):
    M, H = t["h"].shape
    f32, dev = t["h"].dtype == F32, t["h"].device
    o = dict(h=t["h"] if over_h else torch.full((M, H), 7, dtype=t["h"].dtype, device=dev), x=torch.full((M, H), 7, dtype=H16, device=dev),
             q=torch.full((M, H), 7, dtype=torch.uint8, device=dev), s=torch.full((M, F.blocks(H)), 7.0, device=dev))
    tail = (p(t["w_post"]), eps[0], p(t["gate"]), every or 1, alpha, p(t["w_pre"]), eps[1], p(o["h"]) if "h" in outs else None,
            p(o["x"]) if "x" in outs else None, p(o["q"]) if "q" in outs else None, p(o["s"]) if "q" in outs else None)
    if "slot" in t:
        fn = lib.rocket_moe_add_norm_f32 if f32 else lib.rocket_moe_add_norm_fp16
        rc = fn(fd, M, H, p(t["h"]), t["y"].shape[0], t["slot"].shape[1], p(t["y"]), p(t["slot"]), p(t["weight"]), p(t.get("shared")), *tail)
    else:
        fn = lib.rocket_add_norm_f32 if f32 else lib.rocket_add_norm_fp16
        rc = fn(fd, M, H, p(t["h"]), p(t["y"]) if y else None, t["y"].stride(0), *tail)
    return rc, o


def norm_check(t, o, every, eps, outs=("h", "x", "q"), y=True, alpha=0.75, h=None):
    """`h`: the residual rows as they were, where the call wrote over them."""
    h = t["h"] if h is None else h
    hn, eh, x, ex = F.add_norm(h, t["y"] if y else None, t["w_post"], eps[0], t["gate"], every or 1, alpha, t["w_pre"], eps[1],
                               *((t["slot"], t["weight"], t.get("shared")) if "slot" in t else ()))
    if "h" in outs:
        within(o["h"], hn, F.rounded(hn, eh, h.dtype))
    if "x" in outs:
        within(o["x"], x, F.rounded(x, ex, H16))
    if "q" in outs:
        assert F.near_codes(o["q"], o["s"], x, ex)


NORMS = [  # rows, H, post, pre, gate_every, eps, y, outs
    (1, 8, True, True, 0, (1e-6, 1e-6), True, ("h", "x", "q")), (5, 264, True, False, 2, (1e-5, 0.01), True, ("h", "q")),
    (3, 128, False, True, 1, (-1.0, 1e-6), True, ("x",)), (4, 136, False, False, 4, (1e-6, -1.0), True, ("h", "x", "q")),
    (2, 512, False, True, 0, (-1.0, 1e-6), False, ("x", "q")), (2, 1032, True, False, 3, (1e-6, -1.0), True, ("h",)),
]


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("case", NORMS)
def test_norm_host(lib, case, dtype):
    M, H, post, pre, every, eps, y, outs = case
    t = norm_inputs(gen(5), M, H, dtype, post, pre, every)
    rc, o = norm_call(lib, -1, t, every, eps, outs, y)
    assert rc == 0
    norm_check(t, o, every, eps, outs, y)


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("k,shared", [(1, False), (6, True)])
def test_moe_norm_host(lib, k, shared, dtype):
    t = norm_inputs(gen(6), 5, 200, dtype, True, True, 2, k, shared)
    h = t["h"].clone()
    rc, o = norm_call(lib, -1, t, 2, (1e-6, 1e-6), over_h=True)
    assert rc == 0
    norm_check(t, o, 2, (1e-6, 1e-6), h=h)


def test_norm_refusals(lib):
    x, w, o = torch.ones(8192, dtype=H16), torch.ones(8192, dtype=H16), [torch.full((8192,), 7, dtype=H16) for _ in range(4)]
    i = torch.zeros(64, dtype=torch.int32)
    wt = torch.ones(64)
    base = dict(M=4, H=128, h=x, y=x, rs=128, wp=w, ep=1e-6, g=w, ge=1, al=1.0, wq=w, eq=1e-6, ho=o[0], x=o[1], q=o[2], s=o[3], k=2, rows=8, slot=i, weight=wt, sh=x)
    both = [dict(M=0), dict(M=1 << 25), dict(H=0), dict(H=4), dict(H=132), dict(H=16392, rs=16392), dict(h=None), dict(ep=math.nan), dict(eq=math.nan),
            dict(al=math.inf), dict(al=math.nan), dict(ep=-1.0), dict(eq=-1.0), dict(ho=None, x=None, q=None, s=None), dict(q=None), dict(s=None), dict(ge=0),
            dict(ho=o[1]), dict(x=o[2]), dict(x=x), dict(q=w), dict(s=x), dict(ho=w), dict(ho=x)]   # (the last: in place, but h is y too)
    near = x[8:]   # a result a few values behind the rows that it would replace
    for kw in both + [dict(ho=near), dict(rs=120), dict(rs=132), dict(rs=(1 << 38) + 8), dict(M=1 << 20, rs=1 << 40)]:
        a = dict(base, **kw)
        for fn in (lib.rocket_add_norm_fp16, lib.rocket_add_norm_f32):
            assert fn(-1, a["M"], a["H"], p(a["h"]), p(a["y"]), a["rs"], p(a["wp"]), a["ep"], p(a["g"]), a["ge"], a["al"], p(a["wq"]), a["eq"], p(a["ho"]),
                      p(a["x"]), p(a["q"]), p(a["s"])) == S, kw
    for kw in both + [dict(k=0), dict(k=33), dict(rows=0), dict(rows=1 << 25), dict(y=None), dict(slot=None), dict(weight=None), dict(ho=i), dict(x=wt)]:
        a = dict(base, **kw)
        for fn in (lib.rocket_moe_add_norm_fp16, lib.rocket_moe_add_norm_f32):
            assert fn(-1, a["M"], a["H"], p(a["h"]), a["rows"], a["k"], p(a["y"]), p(a["slot"]), p(a["weight"]), p(a["sh"]), p(a["wp"]), a["ep"], p(a["g"]),
                      a["ge"], a["al"], p(a["wq"]), a["eq"], p(a["ho"]), p(a["x"]), p(a["q"]), p(a["s"])) == S, kw
    assert all((t == 7).all() for t in o) and (x == 1).all() and (w == 1).all()
    assert lib.rocket_add_norm_fp16(999, 4, 128, p(x), p(x), 128, None, -1.0, None, 1, 1.0, None, -1.0, p(o[0]), None, None, None) == R.ROCKET_E_DEVICE


# ---- routing ---------------------------------------------------------------------------

def route_call(lib, fd, logits, k, sigmoid=False, bias=None, groups=1, best=1, top_groups=1, renorm=True, scale=1.0, active=None, plan=True):
    M, n = logits.shape
    dev = logits.device
    new = lambda *sh, dtype=torch.int32: torch.full(sh, 77, dtype=dtype, device=dev)  # noqa: E731
    o = dict(ids=new(M, k), weight=new(M, k, dtype=F32), off=new(n + 1), src=new(M * k), slot=new(M, k))
    fn = lib.rocket_moe_route_f32 if logits.dtype == F32 else lib.rocket_moe_route_fp16
    rc = fn(fd, M, n, p(logits), logits.stride(0), int(sigmoid), p(bias), groups, best, top_groups, k, int(renorm), scale, p(active), p(o["ids"]), p(o["weight"]),
            *((p(o["off"]), p(o["src"]), p(o["slot"])) if plan else (None, None, None)))
    return rc, o


def route_check(o, logits, k, plan=True, **kw):
    kw = {n: v.cpu() if torch.is_tensor(v) else v for n, v in kw.items()}
    ids, weight, off, src, slot = F.route(logits.cpu(), k, **kw)
    o = {n: v.cpu() for n, v in o.items()}
    assert torch.equal(o["ids"].long(), ids)
    nan = weight.isnan()
    assert torch.equal(nan, o["weight"].isnan())
    within(o["weight"][~nan], weight[~nan], weight[~nan].abs() * (F.e32 + 1e-12) + 2.0 ** -150)
    if plan:
        rows = len(src)
        assert torch.equal(o["off"].long(), off) and torch.equal(o["slot"].long(), slot) and torch.equal(o["src"][:rows].long(), src)
        assert (o["src"][rows:] == 77).all()
    else:
        assert all((o[n] == 77).all() for n in ("off", "src", "slot"))


ROUTES = [  # tokens, experts, top_k, other arguments
    (1, 1, 1, dict()), (3, 8, 2, dict()), (5, 60, 6, dict(sigmoid=True, renorm=False, scale=2.5)), (2, 64, 32, dict(scale=-1.0)),
    (4, 64, 6, dict(groups=8, best=2, top_groups=3, sigmoid=True, bias=True)), (3, 128, 8, dict(groups=64, best=2, top_groups=5)),
    (6, 96, 4, dict(groups=3, best=1, top_groups=3, bias=True)), (2, 257, 8, dict(bias=True)), (3, 1024, 8, dict(groups=16, best=2, top_groups=4, sigmoid=True)),
]


def logits_of(g, M, n, dtype, off=0.0):
    x = torch.randn((M, n + 3), generator=g) * 2
    if off:
        x[torch.rand(x.shape, generator=g) < off] = -math.inf
    return x.to(dtype)[:, :n]


@pytest.mark.parametrize("dtype", [H16, F32])
@pytest.mark.parametrize("case", ROUTES)
def test_route_host(lib, case, dtype):
    M, n, k, kw = case
    g = gen(7)
    x = logits_of(g, M, n, dtype, 0.3 if n % 2 == 0 else 0.0)
    if dtype == H16:
        kw = dict(kw, active=(torch.arange(M) % 3 != 1).to(torch.uint8))
    if kw.get("bias"):
        kw = dict(kw, bias=torch.randn(n, generator=g) * 0.1)
    rc, o = route_call(lib, -1, x, k, **kw)
    assert rc == 0
    route_check(o, x, k, **kw)


EDGES = [  # a row of eight logits
    [0.0] * 8, [-math.inf] * 8, [-math.inf] * 5 + [1.0, 1.0, 0.5], [math.inf, 1, math.inf, 0, 0, 0, 0, 0], [math.nan, 1, 2, 3, -math.inf, 0, 0, 2],
    [math.nan] * 8, [0.5, 3.4028234663852886e38, math.inf, 3.4028234663852886e38, 0, 0, 0, 0], [math.nan, math.nan, 0, 1, 0, 0, 0, 0],
    [-3.4e38, 3.4e38, 0, -0.0, 0, 1e-45, -1e-45, 0], [-800.0, -801, -799, -800, -1e4, -1e5, -800, -799], [90.0, 91, 92, 40, 41, 42, 43, 90],
]


@pytest.mark.parametrize("kw", [dict(), dict(sigmoid=True), dict(sigmoid=True, bias=True), dict(bias=True), dict(groups=4, best=2, top_groups=2),
                                dict(groups=2, best=1, top_groups=1, sigmoid=True, bias=True, renorm=False), dict(bias=math.nan), dict(bias=math.inf), dict(bias=-math.inf),
                                dict(groups=4, best=2, top_groups=2, sigmoid=True, bias=-math.inf)])
def test_route_edges_host(lib, kw):
    x = torch.tensor(EDGES)
    if "bias" in kw:
        bias = torch.tensor([0.0, 0, 0.5, 0, -1, 0, 0, 0.25])
        bias[3] = bias[3] if kw["bias"] is True else kw["bias"]
        kw = dict(kw, bias=bias)
    rc, o = route_call(lib, -1, x, 3, **kw)
    assert rc == 0
    route_check(o, x, 3, **kw)
    rc, o = route_call(lib, -1, x, 3, plan=False, **kw)
    assert rc == 0
    route_check(o, x, 3, plan=False, **kw)


def test_route_refusals(lib):
    x, b, act = torch.ones(4096), torch.ones(64), torch.ones(8, dtype=torch.uint8)
    o = [torch.full((4096,), 7, dtype=torch.int32) for _ in range(5)]
    base = dict(M=8, E=64, x=x, rs=64, score=0, b=b, g=8, best=2, tg=4, k=6, scale=1.0, act=act, ids=o[0], w=o[1], off=o[2], src=o[3], slot=o[4])
    for kw in (dict(M=0), dict(M=1 << 25), dict(M=(1 << 24) // 6 + 1), dict(E=0), dict(E=1025, rs=1025), dict(E=60), dict(rs=63), dict(rs=(1 << 37) + 1), dict(M=1 << 20, k=1, rs=1 << 40), dict(score=2), dict(score=-1),
               dict(g=0), dict(g=65), dict(best=0), dict(best=3), dict(tg=0), dict(tg=9), dict(k=0), dict(k=33), dict(E=4, g=1, tg=1, k=5), dict(scale=math.nan),
               dict(scale=math.inf), dict(x=None), dict(ids=None), dict(w=None), dict(off=None), dict(src=None), dict(slot=None), dict(ids=o[1]), dict(w=x), dict(src=b),
               dict(slot=act), dict(off=o[4])):
        a = dict(base, **kw)
        for fn in (lib.rocket_moe_route_f32, lib.rocket_moe_route_fp16):
            assert fn(-1, a["M"], a["E"], p(a["x"]), a["rs"], a["score"], p(a["b"]), a["g"], a["best"], a["tg"], a["k"], 1, a["scale"], p(a["act"]), p(a["ids"]),
                      p(a["w"]), p(a["off"]), p(a["src"]), p(a["slot"])) == S, kw
    assert all((t == 7).all() for t in o)
    assert lib.rocket_moe_route_f32(999, 8, 64, p(x), 64, 0, None, 1, 1, 1, 6, 1, 1.0, None, p(o[0]), p(o[1]), None, None, None) == R.ROCKET_E_DEVICE
