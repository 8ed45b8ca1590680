"""Rows of rocket_layer.h's norms at the ends of fp32, rows without a value and rows of infinities and NaN, and infinite groups of
rocket_quantize_rows_fp8, on the host paths; test_gpu_layer_range.py runs the same on the GPU."""
import math

import pytest
import torch

import layerforms as F
from test_layer import F32, H16, gen, norm_call, norm_check, quant

# The sizes of a row's values, from subnormal to the largest: their squares pass fp32 from 1.8e19 on, and are below it from 1e-23 on.
SIZES = [1e-44, 1e-40, 3e-37, 1e-30, 1e-22, 1e-18, 1e-10, 1e10, 1e17, 1.7e19, 1e22, 1e30, 3e37]
EPS = [0.0, 1e-38, 1e-6, 1e30]


def ends(g, H):
    """A row of each size, and rows with one large value among small ones."""
    h = torch.randn((len(SIZES), H), generator=g).double() * torch.tensor(SIZES, dtype=torch.float64)[:, None]
    h = h.clamp(-3.3e38, 3.3e38)
    mixed = torch.randn((4, H), generator=g).double()
    for i, big in enumerate((3e38, 1e20, 1e25, 1e12)):
        mixed[i, 3 + 2 * i] = big
    return torch.cat([h, mixed]).float()


def inputs(g, H, where, post):
    e = ends(g, H)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    t = dict(h=e if where == "h" else r(*e.shape) * 3, y=e if where == "y" else r(*e.shape), w_post=(1 + 0.3 * r(H)).to(H16) if post else None,
             w_pre=(1 + 0.3 * r(H)).to(H16), gate=r(1, H).to(H16))
    if where == "experts":   # rows of usual sizes, weights that are not (their products with the rows are normal numbers: those are rounded in fp32)
        t["y"], sizes = r(*e.shape), [1e-30, 1e-28, 1e-26, 1e-24, 1e-22, 1e-18, 1e-10, 1e10, 1e17, 1.7e19, 1e22, 1e30, 1e35, 1e-20, 1e-25, 1e20, 1e25]
        t["slot"] = torch.randint(0, len(e), (len(e), 2), generator=g, dtype=torch.int32)
        t["weight"] = (torch.rand((len(e), 2), generator=g).double() + 0.5).mul(torch.tensor(sizes, dtype=torch.float64)[:, None]).float()
    return t


def run_ends(lib, fd, put, H, where, eps):
    """`where`: "h", the norm behind of the residual rows; "y" and "experts", the norm of a block's result, which then is of
    size 1, or less by eps."""
    t = {n: None if v is None else put(v) for n, v in inputs(gen(40), H, where, where != "h").items()}
    e = (-1.0, eps) if where == "h" else (eps, 1e-6)
    rc, o = norm_call(lib, fd, t, 100, e, y=where != "h")
    assert rc == 0
    norm_check(t, o, 100, e, y=where != "h")


@pytest.mark.parametrize("eps", EPS)
@pytest.mark.parametrize("where", ["h", "y", "experts"])
@pytest.mark.parametrize("H", [72, 1032])
def test_norm_ends_host(lib, H, where, eps):
    run_ends(lib, -1, lambda v: v, H, where, eps)


def run_none(lib, fd, put, dtype):
    """Rows of zeros under eps 0 are 0 / 0; a row with an infinity is NaN there and 0 elsewhere; one with a NaN is NaN. Without a norm
    infinities stay, and their group of codes is NaN there under an infinite scale."""
    H = 264
    h = torch.randn((6, H), generator=gen(41)).to(dtype)
    h[0], h[1, 130], h[2, 5], h[3, 200], h[4, 7], h[4, 8] = 0.0, math.inf, -math.inf, math.nan, math.inf, math.inf
    one = dict(h=put(h), y=put(torch.zeros_like(h)), w_post=None, w_pre=None, gate=None)
    for eps in (0.0, 1e-6):
        rc, o = norm_call(lib, fd, one, 0, (-1.0, eps), y=False)
        assert rc == 0 and torch.equal(o["h"].cpu().nan_to_num(7.0), h.nan_to_num(7.0))
        x = o["x"].cpu()
        nan = torch.zeros((6, H), dtype=torch.bool)
        nan[0], nan[1, 130], nan[2, 5], nan[3], nan[4, 7], nan[4, 8] = eps == 0.0, True, True, True, True, True
        assert torch.equal(x.isnan(), nan) and (x[[0, 1, 2, 4]].nan_to_num(0.0) == 0).all() and x[5].isfinite().all()
        q, s = F.quantise(x[:5].float())
        assert F.same_codes(o["q"][:5].cpu() & 127, q & 127) and torch.equal(o["s"][:5].cpu(), s)   # (a 0 of either sign)
    # the same rows as a block's result: what is NaN spreads over the row by the next norm
    rc, o = norm_call(lib, fd, dict(one, h=one["y"], y=one["h"]), 0, (0.0, 1e-6))
    assert rc == 0 and torch.equal(o["h"].isnan().any(1), put(torch.tensor([True, True, True, True, True, False]))) and o["x"][:5].isnan().all()
    assert (o["h"][[1, 2, 4]].nan_to_num(0.0) == 0).all() and o["x"][5].isfinite().all()
    rc, o = norm_call(lib, fd, one, 0, (-1.0, -1.0), y=False)
    assert rc == 0 and torch.equal(o["x"].cpu().nan_to_num(7.0), h.half().nan_to_num(7.0))
    q, s = F.quantise(h.float())
    assert F.same_codes(o["q"].cpu(), q) and torch.equal(o["s"].cpu(), s) and s.isinf().sum() == 3


@pytest.mark.parametrize("dtype", [H16, F32])
def test_norm_of_nothing_host(lib, dtype):
    run_none(lib, -1, lambda v: v, dtype)


@pytest.mark.parametrize("dtype", [H16, F32])
def test_norm_past_fp16_host(lib, dtype):
    run_past(lib, -1, lambda v: v, dtype)


def run_past(lib, fd, put, dtype):
    """h' past fp16 is an infinity in fp16, x is of h' before it is rounded."""
    h = torch.full((2, 128), 60000.0).to(dtype)
    h[1, ::2] = -60000.0
    t = dict(h=put(h), y=put(h.clone()), w_post=None, w_pre=None, gate=None)
    rc, o = norm_call(lib, fd, t, 0, (-1.0, 0.0), alpha=1.0)
    assert rc == 0
    want = torch.full((2, 128), 120000.0)
    want[1, ::2] *= -1
    assert torch.equal(o["h"].cpu(), want.to(dtype)) and torch.equal(o["x"].cpu().float(), want.sign())
    assert torch.equal(F.decode(o["q"].cpu()), want.double().sign() * 448)


def infinite_rows(dtype):
    x = torch.randn((5, 400), generator=gen(42)).to(dtype)
    x[0, 3], x[1, 399], x[2, 128:256], x[3, 0], x[3, 1] = math.inf, -math.inf, math.inf, math.inf, math.nan
    return x


@pytest.mark.parametrize("dtype", [H16, F32])
def test_quantise_infinities_host(lib, dtype):
    x = infinite_rows(dtype)
    rc, q, s = quant(lib, -1, x, 400)
    wq, ws = F.quantise(x.float())
    assert rc == 0 and torch.equal(s, ws) and F.same_codes(q, wq) and ws.isinf().sum() == 4 and F.decode(wq).isnan().sum() == 1 + 1 + 128 + 2
