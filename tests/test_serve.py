"""rocket_serve.h on the CPU: what each entry refuses, before any device call, and the host paths (fd < 0)
against numpy: the cache's bytes exactly, attention and rotation within the rounding of the result."""
import ctypes as C

import numpy as np
import pytest

import rocketnpu as R
import serveforms as F

S = R.ROCKET_E_SHAPE


def rng(seed):
    return np.random.default_rng(0x52434C00 + seed)


def shape(*dims):
    return C.byref(R.Kv4Shape(*dims))


def test_cache_bytes(lib):
    for dims in ((1, 1, 32, 32, 1), (2, 3, 96, 160, 100), (4, 8, 128, 128, 4096), (1, 2, 256, 64, 33)):
        assert lib.rocket_kv4_bytes(shape(*dims)) == F.Cache(*dims).buf.size
    for dims in ((0, 1, 32, 32, 1), (1, 0, 32, 32, 1), (1, 1, 48, 32, 1), (1, 1, 32, 16, 1), (1, 1, 288, 32, 1), (1, 1, 32, 288, 1),
                 (1, 1, 32, 32, 0), (1, 1, 32, 32, (1 << 23) + 1), (256, 256, 32, 32, 32), (-1, -1, 32, 32, 32), (1, 1, 0, 32, 4)):
        assert lib.rocket_kv4_bytes(shape(*dims)) == 0
    assert lib.rocket_kv4_bytes(None) == 0


ROPE = dict(fd=-1, n_seq=2, n_tokens=3, n_head=4, n_kv=2, dim=64, rot=64, style=0, eps=1e-6, q_rs=256, k_rs=128)


def rope_call(lib, f32=False, null=(), weights=True, over=None, **kw):
    a = dict(ROPE, **kw)
    rows, dt = 6, np.float32 if f32 else np.float16
    o = dict(q=np.ones((rows, 1024), dt), k=np.ones((rows, 1024), dt), wq=np.ones(256, np.float16), wk=np.ones(256, np.float16),
             freq=np.ones(128, np.float32), pos=np.zeros(rows, np.int32), qo=np.full((rows, 1024), 7, np.float16), ko=np.full((rows, 1024), 7, np.float16))
    p = {n: None if n in null else R.ptr(x) for n, x in o.items()}
    if not weights:
        p["wq"] = p["wk"] = None
    if over:
        p[over[0]] = R.ptr(o[over[1]].ctypes.data + over[2])
    fn = lib.rocket_qk_norm_rope_f32in if f32 else lib.rocket_qk_norm_rope_fp16
    rc = fn(a["fd"], a["n_seq"], a["n_tokens"], a["n_head"], a["n_kv"], a["dim"], a["rot"], a["style"], a["eps"], p["q"], a["q_rs"], p["k"], a["k_rs"],
            p["wq"], p["wk"], p["freq"], p["pos"], p["qo"], p["ko"])
    if rc:
        assert (o["qo"] == 7).all() and (o["ko"] == 7).all()
    return rc


@pytest.mark.parametrize("f32", [False, True])
def test_rope_refusals(lib, f32):
    assert rope_call(lib, f32) == 0
    assert rope_call(lib, f32, weights=False) == 0 and rope_call(lib, f32, weights=False, eps=-1.0) == 0
    assert rope_call(lib, f32, rot=0, null=("freq", "pos")) == 0
    for kw in (dict(n_seq=0), dict(n_tokens=0), dict(n_head=0), dict(n_kv=0), dict(n_tokens=1 << 25), dict(n_head=1 << 16), dict(dim=48, rot=48),
               dict(dim=288), dict(dim=0, rot=0), dict(rot=60), dict(rot=72), dict(rot=-8), dict(style=2), dict(style=-1), dict(eps=float("nan")),
               dict(eps=-1.0), dict(q_rs=248), dict(k_rs=120), dict(q_rs=260), dict(k_rs=-128), dict(q_rs=(1 << 40) + 8),
               *(dict(null=(n,)) for n in ("q", "k", "freq", "pos", "qo", "ko")),
               dict(over=("qo", "q", 0)), dict(over=("ko", "q", 64)), dict(over=("qo", "wk", 0)), dict(over=("ko", "pos", 0)),
               dict(over=("ko", "qo", 32))):
        assert rope_call(lib, f32, **kw) == S, kw
    assert rope_call(lib, f32, fd=200) == R.ROCKET_E_DEVICE   # no such handle


@pytest.mark.parametrize("f32", [False, True])
def test_rope_too_many_rows(lib, f32):
    """2^24 rows, a workgroup each, are more threads than a launch takes: refused with the other bad counts, before the handle
    is looked at (no such handle, and nothing behind the addresses)."""
    fn = lib.rocket_qk_norm_rope_f32in if f32 else lib.rocket_qk_norm_rope_fp16
    q, k, qo, ko, freq, pos = (R.ptr(i << 44) for i in range(1, 7))
    call = lambda n: fn(200, 4096, n, 1, 1, 32, 32, 0, 1e-6, q, 32, k, 32, None, None, freq, pos, qo, ko)  # noqa: E731
    assert call(4096) == S and call(4095) == R.ROCKET_E_DEVICE


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dim,rot,pairs,eps,weighted", [(32, 32, False, 1e-6, True), (96, 64, True, 1e-5, True), (256, 128, False, 0.0, False),
                                                        (128, 8, True, -1.0, False), (64, 0, False, 1e-6, True)])
def test_rope_host(lib, f32, dim, rot, pairs, eps, weighted):
    g = rng(1)
    n_seq, T, nq, nk = 2, 3, 3, 1
    x = g.standard_normal((n_seq * T, (nq + 2 * nk) * dim)).astype(np.float32 if f32 else np.float16)
    w = F.f16(1 + 0.2 * g.standard_normal((2, dim))) if weighted else (None, None)
    freq = (10000.0 ** (-np.arange(max(1, rot // 2)) / max(1, rot // 2))).astype(np.float32)
    pos = np.array([0, 1, -5, 100, 70000, 2 ** 31 - 1], np.int32)
    qo, ko = np.empty((n_seq, nq, T, dim), np.float16), np.empty((n_seq, nk, T, dim), np.float16)
    fn = lib.rocket_qk_norm_rope_f32in if f32 else lib.rocket_qk_norm_rope_fp16
    assert fn(-1, n_seq, T, nq, nk, dim, rot, int(pairs), eps, R.ptr(x), x.shape[1], R.ptr(x.ctypes.data + nq * dim * x.itemsize), x.shape[1],
              R.ptr(w[0]), R.ptr(w[1]), R.ptr(freq), R.ptr(pos), R.ptr(qo), R.ptr(ko)) == 0
    for got, (want, tol) in ((qo, F.rope(x, nq, dim, rot, pairs, eps, w[0], freq, pos, n_seq)),
                             (ko, F.rope(x[:, nq * dim:], nk, dim, rot, pairs, eps, w[1], freq, pos, n_seq))):
        assert (np.abs(got.astype(np.float64) - want) <= tol).all()


DIMS = (3, 2, 64, 96, 40)


def kv4_call(lib, op, fd=-1, dims=DIMS, seq0=1, n_seq=2, T=2, lens=(5, 9), null=(), over=None, shift=0, **kw):
    a = dict(strides=(512, 256, 64) * 2, max_kv=40, heads=4, scale=0.1, cap=0.0, window=0, sinks=0)
    a.update(kw)
    o = dict(cache=np.zeros(1 << 20, np.uint8), K=np.ones(1 << 14, np.float16), V=np.ones(1 << 14, np.float16), Q=np.ones(1 << 14, np.float16),
             out=np.full(1 << 14, 7, np.float16), out2=np.full(1 << 14, 7, np.float16), lens=np.array(lens, np.int32))
    base = o["cache"].ctypes.data
    p = {n: None if n in null else R.ptr(x) for n, x in o.items()}
    if "cache" not in null:
        p["cache"] = R.ptr(base + (-base) % 16 + shift)
    if over:
        p[over[0]] = R.ptr(o[over[1]].ctypes.data + over[2])
    sh = None if "shape" in null else shape(*dims)
    if op == "append":
        k, v = a["strides"][:3], a["strides"][3:]
        rc = lib.rocket_kv4_append_fp16(fd, sh, p["cache"], seq0, n_seq, T, p["K"], *k, p["V"], *v, p["lens"])
    elif op == "read":
        rc = lib.rocket_kv4_read_fp16(fd, sh, p["cache"], seq0, n_seq, T, p["lens"], p["out"], p["out2"])
    else:
        rc = lib.rocket_kv4_attn_fp16(fd, sh, p["cache"], seq0, n_seq, T, a["max_kv"], a["heads"], a["scale"], a["cap"], a["window"], a["sinks"],
                                      p["Q"], p["lens"], p["out"])
    if rc:
        assert (o["out"] == 7).all() and not o["cache"].any()
    return rc


@pytest.mark.parametrize("op", ["append", "read", "attn"])
def test_kv4_refusals(lib, op):
    assert kv4_call(lib, op) == 0
    assert kv4_call(lib, op, lens=(0, -7)) == 0
    for kw in (dict(dims=(3, 2, 48, 96, 40)), dict(null=("shape",)), dict(null=("cache",)), dict(null=("lens",)), dict(seq0=-1), dict(seq0=2),
               dict(n_seq=0), dict(n_seq=4, seq0=0), dict(T=0), dict(T=(1 << 23) + 1), dict(shift=8)):
        assert kv4_call(lib, op, **kw) == S, kw
    assert kv4_call(lib, op, fd=200) == R.ROCKET_E_DEVICE
    if op == "append":
        for kw in (dict(null=("K",)), dict(null=("V",)), dict(strides=(512, 256, 60, 512, 256, 64)), dict(strides=(512, 256, 64, 512, -256, 64)),
                   dict(strides=(512, 256, 64, (1 << 40) + 8, 256, 64)), dict(lens=(5, 41)), dict(over=("K", "cache", 64)), dict(over=("lens", "cache", 64))):
            assert kv4_call(lib, op, **kw) == S, kw
        assert kv4_call(lib, op, lens=(5, 40)) == 0 and kv4_call(lib, op, strides=(0, 0, 0) * 2) == 0
    elif op == "read":
        assert kv4_call(lib, op, null=("out",)) == 0 and kv4_call(lib, op, null=("out", "out2")) == 0
        for kw in (dict(over=("out", "cache", 1024)), dict(over=("out2", "out", 64)), dict(over=("out", "lens", 0))):
            assert kv4_call(lib, op, **kw) == S, kw
    else:
        for kw in (dict(null=("Q",)), dict(null=("out",)), dict(max_kv=0), dict(max_kv=41), dict(heads=3), dict(heads=0), dict(heads=1 << 16), dict(window=-1),
                   dict(window=4, sinks=-1), dict(sinks=2), dict(scale=float("nan")), dict(cap=float("nan")), dict(lens=(5, 21), max_kv=20),
                   dict(over=("out", "Q", 128)), dict(over=("out", "cache", 2048)), dict(over=("out", "lens", 0))):
            assert kv4_call(lib, op, **kw) == S, kw


def test_cache_host(lib):
    """Bytes of appended rows, nothing else written, skipped and dropped positions, what non-finite inputs are stored
    as, and the values read back (one rounding of code * scale + minimum)."""
    g = rng(2)
    n_seq, H, dk, dv, cap = 3, 2, 64, 96, 40
    c = F.Cache(n_seq, H, dk, dv, cap, fill=0xAB)
    T = 4
    K, V = F.f16(g.standard_normal((2, T, H, dk))), F.f16(g.standard_normal((2, H, T, dv)) * 100)
    K[0, 1, 0, :32] = 3.5            # one value: scale 0
    K[0, 2, 1, 40] = -0.0
    V[1, 1, 0, :32] = np.linspace(-65504, 65504, 32)
    lens = np.array([6, 2], np.int32)   # the second sequence's first two tokens are padding
    buf = c.buf.copy()
    al = np.zeros(buf.size + 16, np.uint8)
    off = (-al.ctypes.data) % 16
    mem = al[off:off + buf.size]
    mem[:] = buf
    sh = R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_append_fp16(-1, C.byref(sh), R.ptr(mem), 1, 2, T, R.ptr(K), T * H * dk, dk, H * dk, R.ptr(V), H * T * dv, T * dv, dv, R.ptr(lens)) == 0
    for s in range(2):
        for t in range(T):
            j = lens[s] - T + t
            for h in range(H):
                if j >= 0:
                    c.put(s + 1, h, j, K[s, t, h], V[s, h, t])
    assert np.array_equal(mem, c.buf)
    k, v = c.rows()
    Ko, Vo = np.empty((2, H, T, dk), np.float16), np.empty((2, H, T, dv), np.float16)
    assert lib.rocket_kv4_read_fp16(-1, C.byref(sh), R.ptr(mem), 1, 2, T, R.ptr(lens), R.ptr(Ko), R.ptr(Vo)) == 0
    for s in range(2):
        at = lens[s] - T + np.arange(T)
        ok = at >= 0
        assert np.array_equal(Ko[s][:, ok], F.f16(k[s + 1][:, at[ok]])) and np.array_equal(Vo[s][:, ok], F.f16(v[s + 1][:, at[ok]]))
        assert not Ko[s][:, ~ok].any() and not Vo[s][:, ~ok].any()
    # infinities and NaN are stored as finite values
    K[0, 0, 0, :3] = np.inf, -np.inf, np.nan
    one = np.array([1], np.int32)
    assert lib.rocket_kv4_append_fp16(-1, C.byref(sh), R.ptr(mem), 0, 1, 1, R.ptr(K), 0, 0, 0, R.ptr(V), 0, 0, 0, R.ptr(one)) == 0
    x = K[0, 0, 0].copy()
    x[:3] = 65504, -65504, 0
    c.put(0, 0, 0, x, V[0, 0, 0])
    assert np.array_equal(c.parts(mem)[0][0, 0, 0], c.parts()[0][0, 0, 0]) and np.array_equal(c.parts(mem)[1][0, 0, 0], c.parts()[1][0, 0, 0])


@pytest.mark.parametrize("window,sinks,cap", [(0, 0, 0.0), (5, 2, 0.0), (1, 0, 20.0), (3, 9, 0.0)])
def test_attention_host(lib, window, sinks, cap):
    g = rng(3)
    n_seq, H, dk, dv, capacity, heads, T = 3, 2, 64, 32, 24, 4, 3
    c = F.Cache(n_seq, H, dk, dv, capacity, fill=0xFF)   # (scales of all ones are NaN: not to be reached)
    lens = np.array([20, 0, 2], np.int32)
    for s in range(n_seq):
        for h in range(H):
            for j in range(lens[s]):
                c.put(s, h, j, F.f16(g.standard_normal(dk)), F.f16(g.standard_normal(dv)))
    mem = np.zeros(c.buf.size + 16, np.uint8)
    mem = mem[(-mem.ctypes.data) % 16:][:c.buf.size]
    mem[:] = c.buf
    Q, out = F.f16(g.standard_normal((n_seq, heads, T, dk)) * 2), np.full((n_seq, heads, T, dv), 7, np.float16)
    sh = R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_attn_fp16(-1, C.byref(sh), R.ptr(mem), 0, n_seq, T, 20, heads, 0.125, cap, window, sinks, R.ptr(Q), R.ptr(lens), R.ptr(out)) == 0
    k, v = c.rows()
    for s in range(n_seq):
        n = max(1, lens[s])
        see = F.visible(lens[s], T, window, sinks, n)
        want, tol = F.attend(Q[s], k[s, :, :n], v[s, :, :n], see, 0.125, cap, False)
        assert (np.abs(out[s].astype(np.float64) - want) <= tol).all(), s
        assert not out[s][:, ~see.any(1)].any()


WIN = dict(fd=-1, T=3, n=7, stride=9, dk=32, dv=16, heads=4, kvh=2, scale=0.2, cap=0.0, window=3, sinks=1)


def win_call(lib, null=(), over=None, **kw):
    a = dict(WIN, **kw)
    o = dict(Q=np.ones(4096, np.float16), K=np.ones(4096, np.float16), V=np.ones(4096, np.float16), out=np.full(4096, 7, np.float16))
    p = {n: None if n in null else R.ptr(x) for n, x in o.items()}
    if over:
        p[over[0]] = R.ptr(o[over[1]].ctypes.data + over[2])
    rc = lib.rocket_flash_attn_window_fp16(a["fd"], a["T"], a["n"], a["stride"], a["dk"], a["dv"], a["heads"], a["kvh"], a["scale"], a["cap"], a["window"],
                                           a["sinks"], p["Q"], p["K"], p["V"], p["out"])
    if rc:
        assert (o["out"] == 7).all()
    return rc


def test_window_refusals(lib):
    assert win_call(lib) == 0 and win_call(lib, window=0, sinks=0) == 0
    for kw in (dict(T=0), dict(n=0), dict(stride=6), dict(stride=(1 << 22) + 1), dict(T=(1 << 23) + 1), dict(dk=48), dict(dk=288), dict(dv=24), dict(dv=272),
               dict(heads=3), dict(kvh=0), dict(heads=0), dict(window=-1), dict(sinks=-1), dict(window=0), dict(scale=float("nan")), dict(cap=float("nan")),
               *(dict(null=(n,)) for n in ("Q", "K", "V", "out")), *(dict(over=("out", n, 64)) for n in ("Q", "K", "V"))):
        assert win_call(lib, **kw) == S, kw
    assert win_call(lib, fd=200) == R.ROCKET_E_DEVICE


@pytest.mark.parametrize("T,n,window,sinks", [(1, 1, 0, 0), (3, 20, 4, 2), (5, 3, 2, 1), (2, 9, 100, 100)])
def test_window_host(lib, T, n, window, sinks):
    g = rng(4)
    heads, kvh, dk, dv, stride = 4, 2, 32, 48, n + 3
    Q, K, V = F.f16(g.standard_normal((heads, T, dk)) * 2), F.f16(g.standard_normal((kvh, stride, dk))), F.f16(g.standard_normal((kvh, dv, stride)))
    see = F.visible(n, T, window, sinks, stride)
    see[:, n:] = False
    K[:, ~see.any(0)], V[:, :, ~see.any(0)] = np.nan, np.inf
    out = np.full((heads, T, dv), 7, np.float16)
    assert lib.rocket_flash_attn_window_fp16(-1, T, n, stride, dk, dv, heads, kvh, 0.2, 0.0, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
    want, tol = F.attend(Q, K.astype(np.float64), V.astype(np.float64).transpose(0, 2, 1), see, 0.2, 0.0, False)
    assert (np.abs(out.astype(np.float64) - want) <= tol).all()


@pytest.mark.parametrize("x", [float("inf"), -float("inf"), 3e38])
def test_attention_refuses_scales_and_caps_past_fp32(lib, x):
    """An infinite scale or cap has no result but NaN; a scale whose log2 form is infinite has none on the GPU."""
    assert kv4_call(lib, "attn", scale=x) == S and win_call(lib, scale=x) == S
    want = 0 if x == 3e38 else S   # (a cap of that size is one that means none)
    assert kv4_call(lib, "attn", cap=x) == want and win_call(lib, cap=x) == want
