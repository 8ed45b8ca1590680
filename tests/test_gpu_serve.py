"""rocket_serve.h on the GPU against numpy in 64 bits (serveforms.py, which derives each bound): every head
size, one token to long prompts, lengths that end inside every tile, windows and sinks at their edges, rows
that see no key, memory behind and between the visible keys that holds NaN, batches with idle places, captured
calls that are replayed with other lengths, and the operators in a row as a layer calls them."""
import ctypes as C

import numpy as np
import pytest

import rocketnpu as R
import serveforms as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rng(seed):
    return np.random.default_rng(0x52434D80 + seed)


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def near(got, want, tol):
    got = got.astype(np.float64)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3], tol[bad][:3])


# ---- norms and rotation ----------------------------------------------------------------

ROPE = [  # sequences, tokens, query heads, key heads, dim, rotated, pairs, eps, weights, spare columns
    (1, 1, 1, 1, 32, 32, False, 1e-6, True, 0), (5, 1, 16, 8, 256, 256, False, 1e-6, True, 8), (1, 67, 10, 2, 96, 64, True, 1e-5, True, 192),
    (3, 9, 5, 1, 160, 80, False, 1e-6, False, 0), (2, 33, 32, 8, 128, 128, True, -1.0, False, 1024), (1, 40, 3, 3, 224, 8, False, 1e-6, True, 0),
    (1, 7, 4, 4, 64, 0, False, 0.0, True, 0), (2, 3, 7, 5, 192, 184, True, 1e-6, True, 16), (1, 130, 40, 8, 128, 64, False, 1e-6, True, 0),
]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("case", ROPE)
def test_qk_norm_rope(lib, fd, case, f32):
    n_seq, T, nq, nk, d, rot, pairs, eps, weighted, spare = case
    print("rope", case, f32, flush=True)
    g = rng(1)
    rows = n_seq * T
    x = (g.standard_normal((rows, (nq + nk) * d + spare)) * 3).astype(np.float32 if f32 else np.float16)
    w = F.f16(1 + 0.3 * g.standard_normal((2, d))) if weighted else (None, None)
    freq = (10000.0 ** (-np.arange(max(4, rot // 2)) / max(1, rot // 2))).astype(np.float32)
    pos = g.integers(0, 1 << 20, rows).astype(np.int32)
    pos[: min(rows, 4)] = np.array([0, -3, 2 ** 31 - 1, -2 ** 31])[: min(rows, 4)]
    qo, ko = np.empty((n_seq, nq, T, d), np.float16), np.empty((n_seq, nk, T, d), np.float16)
    fn = lib.rocket_qk_norm_rope_f32in if f32 else lib.rocket_qk_norm_rope_fp16
    assert fn(fd, n_seq, T, nq, nk, d, rot, int(pairs), eps, R.ptr(x), x.shape[1], R.ptr(x.ctypes.data + nq * d * x.itemsize), x.shape[1],
              R.ptr(w[0]), R.ptr(w[1]), R.ptr(freq), R.ptr(pos), R.ptr(qo), R.ptr(ko)) == 0
    freq = freq[:rot // 2]
    near(qo, *F.rope(x, nq, d, rot, pairs, eps, w[0], freq, pos, n_seq))
    near(ko, *F.rope(x[:, nq * d:], nk, d, rot, pairs, eps, w[1], freq, pos, n_seq))


# ---- the cache -------------------------------------------------------------------------

@pytest.mark.parametrize("n_seq,seq0,places,H,dk,dv,cap,T,lens", [
    (1, 0, 1, 1, 32, 32, 1, 1, [1]), (3, 1, 2, 2, 96, 160, 45, 5, [45, 3]), (4, 0, 4, 8, 128, 128, 300, 1, [300, 0, 17, 1]),
    (1, 0, 1, 2, 256, 64, 700, 613, [613]), (2, 0, 2, 3, 64, 224, 64, 70, [64, 33]),
])
def test_cache(lib, fd, n_seq, seq0, places, H, dk, dv, cap, T, lens):
    """Every byte of the cache after an append, with what was there kept, and the values read back: exactly."""
    print("cache", n_seq, H, dk, dv, cap, T, lens, flush=True)
    g = rng(2)
    c = F.Cache(n_seq, H, dk, dv, cap)
    c.buf[:] = g.integers(0, 256, c.buf.size)
    mem = dev(c.buf)
    K, V = F.f16(g.standard_normal((places, T, H, dk)) * 4), F.f16(g.standard_normal((places, H, T, dv)) * 1000)
    K[0, -1, 0, :32] = 2.25
    V[0, 0, -1, :32] = np.where(np.arange(32) % 2, 6e-8, -6e-8)      # a range of subnormals
    V[0, -1, -1, -32:] = np.linspace(-65504, 65504, 32)
    L = np.array(lens, np.int32)
    for s in range(places):
        for t in range(T):
            j = L[s] - T + t
            if 0 <= j < cap:
                for h in range(H):
                    c.put(seq0 + s, h, j, K[s, t, h], V[s, h, t])
    sh = R.Kv4Shape(*c.dims)
    put = lib.rocket_kv4_append_fp16
    dK, dV, dL = dev(K), dev(V), dev(L)
    assert put(fd, C.byref(sh), R.ptr(mem), seq0, places, T, R.ptr(dK), T * H * dk, dk, H * dk, R.ptr(dV), H * T * dv, T * dv, dv, R.ptr(dL)) == 0
    assert np.array_equal(mem.cpu().numpy(), c.buf)
    if max(lens) <= cap:   # and from host operands
        mem2 = dev(c.buf)
        assert put(fd, C.byref(sh), R.ptr(mem2), seq0, places, T, R.ptr(K), T * H * dk, dk, H * dk, R.ptr(V), H * T * dv, T * dv, dv, R.ptr(L)) == 0
        assert np.array_equal(mem2.cpu().numpy(), c.buf)
    with np.errstate(all="ignore"):   # (unwritten scales are any bits)
        k, v = c.rows()
    Ko, Vo = np.full((places, H, T, dk), 7, np.float16), np.full((places, H, T, dv), 7, np.float16)
    assert lib.rocket_kv4_read_fp16(fd, C.byref(sh), R.ptr(mem), seq0, places, T, R.ptr(L), R.ptr(Ko), R.ptr(Vo)) == 0
    for s in range(places):
        at = L[s] - T + np.arange(T)
        ok = (at >= 0) & (at < cap)
        assert np.array_equal(Ko[s][:, ok], F.f16(k[seq0 + s][:, at[ok]])) and np.array_equal(Vo[s][:, ok], F.f16(v[seq0 + s][:, at[ok]]))
        assert not Ko[s][:, ~ok].any() and not Vo[s][:, ~ok].any()
        assert np.isfinite(Ko[s][:, ok]).all() and np.isfinite(Vo[s][:, ok]).all()
    V2 = np.full_like(Vo, 7)
    assert lib.rocket_kv4_read_fp16(fd, C.byref(sh), R.ptr(mem), seq0, places, T, R.ptr(L), None, R.ptr(V2)) == 0
    assert np.array_equal(V2, Vo)


def test_cache_codes_at_halves(lib, fd):
    """Quotients on and next to the halves between codes, where the reciprocal's code has to be the division's: multiples
    of a half step, fp16 neighbours of them, scales of every exponent, subnormal ones among them."""
    g = rng(4)
    T, H, d = 64, 4, 256
    x = g.integers(0, 31, (1, T, H, d)) / 2.0
    x[..., 0::32], x[..., 1::32] = 0, 15
    x = F.f16(x * 2.0 ** g.integers(-26, 12, (1, T, H, 1)))
    near = (x.view(np.uint16) + g.integers(-1, 2, x.shape)).astype(np.uint16).view(np.float16)
    K, V = x, F.f16(np.where(np.isfinite(near), near, x))
    any_bits = g.integers(0, 1 << 16, x.shape).astype(np.uint16).view(np.float16)
    for rows in (K, V, F.f16(np.where(np.isfinite(any_bits), any_bits, 1))):
        c = F.Cache(1, H, d, d, T)
        for t in range(T):
            for h in range(H):
                c.put(0, h, t, rows[0, t, h], rows[0, t, h])
        sh, mem, L, dR = R.Kv4Shape(*c.dims), dev(c.buf * 0), dev(np.array([T], np.int32)), dev(rows)
        assert lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, T, R.ptr(dR), 0, d, H * d, R.ptr(dR), 0, d, H * d, R.ptr(L)) == 0
        assert np.array_equal(mem.cpu().numpy(), c.buf)
        assert all(np.isfinite(F.f16(v)).all() for v in c.rows())


def test_cache_lengths_past_the_capacity(lib, fd):
    """Device lengths that no capacity holds, or far negative: the tokens are dropped, nothing else is touched."""
    c = F.Cache(3, 1, 32, 32, 40, fill=0x5A)
    mem, K = dev(c.buf), dev(F.f16(np.ones((3, 2, 32))))
    L = dev(np.array([43, 2 ** 31 - 1, -2 ** 31], np.int32))
    sh = R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), 0, 3, 2, R.ptr(K), 64, 0, 32, R.ptr(K), 64, 0, 32, R.ptr(L)) == 0
    assert np.array_equal(mem.cpu().numpy(), c.buf)
    assert lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(c.buf), 0, 3, 2, R.ptr(K), 64, 0, 32, R.ptr(K), 64, 0, 32, R.ptr(L)) == R.ROCKET_E_SHAPE


@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_cache_holds_finite_values(lib, fd, what):
    K = F.f16(rng(3).standard_normal((1, 1, 1, 64)))
    K[..., 5] = what
    c = F.Cache(1, 1, 64, 64, 8)
    sh, mem, L = R.Kv4Shape(*c.dims), dev(c.buf), np.array([1], np.int32)
    assert lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, 1, R.ptr(K), 0, 0, 0, R.ptr(K), 0, 0, 0, R.ptr(L)) == 0
    x = K[0, 0, 0].copy()
    x[5] = {np.inf: 65504, -np.inf: -65504}.get(what, 0)
    c.put(0, 0, 0, x, x)
    assert np.array_equal(mem.cpu().numpy(), c.buf)


# ---- attention over the cache ----------------------------------------------------------

KV4 = [  # heads, kv heads, dk, dv, tokens, lengths (the largest is max_kv), window, sinks, softcap
    (1, 1, 32, 32, 1, [1], 0, 0, 0.0), (2, 1, 64, 64, 1, [31, 32, 33], 0, 0, 0.0), (8, 2, 64, 96, 1, [257, 0, 5, 64], 0, 0, 0.0),
    (16, 8, 256, 256, 1, [1000], 0, 0, 0.0), (32, 8, 128, 128, 1, [700, 127, 128, 1, 0], 0, 0, 0.0), (5, 1, 96, 32, 3, [130, 2], 0, 0, 0.0),
    (4, 4, 160, 224, 2, [333], 0, 0, 30.0), (2, 2, 192, 128, 16, [100, 17], 0, 0, 0.0), (4, 2, 128, 128, 7, [300, 200], 0, 0, 0.0),
    (4, 2, 128, 64, 17, [300, 40], 0, 0, 0.0), (2, 1, 256, 256, 70, [200], 0, 0, 0.0), (8, 8, 64, 64, 130, [130, 300, 77], 0, 0, 0.0),
    (6, 2, 96, 160, 200, [900], 0, 0, 50.0), (4, 1, 128, 128, 129, [64, 513], 0, 0, 0.0),
    (4, 1, 64, 64, 9, [500, 36, 35], 0, 0, 0.0), (8, 2, 128, 128, 16, [300, 15], 50, 3, 0.0), (4, 2, 96, 64, 32, [700], 0, 0, 20.0), (2, 1, 128, 32, 24, [65, 24, 7], 9, 2, 0.0),
    (2, 1, 64, 64, 33, [300, 60], 0, 0, 0.0), (5, 1, 128, 128, 13, [400], 100, 0, 0.0), (2, 1, 160, 160, 16, [200, 31], 0, 0, 0.0), (2, 1, 256, 256, 17, [200, 31], 40, 4, 0.0),
    # two blocks of up to 32 rows of heads above 128
    (3, 1, 192, 160, 11, [333, 5], 0, 0, 0.0), (5, 1, 160, 256, 12, [400, 0, 33], 0, 0, 0.0), (4, 2, 256, 96, 20, [70, 200, 19], 50, 3, 20.0),
    (1, 1, 256, 256, 64, [64, 500], 0, 0, 0.0), (5, 1, 224, 224, 7, [2000], 0, 0, 0.0), (8, 2, 160, 160, 12, [5000, 700], 600, 9, 0.0),
    (1, 1, 64, 64, 100, [9000, 40, 130], 0, 0, 0.0), (2, 1, 256, 160, 70, [9001], 0, 0, 0.0),   # tiles in 17 to 32 shares
    # windows: inside a chunk, across chunks, one key, more than the keys; sinks that meet the window, and that lie past it
    (4, 2, 64, 64, 1, [500, 20], 64, 4, 0.0), (4, 2, 128, 128, 5, [411, 3, 70], 33, 1, 0.0), (2, 2, 256, 128, 1, [1025], 1, 0, 0.0),
    (8, 2, 128, 128, 40, [600, 90], 100, 5, 0.0), (2, 1, 64, 64, 300, [1000], 129, 70, 0.0), (3, 1, 64, 64, 33, [200, 100], 1000, 1000, 20.0),
    (2, 1, 128, 128, 300, [310], 64, 300, 0.0), (1, 1, 64, 64, 130, [4000], 17, 3, 0.0),
    (2, 1, 64, 64, 2, [70, 9], 2 ** 31 - 1, 2 ** 31 - 1, 0.0), (4, 1, 256, 256, 1, [4003], 1500, 33, 0.0),
]


def kv4_case(seed, heads, kvh, dk, dv, T, lens, uniform=False, spare=9):
    """A cache of random rows behind which (and in whose unused places) every byte is 0xFF: codes of 15, NaN scales."""
    g = rng(seed)
    cap = max(lens) + spare
    c = F.Cache(len(lens) + 2, kvh, dk, dv, cap, fill=0xFF)
    for s, n in enumerate(lens):
        if n:
            # dims of their own offset, as keys have after a rotation
            c.put_all(s + 1, F.f16(g.standard_normal((kvh, n, dk)) + 0.5 * g.standard_normal(dk)), F.f16(g.standard_normal((kvh, n, dv))))
    Q = F.f16(np.zeros((len(lens), heads, T, dk)) if uniform else g.standard_normal((len(lens), heads, T, dk)) * 1.5)
    return c, Q


def kv4_want(c, Q, lens, window, sinks, scale, cap):
    k, v = c.rows()
    T = Q.shape[2]
    for s, n in enumerate(lens):
        yield F.attend(Q[s], k[s + 1, :, :max(1, n)], v[s + 1, :, :max(1, n)], F.visible(n, T, window, sinks, max(1, n)), scale, cap, True)


@pytest.mark.parametrize("uniform", [False, True])
@pytest.mark.parametrize("case", KV4)
def test_kv4_attn(lib, fd, case, uniform):
    """Random queries; and queries of zero, whose results are the plain means of the visible values: a key too many or
    too few would show. Rows of other places and keys behind the lengths hold NaN scales."""
    heads, kvh, dk, dv, T, lens, window, sinks, cap = case
    print("kv4", case, uniform, flush=True)
    c, Q = kv4_case(10, heads, kvh, dk, dv, T, lens, uniform)
    scale = dk ** -0.5
    mem, dQ, dL = dev(c.buf), dev(Q), dev(np.array(lens, np.int32))
    out = dev(np.full((len(lens), heads, T, dv), 7, np.float16))
    sh = R.Kv4Shape(*c.dims)
    call = lambda o: lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 1, len(lens), T, max(lens), heads, scale, cap, window, sinks,  # noqa: E731
                                              R.ptr(dQ), R.ptr(dL), R.ptr(o))
    assert call(out) == 0
    got = out.cpu().numpy()
    for s, (want, tol) in enumerate(kv4_want(c, Q, lens, window, sinks, scale, cap)):
        near(got[s], want, tol)
        empty = ~F.visible(lens[s], T, window, sinks, max(1, lens[s])).any(1)
        assert not got[s][:, empty].any()
    again = dev(np.full((len(lens), heads, T, dv), 7, np.float16))
    assert call(again) == 0
    assert np.array_equal(again.cpu().numpy(), got)


def test_kv4_attn_larger_bound_and_host_operands(lib, fd):
    """max_kv above every length, lengths above max_kv (idle), host Q, lengths and results."""
    lens = [50, 7, 90]
    c, Q = kv4_case(11, 4, 2, 128, 128, 2, lens, spare=400)
    out = np.full((3, 4, 2, 128), 7, np.float16)
    L = np.array(lens, np.int32)
    sh, mem = R.Kv4Shape(*c.dims), dev(c.buf)
    call = lib.rocket_kv4_attn_fp16
    assert call(fd, C.byref(sh), R.ptr(mem), 1, 3, 2, 490, 4, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
    for s, (want, tol) in enumerate(kv4_want(c, Q, lens, 0, 0, 0.1, 0.0)):
        near(out[s], want, tol)
    assert call(fd, C.byref(sh), R.ptr(mem), 1, 3, 2, 60, 4, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == R.ROCKET_E_SHAPE
    first = out.copy()
    dL = dev(L)
    assert call(fd, C.byref(sh), R.ptr(mem), 1, 3, 2, 60, 4, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(dL), R.ptr(out)) == 0
    assert not out[2].any()
    for s, (want, tol) in list(enumerate(kv4_want(c, Q, lens, 0, 0, 0.1, 0.0)))[:2]:
        near(out[s], want, tol)
    assert first.any()


@pytest.mark.parametrize("T", [1, 9, 40])
def test_kv4_attn_short_lengths_under_a_long_bound(lib, fd, T):
    """A bound of 40000 keys over sequences of a few: the work is shared out by the lengths themselves."""
    lens = [1, 40, 700, 1500, 0]
    c, Q = kv4_case(15, 4, 2, 64, 64, T, lens, spare=40000)
    dQ, dL, sh, mem = dev(Q), dev(np.array(lens, np.int32)), R.Kv4Shape(*c.dims), dev(c.buf)
    out = dev(np.full((len(lens), 4, T, 64), 7, np.float16))
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 1, len(lens), T, 40000, 4, 0.125, 0.0, 0, 0, R.ptr(dQ), R.ptr(dL), R.ptr(out)) == 0
    got = out.cpu().numpy()
    k, v = c.rows()
    for s, n in enumerate(lens):
        m = max(1, n)
        near(got[s], *F.attend(Q[s], k[s + 1, :, :m], v[s + 1, :, :m], F.visible(n, T, 0, 0, m), 0.125, 0.0, True))


def test_kv4_attn_large_scores(lib, fd):
    """Scores in the thousands, growing and falling along the keys: the running maximum moves in every tile."""
    for T in (1, 40):
        for flip in (False, True):
            heads, kvh, d, n = 4, 2, 128, 600
            g = rng(12)
            c = F.Cache(3, kvh, d, d, n, fill=0xFF)
            up = np.linspace(0.1, 8, n)[::-1 if flip else 1]
            c.put_all(1, F.f16(np.abs(g.standard_normal((kvh, n, d))) * up[None, :, None]), F.f16(g.standard_normal((kvh, n, d))))
            Q = F.f16(np.abs(g.standard_normal((1, heads, T, d))) * 3)
            out, sh = np.full((1, heads, T, d), 7, np.float16), R.Kv4Shape(*c.dims)
            assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, d ** -0.5, 0.0, 0, 0, R.ptr(Q),
                                            R.ptr(np.array([n], np.int32)), R.ptr(out)) == 0
            (want, tol), = kv4_want(c, Q, [n], 0, 0, d ** -0.5, 0.0)
            near(out[0], want, tol)


@pytest.mark.parametrize("bits", [15.3, 20.5, 26.0])
@pytest.mark.parametrize("T", [3, 70, 65600])
def test_attn_many_small_weights(lib, fd, T, bits):
    """One key outweighs each of 2^17 others by 2^bits: together those count, and no weight may be lost for being small
    beside the largest; the prompt is so long that no workgroup's keys are split. Keys and values are exact in 4 bits. A
    token that sees v keys gets ((v - 1) w - 1) / ((v - 1) w + 1), off by what attend() allows for exact keys and values
    of 1: half a step of the result and of the weights, the scores' (within bits ln 2) fp32 steps, 2^-18."""
    print("small weights", T, bits, flush=True)
    n, d = 1 << 17, 32
    K, V = np.zeros((1, n, d), np.float16), np.ones((1, n, d), np.float16)
    K[0, 0, 0], V[0, 0] = 15, -1
    Q = np.zeros((1, T, d), np.float16)
    Q[..., 0] = 1
    scale = float(np.float32(bits * np.log(2) / 15))
    w = np.exp(-15 * scale) * (n - T + np.arange(T))
    want = np.repeat(((w - 1) / (w + 1))[None, :, None], d, 2)
    tol = np.abs(want) * F.U + 2 * np.expm1(2.0 ** -22 * 15 * scale + 2.0 ** -20) + F.U + 2.0 ** -18 + 2.0 ** -24
    c = F.Cache(1, 1, d, d, n)
    c.put_all(0, K, V)
    sh, mem, dQ, L, out = R.Kv4Shape(*c.dims), dev(c.buf), dev(Q), dev(np.array([n], np.int32)), np.empty((1, T, d), np.float16)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, T, n, 1, scale, 0.0, 0, 0, R.ptr(dQ), R.ptr(L), R.ptr(out)) == 0
    near(out, want, tol)
    dK, dV, out = dev(K), dev(V.transpose(0, 2, 1)), np.empty((1, T, d), np.float16)
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, 1, 1, scale, 0.0, 0, 0, R.ptr(dQ), R.ptr(dK), R.ptr(dV), R.ptr(out)) == 0
    near(out, want, tol)


@pytest.mark.parametrize("T,heads", [(1, 2), (9, 4), (20, 4), (70, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attn_of_equal_values(lib, fd, T, heads, d):
    """Keys whose values are all the same give that value, whatever their weights: a weight and its share of the sum round
    alike. In every 32 keys one weighs most and the others (1 + 0.98 2^-11) / 2 of it, which fp16 rounds down by nearly half a
    step, and the value is the largest fp16 below 2, whose half step is 2^-12 of it: a sum of unrounded weights is off by
    nearly twice that. With one of rounded weights 2^-18, for the fp32 steps, stands between the mean and the value, which is
    the result."""
    kvh, value = 2, 2047 / 1024
    scale = float(np.float32((1 - np.log2(1 + 0.98 * 2.0 ** -11)) * np.log(2) / 15))
    for n in (500, 3000):
        K, V, Q = np.zeros((kvh, n, d), np.float16), np.full((kvh, n, d), value, np.float16), np.zeros((heads, T, d), np.float16)
        K[:, ::32, 0], Q[..., 0] = 15, 1
        c = F.Cache(1, kvh, d, d, n)
        c.put_all(0, K, V)
        sh, out, L = R.Kv4Shape(*c.dims), np.empty((heads, T, d), np.float16), np.array([n], np.int32)
        assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 0, 1, T, n, heads, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
        assert (out == value).all()
        Vt = np.ascontiguousarray(V.transpose(0, 2, 1))
        assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(K), R.ptr(Vt), R.ptr(out)) == 0
        assert (out == value).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size,step", [(20.0, 15.6), (21.5, 15.6), (22.3, 15.6), (23.5, 15.8), (24.2, 16.0), (24.7, 16.0), (25.5, 16.0), (25.5, 28.0), (26.4, 40.0)])
def test_attn_scores_of_millions(lib, fd, size, step, sign):
    """Scores of up to 2^26.4 (in log2 units), where fp32 rounds them by up to 4, in 16 levels that grow along the keys by about
    what a weight may grow before the running maximum moves. Keys of a level are equal, so a token's result is the mean of the
    last level's values that it sees. A level weighs 2^-(step - 3 ulp) of the next one (each score off by a sum's ulp and a
    product's half), at most 1.6 of its keys to one of the last that a token sees; fp32 sums 2^-18."""
    g, kvh, n, d = rng(50), 2, 4000, 64
    level = np.arange(n) * 16 // n
    K, V = np.zeros((kvh, n, d), np.float16), F.f16(g.integers(-7, 8, (kvh, n, d)) / 8.0)
    K[:, :, 0], K[..., 32], K[..., 33] = 960, level, 15   # (exact in 4 bits)
    ulp = 2.0 ** (np.floor(size) - 23)
    tolerance = 2.0 ** -18 + 2 * 1.6 * 2.0 ** -(step - 3 * ulp)
    for T, heads in ((1, 2), (20, 4), (70, 2)):
        Q = np.zeros((heads, T, d), np.float16)
        Q[..., 0], Q[..., 32] = sign * 1000, 1000 * 960 * step / 2.0 ** size
        scale = float(np.float32(2.0 ** size * np.log(2) / (1000 * 960)))
        c = F.Cache(1, kvh, d, d, n)
        c.put_all(0, K, V)
        k, v = c.rows()
        assert np.array_equal(k[0, :, :n], K.astype(np.float64))
        sh, out, L = R.Kv4Shape(*c.dims), np.empty((heads, T, d), np.float16), np.array([n], np.int32)
        assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 0, 1, T, n, heads, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
        first = int(np.argmax(level == 15))

        def check(values):
            for h in range(heads):
                top = values[h // (heads // kvh), first:]
                want = (np.cumsum(top, 0) / np.arange(1, len(top) + 1)[:, None])[n - T - first:]
                near(out[h], want, np.abs(want) * F.U + tolerance)
        check(F.f16(v[0, :, :n]).astype(np.float64))
        Vt = np.ascontiguousarray(V.transpose(0, 2, 1))
        assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(K), R.ptr(Vt), R.ptr(out)) == 0
        check(V.astype(np.float64))


def exact_slack(c, s, n, Q, scale):
    """What fp32 sums of codes and minimums add to the bound of exact keys: their magnitudes, 15 scales and a minimum, take the
    place of the keys' and the values', 2^-21 of the scores' and 2^-20 of the values'."""
    _, ks, _, vs = (p.astype(np.float64) for p in c.parts())
    km = np.repeat(np.abs(ks[s, :, :n, :, 1]) + 15 * ks[s, :, :n, :, 0], 32, -1)
    q = np.abs(Q.astype(np.float64)).reshape(km.shape[0], -1, Q.shape[-1]) @ km.transpose(0, 2, 1)
    vm = (np.abs(vs[s, :, :n // 8, ..., 1]) + 15 * vs[s, :, :n // 8, ..., 0]).max()
    return 2 * np.expm1(2.0 ** -21 * abs(scale) * q.max()) * np.abs(c.rows()[1][s, :, :n]).max() + 2.0 ** -20 * vm


@pytest.mark.parametrize("T,heads,kvh", [(1, 16, 8), (5, 8, 2), (20, 4, 4), (40, 2, 2), (64, 2, 2), (70, 2, 2), (130, 4, 2)])
@pytest.mark.parametrize("d", [64, 96, 128, 160, 256])
def test_kv4_attn_multiplies_exact_keys_and_weights(lib, fd, T, heads, kvh, d):
    """Of roundings to fp16 there are the result's and the values', not the keys' and not the weights'. One alone is off by
    2^-11 sqrt(E[1 / m^2] / 3) = 2.07e-4 of its value (m, the mantissa, logarithmic in [1, 2): E = 3 / (8 ln 2)); two by sqrt 2
    of it, over all results, and the others would make it 2. And every result is within the bound of exact keys, whose rounded
    weights are rounded values here."""
    lens = [700, 333, 2000]
    c, Q = kv4_case(53, heads, kvh, d, d, T, lens)
    sh, scale, out = R.Kv4Shape(*c.dims), d ** -0.5, np.full((len(lens), heads, T, d), 7, np.float16)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, len(lens), T, max(lens), heads, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(np.array(lens, np.int32)),
                                    R.ptr(out)) == 0
    K, V = c.rows()
    off = size = 0.0
    for s, n in enumerate(lens):
        want, tol = F.attend(Q[s], K[s + 1, :, :n], V[s + 1, :, :n], F.visible(n, T, 0, 0, n), scale, 0.0, False)
        g = out[s].astype(np.float64) - want
        off, size = off + (g * g).sum(), size + (want * want).sum()
        near(out[s], want, tol + exact_slack(c, s + 1, n, Q[s], scale))
    assert np.sqrt(off / size) <= 1.05 * np.sqrt(2) * 2.07e-4


@pytest.mark.parametrize("T,heads", [(1, 2), (12, 2), (30, 2), (60, 2), (70, 4)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power,signed", [(-22, True), (-9, True), (12, True), (13, False)])
def test_kv4_attn_queries_of_any_size(lib, fd, T, heads, d, power, signed):
    """Queries of 2^-22 (subnormal ones) to 2^13, whose sums over a group's dims pass fp16 where they have one sign, under scales
    that bring the scores back: the bound of exact keys."""
    n, kvh = 300, 2
    c, Q = kv4_case(54, heads, kvh, d, d, T, [n])
    Q = F.f16((Q if signed else np.abs(Q)).astype(np.float64) * 2.0 ** power)
    sh, scale, out = R.Kv4Shape(*c.dims), d ** -0.5 * 2.0 ** -power, np.full((1, heads, T, d), 7, np.float16)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(np.array([n], np.int32)), R.ptr(out)) == 0
    K, V = c.rows()
    want, tol = F.attend(Q[0], K[1, :, :n], V[1, :, :n], F.visible(n, T, 0, 0, n), scale, 0.0, False)
    near(out[0], want, tol + exact_slack(c, 1, n, Q[0], scale))


@pytest.mark.parametrize("T,heads", [(1, 2), (12, 2), (30, 2), (60, 2), (70, 4)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_kv4_attn_keys_and_values_over_the_whole_range(lib, fd, T, heads, d):
    """Groups from -65504 to 65504, whose scale times 15 passes fp16, beside ordinary ones: there a key is off by up to half a
    step of half its code's product, 7.5 scales (the scores by as much times the query), and everything stays finite."""
    n, kvh, g = 300, 2, rng(55)
    K, V = F.f16(g.standard_normal((kvh, n, d))), F.f16(g.standard_normal((kvh, n, d)))
    wide = g.random((kvh, n, d // 32)) < 0.3
    at = np.repeat(wide, 32, -1)
    K[at] = F.f16(np.clip(g.standard_normal(at.sum()) * 30000, -65504, 65504))
    K[:, ::7, 0], K[:, ::7, 1] = 65504, -65504
    V[at] = F.f16(np.clip(g.standard_normal(at.sum()) * 30000, -65504, 65504))
    V[:, ::5, 2], V[:, ::5, 3] = 65504, -65504
    c = F.Cache(1, kvh, d, d, n)
    c.put_all(0, K, V)
    Q = F.f16(g.standard_normal((heads, T, d)) * 2.0 ** -4)
    scale, L, out = 2.0 ** -13 * d ** -0.5, np.array([n], np.int32), np.full((heads, T, d), 7, np.float16)
    sh = R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 0, 1, T, n, heads, scale, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
    k, v = c.rows()
    m = np.repeat(7.5 * c.parts()[1][0, :, :n, :, 0].astype(np.float64), 32, -1)
    q = (np.abs(Q.astype(np.float64)).reshape(kvh, -1, d) @ m.transpose(0, 2, 1)).max()
    want, tol = F.attend(Q, k[0, :, :n], v[0, :, :n], F.visible(n, T, 0, 0, n), scale, 0.0, True)
    near(out, want, tol + exact_slack(c, 0, n, Q, scale) + 2 * np.expm1(F.U * scale * q) * np.abs(v).max())


@pytest.mark.parametrize("T,heads", [(1, 2), (20, 4), (70, 2), (300, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attn_sums_are_fp32(lib, fd, T, heads, d):
    """Queries of zero weigh every key the same, with a power of two, so that results are plain means: half of one sequence's
    values average 1 + 0.98 2^-11 and the others are -1, whose sum is what a rounding of any share's mean to fp16 would lose. Off by
    half a step of the result and 2^-18 of the values, for fp32 sums over the keys and their shares."""
    g, kvh, n = rng(49), 2, 4000
    V = np.full((kvh, n, d), -1, np.float16)
    V[:, :n // 2] = 1
    V[:, g.permutation(n // 2)[:int(0.49 * (n // 2))]] = 1 + 2.0 ** -10
    K, Q = F.f16(g.standard_normal((kvh, n, d))), np.zeros((heads, T, d), np.float16)
    c = F.Cache(1, kvh, d, d, n)
    c.put_all(0, K, V)
    sh, out, L = R.Kv4Shape(*c.dims), np.empty((heads, T, d), np.float16), np.array([n], np.int32)
    seen = n - T + 1 + np.arange(T)
    want = (np.cumsum(V[0, :, 0].astype(np.float64))[seen - 1] / seen)[None, :, None]
    tol = np.abs(want) * F.U + 2.0 ** -18
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 0, 1, T, n, heads, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
    near(out, np.broadcast_to(want, out.shape), np.broadcast_to(tol, out.shape))
    Vt = np.ascontiguousarray(V.transpose(0, 2, 1))
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(K), R.ptr(Vt), R.ptr(out)) == 0
    near(out, np.broadcast_to(want, out.shape), np.broadcast_to(tol, out.shape))


@pytest.mark.parametrize("scale", [-0.2, 0.0, -0.0])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("T", [2, 40])
def test_attn_scale_not_positive(lib, fd, T, cap, scale):
    """A negative scale, and none (plain means of the visible values), over the cache and over fp16 keys."""
    heads, kvh, d, n, window, sinks = 4, 2, 64, 150, 70, 3
    c, Q = kv4_case(13, heads, kvh, d, d, T, [n])
    out, sh = np.full((1, heads, T, d), 7, np.float16), R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, scale, cap, window, sinks, R.ptr(Q),
                                    R.ptr(np.array([n], np.int32)), R.ptr(out)) == 0
    (want, tol), = kv4_want(c, Q, [n], window, sinks, scale, cap)
    near(out[0], want, tol)
    Q, K, V, see = win_case(14, heads, kvh, d, d, T, n, n, window, sinks)
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, cap, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
    near(out[0], *win_want(Q, K, V, see, scale, cap))


@pytest.mark.parametrize("cap", [-30.0, -4.0, 1e-3, 1e4])
@pytest.mark.parametrize("T,d", [(2, 64), (40, 64), (40, 256), (20, 160)])
def test_attn_soft_caps(lib, fd, T, d, cap):
    """c tanh(s / c) is even in c; caps that flatten every score, and that hardly bend one. (A cap's own bound: the
    exponential's and the reciprocal's 2^-22 of it.)"""
    heads, kvh, n, window, sinks, scale = 4, 2, 150, 70, 3, d ** -0.5
    c, Q = kv4_case(15, heads, kvh, d, d, T, [n])
    out, sh = np.full((1, heads, T, d), 7, np.float16), R.Kv4Shape(*c.dims)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, scale, cap, window, sinks, R.ptr(Q),
                                    R.ptr(np.array([n], np.int32)), R.ptr(out)) == 0
    (want, tol), = kv4_want(c, Q, [n], window, sinks, scale, cap)
    near(out[0], want, tol + 2 * np.expm1(abs(cap) * 2.0 ** -22) * np.abs(c.rows()[1][1, :, :n]).max())
    Q, K, V, see = win_case(16, heads, kvh, d, d, T, n, n, window, sinks)
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, cap, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
    want, tol = win_want(Q, K, V, see, scale, cap)
    near(out[0], want, tol + 2 * np.expm1(abs(cap) * 2.0 ** -22) * np.abs(V.astype(np.float64)).max())


# ---- windowed attention over fp16 keys -------------------------------------------------

WIN = [  # heads, kv heads, dk, dv, tokens, keys, stride, window, sinks, softcap
    (1, 1, 32, 16, 1, 1, 1, 0, 0, 0.0), (4, 2, 64, 64, 1, 63, 64, 0, 0, 0.0), (8, 2, 128, 128, 1, 1000, 1000, 0, 0, 0.0), (16, 8, 256, 256, 1, 777, 800, 0, 0, 0.0),
    (4, 4, 96, 80, 3, 130, 131, 0, 0, 30.0), (4, 2, 64, 64, 1, 500, 500, 64, 4, 0.0), (2, 2, 256, 128, 1, 1025, 1030, 1, 0, 0.0), (8, 2, 128, 128, 5, 411, 416, 33, 1, 0.0),
    (4, 1, 160, 224, 4, 600, 600, 100, 40, 0.0), (2, 1, 64, 64, 17, 300, 300, 0, 0, 0.0), (2, 1, 64, 64, 130, 130, 130, 0, 0, 0.0), (4, 2, 128, 128, 200, 512, 512, 0, 0, 0.0),
    (2, 2, 256, 256, 129, 1000, 1001, 0, 0, 20.0), (4, 2, 64, 64, 300, 1000, 1024, 129, 70, 0.0), (2, 1, 128, 64, 257, 900, 904, 64, 3, 0.0), (3, 1, 192, 192, 140, 1111, 1111, 100, 0, 0.0),
    (2, 1, 128, 128, 300, 310, 310, 64, 300, 0.0), (2, 1, 64, 48, 200, 90, 96, 0, 0, 0.0), (2, 1, 64, 64, 150, 100, 100, 20, 2, 0.0), (1, 1, 64, 64, 130, 4000, 4000, 17, 3, 0.0),
    (2, 1, 64, 64, 20, 70, 72, 2 ** 31 - 1, 2 ** 31 - 1, 0.0), (4, 1, 256, 256, 1, 4003, 4003, 1500, 33, 0.0), (2, 1, 128, 128, 40, 5, 7, 3, 1, 0.0), (2, 1, 64, 64, 20, 3000, 3000, 2000, 1, 0.0),
    (4, 1, 64, 64, 9, 500, 500, 0, 0, 0.0), (8, 2, 128, 128, 8, 301, 301, 50, 3, 0.0), (4, 2, 96, 64, 16, 700, 700, 0, 0, 20.0), (2, 1, 64, 32, 24, 65, 70, 9, 2, 0.0),
    (5, 1, 64, 64, 13, 400, 400, 100, 0, 0.0), (4, 2, 128, 80, 15, 333, 333, 300, 1, 0.0), (2, 1, 256, 256, 16, 200, 203, 40, 4, 0.0), (2, 1, 160, 176, 9, 13, 13, 5, 1, 0.0),
    (2, 1, 128, 128, 70, 400, 401, 33, 5, 0.0), (4, 4, 256, 256, 33, 300, 300, 0, 0, 0.0),
    (1, 1, 64, 64, 100, 9000, 9000, 0, 0, 0.0), (2, 1, 256, 160, 70, 9001, 9003, 7000, 4, 0.0),
    # V^T rows that end at every place of a chunk
    *((2, 1, 64, 48, 33, n, n, 0, 0, 0.0) for n in range(185, 201)), (4, 2, 128, 128, 40, 203, 205, 64, 2, 0.0), (2, 1, 256, 192, 40, 195, 195, 0, 0, 0.0), (2, 1, 64, 64, 40, 9, 9, 0, 0, 0.0),
]


def win_case(seed, heads, kvh, dk, dv, T, n, stride, window, sinks, uniform=False):
    g = rng(seed)
    Q = F.f16(np.zeros((heads, T, dk)) if uniform else g.standard_normal((heads, T, dk)) * 1.5)
    K, V = F.f16(g.standard_normal((kvh, stride, dk))), F.f16(g.standard_normal((kvh, dv, stride)))
    see = F.visible(n, T, window, sinks, stride)
    see[:, n:] = False
    return Q, K, V, see


def win_want(Q, K, V, see, scale, cap):
    return F.attend(Q, K.astype(np.float64), V.astype(np.float64).transpose(0, 2, 1), see, scale, cap, False)


@pytest.mark.parametrize("kind", ["random", "uniform", "nan"])
@pytest.mark.parametrize("case", WIN)
def test_window_attn(lib, fd, case, kind):
    """Random queries; queries of zero, whose results are plain means of the visible values; and NaN and infinities in
    every key and value that no token sees."""
    heads, kvh, dk, dv, T, n, stride, window, sinks, cap = case
    print("window", case, kind, flush=True)
    Q, K, V, see = win_case(20, heads, kvh, dk, dv, T, n, stride, window, sinks, kind == "uniform")
    if kind == "nan":
        dead = ~see.any(0)
        K[:, dead], V[:, :, dead] = np.nan, np.inf
        V[:, ::2, dead] = np.nan
    scale = dk ** -0.5
    dQ, dK, dV = dev(Q), dev(K), dev(V)
    outs = []
    for _ in range(2):
        out = dev(np.full((heads, T, dv), 7, np.float16))
        assert lib.rocket_flash_attn_window_fp16(fd, T, n, stride, dk, dv, heads, kvh, scale, cap, window, sinks, R.ptr(dQ), R.ptr(dK), R.ptr(dV), R.ptr(out)) == 0
        outs.append(out.cpu().numpy())
    near(outs[0], *win_want(Q, K, V, see, scale, cap))
    assert not outs[0][:, ~see.any(1)].any()
    assert np.array_equal(*outs)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("T,n,window,sinks", [(5, 200, 30, 2), (130, 400, 50, 3), (130, 403, 50, 3), (16, 333, 0, 0), (30, 333, 100, 1)])
def test_window_attn_values_that_some_tokens_see(lib, fd, T, n, window, sinks, d):
    """An infinite value reaches the tokens that see its key, and no other (0 times it would be NaN)."""
    heads, kvh = 2, 1
    Q, K, V, see = win_case(21, heads, kvh, d, d, T, n, n, window, sinks)
    j = n - T + T // 2   # the middle token's own position
    V[0, 3, j] = np.inf
    out = np.full((heads, T, d), 7, np.float16)
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, 0.125, 0.0, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
    hit = see[:, j]
    assert np.isposinf(out[:, hit, 3]).all()
    V[0, 3, j] = 0
    want, tol = win_want(Q, K, V, see, 0.125, 0.0)
    keep = np.ones((T, d), bool)
    keep[hit, 3] = False
    near(out[:, keep], want[:, keep], tol[:, keep])


def test_window_attn_is_the_masked_one(lib, fd):
    """The library's masked attention under the same visibility, as a causal mask of 0 and -infinity: its scores are
    clamped at -30000, so hidden keys weigh 0 there too wherever a token sees one."""
    heads, kvh, d, T, n = 4, 2, 128, 70, 500
    Q, K, V, see = win_case(22, heads, kvh, d, d, T, n, n, 90, 3)
    mask = F.f16(np.where(see, 0.0, -np.inf))
    a, b = np.empty((heads, T, d), np.float16), np.empty((heads, T, d), np.float16)
    scale = d ** -0.5
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, 0.0, 90, 3, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(a)) == 0
    assert lib.rocket_flash_attn_fp16(fd, T, n, d, d, heads, kvh, scale, 0.0, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(mask), R.ptr(b)) == 0
    want, tol = win_want(Q, K, V, see, scale, 0.0)
    near(a, want, tol)
    near(b, want, tol)


# ---- soft-caps: every kernel that has them, and caps of any size -----------------------

@pytest.mark.parametrize("cap", [1e-38, -1e-40, 1.5e-45])
@pytest.mark.parametrize("T,d", [(1, 128), (20, 64), (20, 160), (70, 64), (70, 256)])
def test_attn_caps_next_to_none(lib, fd, T, d, cap):
    """The smallest caps, by which a score's factor is past fp32: every score is within the cap of 0, one of a product of 0 as
    well, and results are plain means."""
    heads, kvh, n, window, sinks, scale = 4, 2, 150, 70, 3, 1.0
    for uniform in (False, True):
        c, Q = kv4_case(19, heads, kvh, d, d, T, [n], uniform)
        out, sh = np.full((1, heads, T, d), 7, np.float16), R.Kv4Shape(*c.dims)
        assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, scale, cap, window, sinks, R.ptr(Q), R.ptr(np.array([n], np.int32)),
                                        R.ptr(out)) == 0
        (want, tol), = kv4_want(c, Q * 0, [n], window, sinks, scale, 0.0)
        near(out[0], want, tol)
        Q, K, V, see = win_case(19, heads, kvh, d, d, T, n, n, window, sinks, uniform)
        assert lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, cap, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
        near(out[0], *win_want(Q * 0, K, V, see, scale, 0.0))


def tanh_slack(Q, K, V, scale, cap):
    """What 2^-20 of the capped scores moves a result by: e^delta - 1 of the largest value, twice for the weights' sum."""
    per = Q.shape[0] // K.shape[0]
    s = max(np.abs(Q[i].astype(np.float64) @ K[i // per].astype(np.float64).T).max() for i in range(Q.shape[0]))
    return 2 * np.expm1(2.0 ** -20 * min(abs(cap), s * abs(scale))) * np.abs(V.astype(np.float64)).max()


@pytest.mark.parametrize("T,d,heads,kvh", [(1, 256, 4, 2), (5, 128, 8, 2), (20, 160, 4, 2), (40, 128, 4, 2), (70, 64, 4, 2), (70, 128, 2, 2), (66, 256, 2, 2), (65, 192, 2, 1)])
@pytest.mark.parametrize("cap,scale", [(64.5, 1.0), (-300.0, 1.0), (1e4, 0.125), (-1e6, 0.125), (1e9, 0.125), (3e38, 0.125), (65.0, 20.0)])
def test_attn_soft_caps_above_the_scores(lib, fd, T, d, heads, kvh, cap, scale):
    """Caps far above the scores leave them as they are, up to one that means none; and scores of many times the cap. Beside the
    bound of scores without a cap, 2^-20 of the capped score, for tanh's steps, and nothing that grows with the cap: y - y^3 / 3
    + .. is off by a few 2^-24 of itself, and from y = 0.35 on 1 - 2 / (1 + e^2y), whose terms round to 1.7 2^-23, by 5 2^-23."""
    n, window, sinks = 304, 150, 3
    c, Q = kv4_case(17, heads, kvh, d, d, T, [n])
    sh = R.Kv4Shape(*c.dims)
    out = np.full((1, heads, T, d), 7, np.float16)
    assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(dev(c.buf)), 1, 1, T, n, heads, scale, cap, window, sinks, R.ptr(Q), R.ptr(np.array([n], np.int32)),
                                    R.ptr(out)) == 0
    (want, tol), = kv4_want(c, Q, [n], window, sinks, scale, cap)
    k, v = c.rows()
    near(out[0], want, tol + tanh_slack(Q[0], k[1, :, :n], v[1, :, :n], scale, cap))
    for stride in (n, n + 1):   # (V^T rows read by DMA, and through registers)
        Q, K, V, see = win_case(18, heads, kvh, d, d, T, n, stride, window, sinks)
        assert lib.rocket_flash_attn_window_fp16(fd, T, n, stride, d, d, heads, kvh, scale, cap, window, sinks, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(out)) == 0
        want, tol = win_want(Q, K, V, see, scale, cap)
        near(out[0], want, tol + tanh_slack(Q, K[:, :n], V, scale, cap))


CAPPED_KV4 = [  # every soft-capped kernel over codes: rows of heads of up to 64, 128, 256, whole and narrower; tiles
    (4, 2, 64, 64, 3, [300, 31, 0], 0, 0), (4, 2, 32, 64, 13, [300, 60], 100, 5), (2, 1, 64, 64, 32, [400], 50, 3),
    (32, 8, 128, 128, 1, [700, 127, 128, 0], 0, 0), (8, 2, 128, 96, 7, [333, 70], 64, 3), (4, 1, 128, 128, 15, [300, 15], 0, 0), (8, 8, 96, 128, 1, [500], 0, 0),
    (16, 8, 256, 256, 1, [1000, 33], 0, 0), (2, 1, 256, 256, 1, [2000], 700, 4), (4, 1, 256, 256, 6, [400, 31], 90, 2), (5, 1, 224, 256, 12, [500], 0, 0),
    (4, 2, 64, 64, 70, [300, 90], 0, 0), (4, 2, 128, 128, 70, [500, 90], 0, 0), (6, 2, 96, 128, 40, [300, 77], 50, 3), (2, 1, 128, 128, 300, [900], 129, 70),
    (2, 1, 256, 256, 70, [300, 200], 0, 0), (2, 1, 160, 224, 130, [700], 100, 5),
]
CAPPED_WIN = [  # the same over fp16 keys: rows; tiles of V^T rows that are whole chunks of eight keys, and ragged ones
    (8, 2, 64, 64, 3, 300, 304, 0, 0), (2, 1, 64, 48, 12, 300, 301, 50, 3), (2, 1, 64, 64, 25, 400, 400, 100, 2), (16, 8, 128, 128, 1, 777, 784, 0, 0), (4, 2, 128, 112, 9, 333, 333, 60, 4),
    (16, 8, 256, 256, 1, 777, 800, 0, 0), (2, 1, 256, 256, 1, 2001, 2001, 700, 4), (4, 2, 256, 256, 9, 600, 600, 100, 3), (2, 1, 160, 176, 9, 300, 303, 50, 1),
    (4, 2, 64, 64, 70, 400, 400, 0, 0), (2, 1, 64, 64, 300, 1000, 1024, 129, 70), (2, 1, 96, 80, 90, 300, 304, 0, 0), (2, 1, 128, 128, 130, 512, 520, 100, 5),
    (2, 2, 256, 256, 129, 1000, 1000, 200, 3), (2, 1, 160, 224, 70, 600, 600, 150, 4),
    (2, 1, 64, 64, 90, 411, 411, 70, 4), (4, 2, 128, 128, 100, 411, 413, 90, 4), (2, 1, 256, 192, 70, 411, 413, 0, 0),
]


@pytest.mark.parametrize("cap", [30.0, -300.0])
@pytest.mark.parametrize("uniform", [False, True])
@pytest.mark.parametrize("case", CAPPED_KV4)
def test_kv4_attn_capped(lib, fd, case, uniform, cap):
    """The test of every attention call over the cache, for each soft-capped kernel."""
    test_kv4_attn(lib, fd, case + (cap,), uniform)


@pytest.mark.parametrize("cap", [30.0, -300.0])
@pytest.mark.parametrize("kind", ["random", "uniform", "nan"])
@pytest.mark.parametrize("case", CAPPED_WIN)
def test_window_attn_capped(lib, fd, case, kind, cap):
    test_window_attn(lib, fd, case + (cap,), kind)


# ---- together, and as programs call them -----------------------------------------------

def _handle(lib, stream):
    fd = lib.rocket_open()
    assert fd >= 0
    assert lib.rocket_hip_set_stream(fd, R.ptr(stream.cuda_stream)) == 0
    assert lib.rocket_hip_set_mode(fd, R.ROCKET_HIP_ASYNC | R.ROCKET_HIP_DEVICE_OPERANDS) == 0
    return fd


class Layer:
    """A serving layer's attention over a batch: rows of a fused product -> rotated heads -> cache -> attention, on
    buffers that stay where they are, so that a captured step can be replayed."""

    def __init__(self, lib, n_seq, nq, nk, d, cap, window=0, sinks=0):
        import torch
        self.lib, self.dims, self.win = lib, (n_seq, nq, nk, d, cap), (window, sinks)
        self.c = F.Cache(n_seq, nk, d, d, cap, fill=0xFF)
        self.sh = R.Kv4Shape(*self.c.dims)
        self.mem = dev(self.c.buf)
        self.freq = (10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
        self.w = F.f16(1 + 0.2 * rng(30).standard_normal((2, d)))
        self.dfreq, self.dw = dev(self.freq), dev(self.w)
        self.torch = torch

    def buffers(self, T):
        n_seq, nq, nk, d, _ = self.dims
        new = lambda *s: self.torch.zeros(s, dtype=self.torch.float16, device=DEV)  # noqa: E731
        i = lambda *s: self.torch.zeros(s, dtype=self.torch.int32, device=DEV)  # noqa: E731
        return dict(x=new(n_seq * T, (nq + 2 * nk) * d), pos=i(n_seq * T), lens=i(n_seq), q=new(n_seq, nq, T, d), k=new(n_seq, nk, T, d), out=new(n_seq, nq, T, d), T=T)

    def step(self, fd, b):
        n_seq, nq, nk, d, cap = self.dims
        lib, T, W, sh = self.lib, b["T"], b["x"].shape[1], C.byref(self.sh)
        at = lambda h: R.ptr(b["x"].data_ptr() + 2 * h * d)  # noqa: E731
        assert lib.rocket_qk_norm_rope_fp16(fd, n_seq, T, nq, nk, d, d, R.ROCKET_ROPE_HALVES, 1e-6, at(0), W, at(nq), W, R.ptr(self.dw[0]), R.ptr(self.dw[1]),
                                            R.ptr(self.dfreq), R.ptr(b["pos"]), R.ptr(b["q"]), R.ptr(b["k"])) == 0
        assert lib.rocket_kv4_append_fp16(fd, sh, R.ptr(self.mem), 0, n_seq, T, R.ptr(b["k"]), nk * T * d, T * d, d, at(nq + nk), T * W, d, W, R.ptr(b["lens"])) == 0
        assert lib.rocket_kv4_attn_fp16(fd, sh, R.ptr(self.mem), 0, n_seq, T, cap, nq, d ** -0.5, 0.0, *self.win, R.ptr(b["q"]), R.ptr(b["lens"]), R.ptr(b["out"])) == 0

    def feed(self, b, x, lens):
        T = b["T"]
        pos = (np.array(lens)[:, None] - T + np.arange(T)).astype(np.int32).reshape(-1)
        b["x"].copy_(dev(x))
        b["pos"].copy_(dev(pos))
        b["lens"].copy_(dev(np.array(lens, np.int32)))
        return pos

    def check(self, b, x, pos, lens):
        """This step's results from the GPU's own rotated rows (checked first) and the cache built so far."""
        n_seq, nq, nk, d, cap = self.dims
        T = b["T"]
        q, k, out = (b[n].cpu().numpy() for n in ("q", "k", "out"))
        near(q, *F.rope(x, nq, d, d, False, 1e-6, self.w[0], self.freq, pos, n_seq))
        near(k, *F.rope(x[:, nq * d:], nk, d, d, False, 1e-6, self.w[1], self.freq, pos, n_seq))
        v = x[:, (nq + nk) * d:].reshape(n_seq, T, nk, d)
        for s, n in enumerate(lens):
            for t in range(T):
                if 0 <= n - T + t < cap:
                    for h in range(nk):
                        self.c.put(s, h, n - T + t, k[s, h, t], v[s, t, h])
        assert np.array_equal(self.mem.cpu().numpy(), self.c.buf)
        K, V = self.c.rows()
        for s, n in enumerate(lens):
            see = F.visible(n, T, *self.win, max(1, n))
            near(out[s], *F.attend(q[s], K[s, :, :max(1, n)], V[s, :, :max(1, n)], see, d ** -0.5, 0.0, True))


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_layer_prompt_then_steps(lib, window, sinks):
    """A ragged prompt (padded in front), then single tokens, then drafts of three: eager, on a stream of the caller's."""
    import torch
    stream = torch.cuda.Stream()
    fd = _handle(lib, stream)
    g = rng(31)
    with torch.cuda.stream(stream):
        L = Layer(lib, 3, 4, 2, 64, 120, window, sinks)
        lens = np.array([40, 17, 0])
        for T, grow in ((40, [0, 0, 0]), (1, [1, 1, 0]), (1, [1, 1, 1]), (3, [3, 3, 3])):
            lens = lens + grow
            b = L.buffers(T)
            x = F.f16(g.standard_normal(b["x"].shape))
            pos = L.feed(b, x, lens)
            L.step(fd, b)
            stream.synchronize()
            L.check(b, x, pos, lens)
    lib.rocket_close(fd)


def test_layer_captured(lib):
    """One step captured into a graph and replayed with growing lengths, eager work between the replays: every replay
    is checked. Two graphs of two handles run side by side."""
    import torch
    g = rng(32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    fds = [_handle(lib, s) for s in streams]
    layers, bufs, graphs, lens = [], [], [], [np.array([4, 0, 30]), np.array([1, 63, 64])]
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            L = Layer(lib, 3, 8, 2, 128, 400)
            for s, n in enumerate(lens[i]):   # what the sequences hold already
                if n:
                    L.c.put_all(s, F.f16(g.standard_normal((2, n, 128))), F.f16(g.standard_normal((2, n, 128))))
            L.mem.copy_(dev(L.c.buf))
            b = L.buffers(1)
            x = F.f16(g.standard_normal(b["x"].shape))
            lens[i] = lens[i] + 1
            pos = L.feed(b, x, lens[i])
            L.step(fds[i], b)   # eager first: the kernels' one-time set-up and the handle's scratch
            streams[i].synchronize()
            L.check(b, x, pos, lens[i])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            L.step(fds[i], b)
        layers.append(L)
        bufs.append(b)
        graphs.append(graph)
    for rep in range(4):
        state = []
        for i in range(2):
            lens[i] = lens[i] + (1 if rep < 3 else [1, 300, 0])
            with torch.cuda.stream(streams[i]):
                if rep == 3:   # a long jump: rows put in by hand
                    old = lens[i] - [1, 300, 0]
                    n = int(lens[i][1]) - 1
                    L = layers[i]
                    L.c.put_all(1, F.f16(g.standard_normal((2, n, 128))), F.f16(g.standard_normal((2, n, 128))))
                    assert old[1] <= n
                    L.mem.copy_(dev(L.c.buf))
                x = F.f16(g.standard_normal(bufs[i]["x"].shape))
                state.append((x, layers[i].feed(bufs[i], x, lens[i])))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            layers[i].check(bufs[i], *state[i], lens[i])
    del graphs
    for fd in fds:
        lib.rocket_close(fd)


@pytest.mark.parametrize("T,n", [(1, 700), (150, 700)])
def test_window_attn_captured(lib, T, n):
    import torch
    heads, kvh, d, window, sinks = 4, 2, 128, 200, 4
    stream = torch.cuda.Stream()
    fd = _handle(lib, stream)
    with torch.cuda.stream(stream):
        Q, K, V, see = win_case(33, heads, kvh, d, d, T, n, n + 4, window, sinks)
        dQ, dK, dV = dev(Q), dev(K), dev(V)
        out = dev(np.full((heads, T, d), 7, np.float16))
        call = lambda: lib.rocket_flash_attn_window_fp16(fd, T, n, n + 4, d, d, heads, kvh, 0.1, 0.0, window, sinks, R.ptr(dQ), R.ptr(dK), R.ptr(dV), R.ptr(out))  # noqa: E731
        assert call() == 0
        stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        rc = call()
    assert rc == 0
    for rep in range(3):
        Q = win_case(34 + rep, heads, kvh, d, d, T, n, n + 4, window, sinks)[0]
        with torch.cuda.stream(stream):
            dQ.copy_(dev(Q))
            out.fill_(7)
            graph.replay()
        stream.synchronize()
        near(out.cpu().numpy(), *win_want(Q, K, V, see, 0.1, 0.0))
    del graph
    lib.rocket_close(fd)


def _calls(lib, seed):
    """Every entry on device operands: name -> (call(fd), its results)."""
    g = rng(seed)
    heads, kvh, d, cap, n = 8, 2, 128, 2500, 2400
    c = F.Cache(1, kvh, d, d, cap)
    c.put_all(0, F.f16(g.standard_normal((kvh, n, d))), F.f16(g.standard_normal((kvh, n, d))))
    sh, mem, L = R.Kv4Shape(*c.dims), dev(c.buf), dev(np.array([n], np.int32))
    K, V = dev(F.f16(g.standard_normal((kvh, n, d)))), dev(F.f16(g.standard_normal((kvh, d, n))))
    x, pos, freq = dev(F.f16(g.standard_normal((3, (heads + kvh) * d)))), dev(np.arange(3, dtype=np.int32)), dev(np.linspace(0.01, 1, d // 2, dtype=np.float32))
    new = lambda *s: dev(np.zeros(s, np.float16))  # noqa: E731
    q, k = new(heads, 3, d), new(kvh, 3, d)
    calls = dict(rope=(lambda fd: lib.rocket_qk_norm_rope_fp16(fd, 1, 3, heads, kvh, d, d, 0, 1e-6, R.ptr(x), (heads + kvh) * d, R.ptr(x.data_ptr() + 2 * heads * d),
                                                                    (heads + kvh) * d, None, None, R.ptr(freq), R.ptr(pos), R.ptr(q), R.ptr(k)), [q, k]),
                 append=(lambda fd: lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, 3, R.ptr(K), 0, n * d, d, R.ptr(K), 0, n * d, d, R.ptr(L)), [mem]))
    for T in (1, 8, 12, 90):
        Q, a, b = dev(F.f16(g.standard_normal((heads, T, d)))), new(heads, T, d), new(heads, T, d)
        calls[f"kv4 {T}"] = (lambda fd, T=T, Q=Q, a=a: lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, T, cap, heads, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(a)), [a])
        calls[f"window {T}"] = (lambda fd, T=T, Q=Q, b=b: lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, 0.1, 0.0, 1500, 4, R.ptr(Q), R.ptr(K), R.ptr(V), R.ptr(b)), [b])
    return calls


def _captured(fd, call, stream):
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        rc = call(fd)
    assert rc == 0
    return graph


@pytest.mark.parametrize("name", ["rope", "append", "kv4 1", "kv4 12", "kv4 90", "window 1", "window 8", "window 90"])
def test_serve_capture_on_a_fresh_handle(lib, name):
    """A handle's first call is a captured one: it has no scratch to split keys on, and takes as many workgroups as it can
    without. Up to the splits' order of sums the eager results."""
    import torch
    print("fresh handle", name, flush=True)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call, outs = _calls(lib, 40)[name]
    warm, fd = _handle(lib, stream), _handle(lib, stream)
    with torch.cuda.stream(stream):
        assert call(warm) == 0
        want = [o.cpu().numpy() for o in outs]
    graph = _captured(fd, call, stream)
    for _ in range(3):
        with torch.cuda.stream(stream):
            if name != "append":
                for o in outs:
                    o.fill_(7)
            graph.replay()
            stream.synchronize()
            for o, w in zip(outs, want):
                if name in ("rope", "append"):
                    assert np.array_equal(o.cpu().numpy(), w)
                else:   # each side is off by its weights' and its result's rounding, of values up to 5
                    assert np.abs(o.cpu().numpy().astype(np.float64) - w).max() <= 4 * 5 * F.U
    del graph
    for f in (warm, fd):
        lib.rocket_close(f)


@pytest.mark.parametrize("uniform", [False, True])
@pytest.mark.parametrize("T", [1, 8, 12, 90])
def test_serve_attn_captured_on_a_fresh_handle_counts_every_key(lib, T, uniform):
    """A handle's first call, captured, over keys that it cannot split: against 64 bits, and for queries of zero, whose results
    are plain means of the visible values, in which a key too many or too few shows."""
    import torch
    heads, kvh, d, n, window, sinks = 8, 2, 128, 2400, 1500, 4
    stream = torch.cuda.Stream()
    c, Q = kv4_case(51, heads, kvh, d, d, T, [n], uniform, spare=100)
    Qw, K, V, see = win_case(52, heads, kvh, d, d, T, n, n, window, sinks, uniform)
    sh, scale = R.Kv4Shape(*c.dims), d ** -0.5
    with torch.cuda.stream(stream):
        mem, L, dQ, dQw, dK, dV = dev(c.buf), dev(np.array([n], np.int32)), dev(Q), dev(Qw), dev(K), dev(V)
        outs = [dev(np.zeros((heads, T, d), np.float16)) for _ in range(2)]
    stream.synchronize()
    calls = (lambda fd: lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 1, 1, T, n + 100, heads, scale, 0.0, 0, 0, R.ptr(dQ), R.ptr(L), R.ptr(outs[0])),
             lambda fd: lib.rocket_flash_attn_window_fp16(fd, T, n, n, d, d, heads, kvh, scale, 0.0, window, sinks, R.ptr(dQw), R.ptr(dK), R.ptr(dV), R.ptr(outs[1])))
    wants = (list(kv4_want(c, Q, [n], 0, 0, scale, 0.0))[0], win_want(Qw, K, V, see, scale, 0.0))
    for call, out, want in zip(calls, outs, wants):
        fd = _handle(lib, stream)
        graph = _captured(fd, call, stream)
        for _ in range(3):
            with torch.cuda.stream(stream):
                out.fill_(7)
                graph.replay()
            stream.synchronize()
            near(out.cpu().numpy(), *want)
        del graph
        lib.rocket_close(fd)


def test_serve_part_of_a_batch_captured(lib):
    """Places 1 and 2 of four, their lengths and positions in the middle of the batch's arrays: a fresh handle's first calls
    are captured ones, which only operands in place allow, and every replay takes the lengths of the day."""
    import torch
    stream, g = torch.cuda.Stream(), rng(47)
    fd, heads, kvh, d, cap, T, window, sinks = _handle(lib, stream), 4, 2, 64, 200, 2, 40, 3
    c = F.Cache(4, kvh, d, d, cap)
    for s in range(4):
        c.put_all(s, F.f16(g.standard_normal((kvh, cap, d))), F.f16(g.standard_normal((kvh, cap, d))))
    sh, freq = R.Kv4Shape(*c.dims), np.linspace(0.01, 1, d // 2, dtype=np.float32)
    W = (heads + 2 * kvh) * d
    new = lambda *s: torch.zeros(s, dtype=torch.float16, device=DEV)  # noqa: E731
    with torch.cuda.stream(stream):
        mem, dfreq, x, q, k, out, back = dev(c.buf), dev(freq), new(2 * T, W), new(2, heads, T, d), new(2, kvh, T, d), new(2, heads, T, d), new(2, kvh, T, d)
        lens, pos = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(2 * T + 2, dtype=torch.int32, device=DEV)

        def step():
            L, at = R.ptr(lens.data_ptr() + 4), lambda h: R.ptr(x.data_ptr() + 2 * h * d)
            return (lib.rocket_qk_norm_rope_fp16(fd, 2, T, heads, kvh, d, d, 0, 1e-6, at(0), W, at(heads), W, None, None, R.ptr(dfreq), R.ptr(pos.data_ptr() + 4), R.ptr(q), R.ptr(k)),
                    lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), 1, 2, T, R.ptr(k), kvh * T * d, T * d, d, at(heads + kvh), T * W, d, W, L),
                    lib.rocket_kv4_read_fp16(fd, C.byref(sh), R.ptr(mem), 1, 2, T, L, R.ptr(back), None),
                    lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 1, 2, T, cap, heads, 0.125, 0.0, window, sinks, R.ptr(q), L, R.ptr(out)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        rcs = step()
    assert rcs == (0, 0, 0, 0)
    for day in ([150, 7, 99, 3], [1, 200, 64, 90], [5, 30, 2, 5]):
        with torch.cuda.stream(stream):
            X, P = F.f16(g.standard_normal((2 * T, W))), np.array(day[1:3])[:, None] - T + np.arange(T)
            x.copy_(dev(X))
            lens.copy_(dev(np.array(day, np.int32)))
            pos[1:2 * T + 1].copy_(dev(P.reshape(-1).astype(np.int32)))
            graph.replay()
        stream.synchronize()
        hq, hk, v = q.cpu().numpy(), k.cpu().numpy(), X[:, (heads + kvh) * d:].reshape(2, T, kvh, d)
        near(hq, *F.rope(X, heads, d, d, False, 1e-6, None, freq, P.reshape(-1), 2))
        near(hk, *F.rope(X[:, heads * d:], kvh, d, d, False, 1e-6, None, freq, P.reshape(-1), 2))
        for s in range(2):
            for t in range(T):
                for h in range(kvh):
                    c.put(s + 1, h, P[s, t], hk[s, h, t], v[s, t, h])
        assert np.array_equal(mem.cpu().numpy(), c.buf)
        K, V = c.rows()
        for s, n in enumerate(day[1:3]):
            assert np.array_equal(back.cpu().numpy()[s], F.f16(K[s + 1][:, P[s]]))
            near(out.cpu().numpy()[s], *F.attend(hq[s], K[s + 1, :, :n], V[s + 1, :, :n], F.visible(n, T, window, sinks, n), 0.125, 0.0, True))
    del graph
    lib.rocket_close(fd)


def test_serve_graphs_of_one_handle(lib):
    """Four attention calls captured one by one on one handle, replayed in turn, with an eager call between the replays that
    makes the handle's scratch grow: the eager results, bit for bit."""
    import torch
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls = {k: v for k, v in _calls(lib, 41).items() if " " in k}
        big = F.Cache(1, 2, 256, 256, 9000, fill=0)
        mem, L, Q, out = dev(big.buf), dev(np.array([9000], np.int32)), dev(np.zeros((2, 300, 256), np.float16)), dev(np.zeros((2, 300, 256), np.float16))
    sh, fd = R.Kv4Shape(*big.dims), _handle(lib, stream)
    want, graphs = {}, {}
    with torch.cuda.stream(stream):
        for k, (call, outs) in calls.items():
            assert call(fd) == 0
            want[k] = outs[0].cpu().numpy()
    for k, (call, _) in calls.items():
        graphs[k] = _captured(fd, call, stream)
    with torch.cuda.stream(stream):
        for rep in range(3):
            for k in list(calls)[rep:] + list(calls)[:rep]:
                calls[k][1][0].fill_(7)
                graphs[k].replay()
                assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), 0, 1, 100 * (rep + 1), 9000, 2, 0.1, 0.0, 0, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
            stream.synchronize()
            for k, (_, outs) in calls.items():
                assert np.array_equal(outs[0].cpu().numpy(), want[k]), (rep, k)
    graphs.clear()
    lib.rocket_close(fd)


def test_serve_from_two_threads(lib):
    """Two threads with a handle each, and two that share one: every call's results are the first's, bit for bit."""
    import threading

    import torch
    calls = [_calls(lib, 42 + i) for i in range(2)]
    torch.cuda.synchronize()
    fds, wrong = [lib.rocket_open() for _ in range(3)], []
    want = []
    for cs in calls:
        want.append({})
        for k, (call, outs) in cs.items():
            assert call(fds[0]) == 0
            want[-1][k] = [o.cpu().numpy() for o in outs]

    def work(i, fd):
        for _ in range(5):
            for k, (call, outs) in calls[i].items():
                if call(fd) != 0 or any(not np.array_equal(o.cpu().numpy(), w) for o, w in zip(outs, want[i][k])):
                    wrong.append((i, k))
    for pair in ((fds[0], fds[1]), (fds[2], fds[2])):
        ts = [threading.Thread(target=work, args=(i, pair[i])) for i in range(2)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    assert not wrong
    for f in fds:
        lib.rocket_close(f)


def test_measured_calls_are_on_the_current_stream(lib):
    """perf/operators.py's calls are ordered with what torch does next: its stream is the one that they are queued on, and a
    result may be read, and its state dropped, with no wait between."""
    import importlib.util
    import os

    import torch
    spec = importlib.util.spec_from_file_location("measured_operators", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    M.own, before = True, torch.cuda.current_stream()
    case = next(c for c in M.listed() if c["name"] == "win_prefill")
    try:
        first = M.prepare(case, 1)   # (made on another stream than the calls')
        M.run(first)
        assert torch.cuda.current_stream().cuda_stream == lib.rocket_hip_stream(M._lib["fd"])
        torch.cuda.synchronize()
        want = first["out"].clone()
        first["out"].zero_()
        got = M.run(first).clone()
        del first
        M.prepare(case, 2)           # (takes the memory that the first state left)
        assert torch.equal(got, want)
    finally:
        torch.cuda.synchronize()
        torch.cuda.set_stream(before)
        if M._lib:
            lib.rocket_close(M._lib["fd"])


# ---- the largest sizes -----------------------------------------------------------------

def test_cache_past_32_bits(lib, fd):
    """Parts of more than 4 GiB: the last two places' tokens, at the front of one and the end of the other."""
    import torch
    S, H, d, cap, new, window = 64, 8, 256, 1 << 16, 300, 200
    sh = R.Kv4Shape(S, H, d, d, cap)
    size = lib.rocket_kv4_bytes(C.byref(sh))
    assert size >= 10 << 30
    mem = torch.empty(size, dtype=torch.uint8, device=DEV)
    g = rng(45)
    lens = np.array([new, cap], np.int32)
    K, V = F.f16(g.standard_normal((2, H, new, d))), F.f16(g.standard_normal((2, H, new, d)))
    dK, dV, L = dev(K), dev(V), dev(lens)
    ss, hs = H * new * d, new * d
    assert lib.rocket_kv4_append_fp16(fd, C.byref(sh), R.ptr(mem), S - 2, 2, new, R.ptr(dK), ss, hs, d, R.ptr(dV), ss, hs, d, R.ptr(L)) == 0
    c = F.Cache(2, H, d, d, new)
    for s in range(2):
        c.put_all(s, K[s], V[s])
    k, v = c.rows()
    a, b = np.empty((2, H, new, d), np.float16), np.empty((2, H, new, d), np.float16)
    assert lib.rocket_kv4_read_fp16(fd, C.byref(sh), R.ptr(mem), S - 2, 2, new, R.ptr(L), R.ptr(a), R.ptr(b)) == 0
    assert np.array_equal(a, F.f16(k[:, :, :new])) and np.array_equal(b, F.f16(v[:, :, :new]))
    for T in (1, 40):
        Q, out = F.f16(g.standard_normal((2, H, T, d))), np.empty((2, H, T, d), np.float16)
        assert lib.rocket_kv4_attn_fp16(fd, C.byref(sh), R.ptr(mem), S - 2, 2, T, cap, H, d ** -0.5, 0.0, window, 0, R.ptr(Q), R.ptr(L), R.ptr(out)) == 0
        for s in range(2):   # (under the window the end of a long sequence is that of a short one)
            near(out[s], *F.attend(Q[s], k[s, :, :new], v[s, :, :new], F.visible(new, T, window, 0, new), d ** -0.5, 0.0, True))


@pytest.mark.parametrize("T", [2, 150])
def test_window_longest(lib, fd, T):
    """The longest keys and V^T rows that the call takes, NaN where no token sees them."""
    import torch
    stride, d, window, sinks, end = (1 << 22) - 64, 256, 300, 2, 600
    n = stride - 3
    g = rng(46)
    at = np.concatenate([np.arange(sinks), np.arange(n - end, n)])
    K, V, Q = F.f16(g.standard_normal((1, at.size, d))), F.f16(g.standard_normal((1, at.size, d))), F.f16(g.standard_normal((1, T, d)))
    dK = torch.full((stride, d), float("nan"), dtype=torch.float16, device=DEV)
    dV = torch.full((d, stride), float("nan"), dtype=torch.float16, device=DEV)
    first = n - T - window + 1
    seen = (at >= first) | (at < sinks)
    i = dev(at[seen])
    dK[i] = dev(K[0, seen])
    dV[:, i] = dev(V[0, seen].T)
    p = (n - T + np.arange(T))[:, None]
    see = (at[None] <= p) & ((at[None] > p - window) | (at[None] < sinks))
    dQ, out = dev(Q), np.empty((1, T, d), np.float16)
    assert lib.rocket_flash_attn_window_fp16(fd, T, n, stride, d, d, 1, 1, d ** -0.5, 0.0, window, sinks, R.ptr(dQ), R.ptr(dK), R.ptr(dV), R.ptr(out)) == 0
    near(out, *F.attend(Q, K.astype(np.float64), V.astype(np.float64), see, d ** -0.5, 0.0, False))
