"""The operators of rocket_serve.h in numpy, in 64 bits: what the CPU and GPU tests compare with, and
bounds of the roundings that an fp16 result may carry."""
import numpy as np

U = 2.0 ** -11   # half a step of fp16, relative


def rope(x, heads, d, rot, pairs, eps, w, freq, pos, n_seq):
    """Heads [n_seq][heads][tokens][d] of rows x[rows, >= heads * d], and the bound of an fp16 result made in fp32
    steps: half a step of the value (and the least normal's, 2^-25), and 2^-20 of the pair's magnitudes (sine and
    cosine within 2^-22, the norm's factor within a few 2^-24)."""
    rows = x.shape[0]
    y = x[:, :heads * d].astype(np.float64).reshape(rows, heads, d)
    if eps >= 0:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
        if w is not None:
            y = y * w.astype(np.float64)
    out, size = y.copy(), np.abs(y)
    if rot:
        h = rot // 2
        a = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
        i = np.arange(h)
        i, j = (2 * i, 2 * i + 1) if pairs else (i, i + h)
        c, s = np.cos(a), np.sin(a)
        out[..., i], out[..., j] = y[..., i] * c - y[..., j] * s, y[..., j] * c + y[..., i] * s
        size[..., i] = size[..., j] = np.abs(y[..., i]) + np.abs(y[..., j])
    T = rows // n_seq
    turn = lambda v: np.ascontiguousarray(v.reshape(n_seq, T, heads, d).transpose(0, 2, 1, 3))  # noqa: E731
    return turn(out), turn(np.abs(out) * U + size * 2.0 ** -20 + 2.0 ** -25)


def quantise(x):
    """Codes [..., d] and (scale, minimum) fp16 [..., d / 32, 2] of finite fp16 rows, in fp32 steps."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1, keepdims=True) + np.float32(0), g.max(-1, keepdims=True)
    s = ((hi - lo) / np.float32(15)).astype(np.float16)
    s = np.where(s.astype(np.float64) * 15 + lo < 65520, s, (s.view(np.uint16) - 1).astype(np.uint16).view(np.float16))
    f = s.astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(f > 0, np.clip(np.rint((g - lo) / f), 0, 15), 0).astype(np.uint8)
    return c.reshape(x.shape), np.concatenate([s, lo.astype(np.float16)], -1)


def values(codes, sm):
    """code * scale + minimum in 64 bits (exact)."""
    sm = sm.astype(np.float64)
    g = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, 32) * sm[..., :1] + sm[..., 1:]
    return g.reshape(codes.shape)


class Cache:
    """A cache buffer of a shape: its parts as arrays, and rows put into and taken out of it."""

    def __init__(self, n_seq, heads, dk, dv, capacity, fill=None):
        self.dims = n_seq, heads, dk, dv, capacity
        cap = (capacity + 31) // 32 * 32
        rows, at, self.at = n_seq * heads * cap, 0, []
        for n in (rows * dk // 2, rows * dk // 8, rows * dv // 2, rows * dv // 8):
            self.at.append((at, n))
            at = (at + n + 255) // 256 * 256
        self.buf = np.zeros(at, np.uint8) if fill is None else np.full(at, fill, np.uint8)
        self.cap = cap

    def parts(self, buf=None):
        S, H, dk, dv, _ = self.dims
        b = self.buf if buf is None else buf
        kc, ks, vc, vs = (b[a:a + n] for a, n in self.at)
        return (kc.reshape(S, H, self.cap, dk // 2), ks.view(np.float16).reshape(S, H, self.cap, dk // 32, 2),
                vc.reshape(S, H, self.cap // 8, dv // 8, 8, 4), vs.view(np.float16).reshape(S, H, self.cap // 8, dv // 32, 8, 2))

    def put(self, s, h, j, k, v):
        """Position j of head h of place s: fp16 rows k[dk], v[dv]."""
        kc, ks, vc, vs = self.parts()
        c, sm = quantise(k)
        kc[s, h, j], ks[s, h, j] = c[0::2] | c[1::2] << 4, sm
        c, sm = quantise(v)
        vc[s, h, j // 8, :, j % 8], vs[s, h, j // 8, :, j % 8] = (c[0::2] | c[1::2] << 4).reshape(-1, 4), sm

    def put_all(self, s, k, v):
        """The first positions of place s: fp16 rows k[heads][n][dk], v[heads][n][dv]."""
        kc, ks, vc, vs = self.parts()
        n, (c, sm) = k.shape[1], quantise(k)
        kc[s, :, :n], ks[s, :, :n] = c[..., 0::2] | c[..., 1::2] << 4, sm
        c, sm = quantise(v)
        j = np.arange(n)
        vc[s][:, j // 8, :, j % 8] = (c[..., 0::2] | c[..., 1::2] << 4).reshape(*c.shape[:2], -1, 4).transpose(1, 0, 2, 3)
        vs[s][:, j // 8, :, j % 8] = sm.transpose(1, 0, 2, 3)

    def rows(self):
        """Keys [S][H][cap][dk] and values [S][H][cap][dv] in 64 bits."""
        S, H, dk, dv, _ = self.dims
        kc, ks, vc, vs = self.parts()
        both = lambda b: np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)  # noqa: E731
        vc = vc.transpose(0, 1, 2, 4, 3, 5).reshape(S, H, self.cap, dv // 2)
        return values(both(kc), ks), values(both(vc), vs.transpose(0, 1, 2, 4, 3, 5).reshape(S, H, self.cap, dv // 32, 2))


def visible(n, T, window, sinks, keys):
    """[T][keys]: whether token t of the last T positions of n sees key j."""
    p, j = (n - T + np.arange(T))[:, None], np.arange(keys)[None]
    see = j <= p
    return see & ((j > p - window) | (j < sinks)) if window else see


def attend(Q, K, V, see, scale, softcap, rounded):
    """softmax over the visible keys of Q[heads][T][dk] with K[kv][n][dk], V[kv][n][dv] (64 bits), and the bound of
    an fp16 result: half a step of the result, of the probabilities and, where a kernel holds keys and values
    rounded to fp16 (`rounded`), of the values and (through the scores: e^delta - 1, twice for the sum) of the keys;
    2^-18 for the fp32 sums and exponentials; and as much of the scores' magnitudes as fp32 products round (2^-22)."""
    h, T, dk = Q.shape
    kvh = K.shape[0]
    out, tol = np.zeros((h, T, V.shape[2])), np.zeros((h, T, V.shape[2]))
    for i in range(h):
        k, v = K[i // (h // kvh)], V[i // (h // kvh)]
        seen = see.any(0)   # what no token sees may hold anything
        k, v = np.where(seen[:, None], k, 0.0), np.where(seen[:, None], v, 0.0)
        q = Q[i].astype(np.float64)
        s, size = (q @ k.T) * scale, (np.abs(q) @ np.abs(k).T) * abs(scale)
        if softcap:
            s = softcap * np.tanh(s / softcap)
        s = np.where(see, s, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
        l = p.sum(1, keepdims=True)
        p = p / np.where(l > 0, l, 1.0)
        out[i] = p @ v
        delta = ((U if rounded else 0.0) + 2.0 ** -22) * np.where(see, size, 0.0).max(1, keepdims=True) + 2.0 ** -20
        tol[i] = np.abs(out[i]) * U + (p @ np.abs(v)) * (2 * np.expm1(delta) + (U if rounded else 0.0) + U + 2.0 ** -18) + 2.0 ** -24
    return out, tol


def f16(x):
    return np.ascontiguousarray(x).astype(np.float16)
