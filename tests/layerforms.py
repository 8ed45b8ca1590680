"""The operators of rocket_fp8.h and rocket_layer.h in 64 bits, in plain torch, each with the bound that its results keep.

Bounds count roundings: one to type t is off by at most E[t] of the value (half a step), a sum of n fp32 terms by n * E[fp32] of the
terms' sizes. The 8-bit matrix products behind fp16 results add their own: of eight neighbouring products each is cut at 2^-13 of the
largest one's power of two, so seven of them lose less than 7 * 2^-13 of the largest."""
import math

import torch

BLOCK = 128
E = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25}   # half of the smallest step
e32 = E[torch.float32]


def blocks(n):
    return -(-n // BLOCK)


# ---- e4m3 ------------------------------------------------------------------------------

def _value(c):
    e, f = c >> 3 & 15, c & 7
    v = math.nan if (e, f) == (15, 7) else (8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9
    return -v if c & 128 else v


VALUES = torch.tensor([_value(c) for c in range(256)], dtype=torch.float64)


def decode(q):
    return VALUES.to(q.device)[q.long()]


def encode(v):
    """Nearest codes of |v| <= 448 (fp32 or fp64), ties to the even code; NaN to 0x7f."""
    steps = VALUES[:127].to(v.device)                      # 0 .. 448, rising
    x = v.double().abs().nan_to_num(0.0)
    hi = torch.searchsorted(steps, x.contiguous()).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    up, down = steps[hi] - x, x - steps[lo]
    c = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    c = torch.where(x == 0, torch.zeros_like(c), c) + 128 * torch.signbit(v).long()
    return torch.where(v.isnan(), torch.full_like(c, 0x7f), c).to(torch.uint8)


def quantise(x):
    """Codes and scales of fp32 rows by the formula, in fp32."""
    M, K = x.shape
    g = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(M, -1, BLOCK)
    a = g.abs().nan_to_num(0.0, posinf=math.inf).amax(2).clamp_min(2.0 ** -100)
    v = g * (torch.full_like(a, 448.0) / a)[..., None]
    v = torch.where(v > 448, torch.full_like(v, 448), torch.where(v < -448, torch.full_like(v, -448), v))
    return encode(v).flatten(1)[:, :K].contiguous(), a / 448.0


def quantise_weights(w):
    """Codes and scales of [E][N][K] weights, one scale for each block of 128 by 128."""
    n, k = w.shape[-2:]
    b = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).unflatten(-2, (-1, BLOCK)).unflatten(-1, (-1, BLOCK))
    a = b.abs().amax((-3, -1)).clamp_min(2.0 ** -100)
    q = encode((b * (448.0 / a)[..., :, None, :, None]).clamp(-448, 448))
    return q.flatten(-2).flatten(-3, -2)[..., :n, :k].contiguous(), (a / 448.0).contiguous()


def same_codes(got, want):
    """Whether the codes are the same, NaN of either sign alike."""
    nan = lambda q: (q & 127) == 127  # noqa: E731
    return bool(((got == want) | (nan(got) & nan(want))).all())


def near_codes(q, scale, x, ex):
    """Whether codes and scales are those of values within ex of x: each scale's maximum, each code's half step."""
    M, K = x.shape
    pad = lambda t: torch.nn.functional.pad(t, (0, -K % BLOCK)).view(M, -1, BLOCK)  # noqa: E731
    g, eg = pad(x), pad(ex)
    a = g.abs().amax(2).clamp_min(2.0 ** -100)
    if not bool(((scale.double() * 448 - a).abs() <= eg.amax(2) + 3 * e32 * a).all()):
        return False
    s = scale.double()[..., None]
    v = decode(q).view(M, K)
    half = torch.maximum(g.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -10) + 2 * eg
    return bool((((pad(v) * s) - g).abs() <= half).all())


# ---- products --------------------------------------------------------------------------

def _scaled(q, s, rows):
    v = decode(q)
    s = s.double().repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]
    return v * (s.repeat_interleave(rows, -2)[..., :q.shape[-2], :] if rows > 1 else s)


def product(A, sa, B, sb, dtype):
    """A B^T of codes and scales, and the bound of an element."""
    a, b = _scaled(A, sa, 1), _scaled(B, sb, BLOCK)
    r, size = a @ b.t(), a.abs() @ b.abs().t()
    tol = (BLOCK + sa.shape[1] + 4) * e32 * size + E[dtype] * r.abs() + TINY[dtype]
    if dtype == torch.float16:
        # the largest of eight products is at most the largest of each factor
        K = a.shape[1]
        eight = lambda t: torch.nn.functional.pad(t.abs(), (0, -K % 8)).view(t.shape[0], -1, 8).amax(2)  # noqa: E731
        tol = tol + 7 * 2.0 ** -13 * (eight(a) @ eight(b).t())
    return r, tol


def grouped(A, sa, src, off, B, sb, rows, dtype):
    """Experts' products; rows behind the last expert are NaN in both (not written)."""
    out = torch.full((rows, B.shape[1]), math.nan, dtype=torch.float64, device=B.device)
    tol = out.clone()
    for e in range(B.shape[0]):
        i, j = int(off[e]), int(off[e + 1])
        if j > i:
            at = torch.arange(i, j, device=B.device) if src is None else src[i:j].long()
            ok = (at >= 0) & (at < A.shape[0])
            at = at.clamp(0, A.shape[0] - 1)
            out[i:j], tol[i:j] = product(A[at], sa[at], B[e], sb[e], dtype)
            out[i:j][~ok], tol[i:j][~ok] = 0.0, 0.0
    return out, tol


# ---- gated rows ------------------------------------------------------------------------

def gated(act, g, u):
    """act(g) * u, and its bound: GELU's complementary error function is within 1.2e-7 of itself and an exponential of up to
    z^2 = x^2 / 2 adds its argument's rounding; SiLU's exponential the same of |x|."""
    g, u = g.double(), u.double()
    if act == "gelu":
        r = g * torch.special.ndtr(g) * u
        return r, r.abs() * (1.2e-7 + (16 + 2 * g * g) * e32) + 2.0 ** -140
    r = g * torch.sigmoid(g) * u
    return r, r.abs() * (16 + 2 * g.abs()) * e32 + 2.0 ** -126 * u.abs()


# ---- norms -----------------------------------------------------------------------------

NORM = 48 * e32   # of a row's factor: at most 38 additions of squares, halved by the root, and the root, quotient and products


def _norm(v, ev, w, eps):
    if eps < 0:
        return v, ev
    r = 1 / (v.square().mean(1, keepdim=True) + eps).sqrt()
    w = 1.0 if w is None else w.double()
    n = v * r * w
    off = ev.norm(dim=1, keepdim=True) / v.norm(dim=1, keepdim=True).clamp_min(1e-300)
    return n, ev * r * (abs(w) if isinstance(w, float) else w.abs()) + n.abs() * (NORM + off)


def add_norm(h, y, w_post, eps_post, gate, every, alpha, w_pre, eps_pre, slot=None, weight=None, shared=None):
    """(h', its bound, x, its bound), before they are rounded to their types."""
    h = h.double()
    M = h.shape[0]
    eh = torch.zeros_like(h)
    if y is not None:
        z = y.double()
        ez = torch.zeros_like(h)
        if slot is not None:
            ok = (slot >= 0) & (slot < y.shape[0])
            w = torch.where(ok, weight.double(), torch.zeros((), dtype=torch.float64, device=h.device))
            rows = torch.where(ok[..., None], z[slot.long().clamp(0, y.shape[0] - 1)], torch.zeros((), dtype=torch.float64, device=h.device))
            z, size = (rows * w[..., None]).sum(1), (rows * w[..., None]).abs().sum(1)
            if shared is not None:
                z, size = z + shared.double(), size + shared.double().abs()
            ez = (slot.shape[1] + 2) * e32 * size
        z, ez = _norm(z, ez, w_post, eps_post)
        g = alpha if gate is None else alpha * gate.double()[torch.arange(M, device=h.device) // every]
        z, ez = z * g, ez * abs(g)
        eh = ez + 4 * e32 * (h.abs() + z.abs())
        h = h + z
    x, ex = _norm(h, eh, w_pre, eps_pre)
    return h, eh, x, ex + 2 * e32 * x.abs()


def rounded(v, ev, dtype):
    """The bound of v's rounding to dtype, on top of ev."""
    return ev * (1 + 2 * E[dtype]) + E[dtype] * v.abs() + TINY[dtype]


# ---- routing ---------------------------------------------------------------------------

def route(logits, k, sigmoid=False, bias=None, groups=1, best=1, top_groups=1, renorm=True, scale=1.0, active=None):
    """A token at a time: (ids, weights in 64 bits, expert_off, src_row, slot), src_row as long as there are rows."""
    M, n = logits.shape
    ids = torch.full((M, k), -1, dtype=torch.int64)
    weight = torch.zeros((M, k), dtype=torch.float64)
    rank = lambda v: -4e300 if v != v else min(max(v, -1e300), 1e300)  # noqa: E731
    for m in range(M):
        if active is not None and not active[m]:
            continue
        x = logits[m].double().clamp_max(3.4028234663852886e38)
        if sigmoid:
            p = 1 / (1 + torch.exp(-x))
        else:
            top = x[~x.isnan()].max() if bool((~x.isnan()).any()) else torch.tensor(0.0)
            p = torch.exp(x - (top if top > -math.inf else 0.0))
            p = p / p.sum()
        c = p + bias.double() if bias is not None else p
        can = [bool(v != -math.inf) for v in x]
        choice = [rank(float(v)) if ok else -math.inf for v, ok in zip(c, can)]
        key = choice if bias is not None else [rank(float(v)) if ok else -math.inf for v, ok in zip(x, can)]
        if groups > 1:
            run = n // groups
            value = []
            for g in range(groups):
                two = sorted((v for v in choice[g * run:(g + 1) * run] if v > -math.inf), reverse=True)[:best]
                value.append(sum(two) if two else -math.inf)
            stay = [g for g in sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups] if value[g] > -math.inf]
            key = [v if e // run in stay else -math.inf for e, v in enumerate(key)]
        at = [e for e in sorted(range(n), key=lambda e: (-key[e], e))[:k] if key[e] > -math.inf]
        total = float(p[at].sum()) if at else 0.0
        for j, e in enumerate(at):
            ids[m, j] = e
            weight[m, j] = scale * (float(p[e]) if not renorm else 0.0 if total == 0 else float(p[e]) / total)
    rows = sorted((int(ids[m, j]), m, j) for m in range(M) for j in range(k) if ids[m, j] >= 0)
    off = torch.tensor([sum(r[0] < e for r in rows) for e in range(n + 1)])
    slot = torch.full((M, k), -1, dtype=torch.int64)
    for i, (_, m, j) in enumerate(rows):
        slot[m, j] = i
    return ids, weight, off, torch.tensor([r[1] for r in rows], dtype=torch.int64), slot
