"""The attention side of a serving step, as measurable calls: norms and rotation of the query and key
heads, keys and values quantised into a 4-bit cache and read back, attention over that cache for a
batch of sequences, and attention with a sliding window and sinks over fp16 keys and values.

Where `own` is false, run() computes each operator in elementary torch operations, in 32 bits with
64-bit angles; where it is true, it makes the library's calls."""
import ctypes as C
import math
import os
import sys

import torch

own = False

GROUP = 32   # dims of a key that share a scale and a minimum in the 4-bit cache


def listed():
    return [
        # rows of a decode step, one token of 16 sequences, out of a fused fp16 product: latency
        dict(name="rope_decode", op="rope", seqs=16, T=1, heads=16, kv_heads=8, dim=256, rot=256, pairs=False, rows="fp16", norm=True, far=32768),
        # a long prompt's rows out of a quantised product (fp32 results), far positions
        dict(name="rope_prefill", op="rope", seqs=1, T=4096, heads=32, kv_heads=8, dim=128, rot=128, pairs=False, rows="fp32", norm=True, far=1000000),
        # neighbouring pairs, part of the head rotated, odd counts
        dict(name="rope_ragged", op="rope", seqs=3, T=171, heads=10, kv_heads=2, dim=96, rot=64, pairs=True, rows="fp16", norm=True, far=8192),
        # one token of 32 sequences joins the 4-bit cache (read back: the values it stands for)
        dict(name="append_decode", op="append", seqs=32, T=1, kv_heads=8, dim=128, cap=4096),
        # a prompt of 4096 tokens joins it
        dict(name="append_prefill", op="append", seqs=1, T=4096, kv_heads=8, dim=256, cap=8192),
        # one sequence's next token, a cache whose length is no multiple of a tile
        dict(name="kv4_decode_one", op="kv4", seqs=1, T=1, n_kv=3000, cap=4096, heads=16, kv_heads=8, dim=256, window=0, sinks=0, softcap=0.0),
        # a decode batch of 32 sequences of lengths up to 8192
        dict(name="kv4_decode_batch", op="kv4", seqs=32, T=1, n_kv=8192, cap=8192, heads=32, kv_heads=8, dim=128, window=0, sinks=0, softcap=0.0),
        # five drafted tokens of four sequences at once, the last 1024 keys and four sinks
        dict(name="kv4_draft", op="kv4", seqs=4, T=5, n_kv=6001, cap=8192, heads=8, kv_heads=2, dim=64, window=1024, sinks=4, softcap=0.0),
        # a chunk of a prompt over a long cache
        dict(name="kv4_prefill", op="kv4", seqs=1, T=512, n_kv=4096, cap=8192, heads=16, kv_heads=8, dim=256, window=0, sinks=0, softcap=0.0),
        # fp16 keys: a long prompt chunk under a window, the largest call
        dict(name="win_prefill", op="win", T=2048, n_kv=8192, stride=8192, heads=16, kv_heads=8, dim=256, window=1024, sinks=4, softcap=0.0),
        # one token at the end of a long fp16 cache under a window
        dict(name="win_decode", op="win", T=1, n_kv=32768, stride=32768, heads=32, kv_heads=8, dim=128, window=4096, sinks=4, softcap=0.0),
        # no size a multiple of a tile, a cache with room behind the last key, soft-capped scores
        dict(name="win_ragged", op="win", T=333, n_kv=1501, stride=1737, heads=8, kv_heads=2, dim=64, window=257, sinks=3, softcap=50.0),
    ]


def draw(rng):
    def size(lo, hi, step=1):   # log-uniform, a multiple of step
        return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step

    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(["rope", "append", "kv4", "kv4", "win", "win"])
        kv = rng.choice([1, 2, 4, 8])
        heads, dim = kv * rng.choice([1, 2, 4, 5]), rng.choice([64, 64, 96, 128, 128, 160, 256])
        if op == "rope":
            T = rng.choice([1, size(2, 4096)])
            rot = rng.choice([dim, dim, dim // 2])
            c = dict(op=op, seqs=size(1, 64) if T < 64 else 1, T=T, heads=heads, kv_heads=kv, dim=dim, rot=rot, pairs=rng.random() < 0.4,
                     rows=rng.choice(["fp16", "fp32"]), norm=rng.random() < 0.8, far=size(4096, 1000000))
        elif op == "append":
            T = rng.choice([1, size(2, 4096)])
            c = dict(op=op, seqs=size(1, 32) if T < 64 else 1, T=T, kv_heads=kv, dim=dim, cap=T + size(32, 4096))
        else:
            T = rng.choice([1, 1, size(2, 16), size(16, 2048)])
            n = max(T, size(32, 16384))
            w = rng.choice([0, size(16, 4096)])
            c = dict(op=op, T=T, n_kv=n, heads=heads, kv_heads=kv, dim=dim, window=w, sinks=rng.choice([0, 1, 4, 17]) if w else 0,
                     softcap=rng.choice([0.0, 0.0, 50.0]))
            if op == "kv4":
                c.update(seqs=size(1, 32) if T <= 16 else rng.choice([1, 2]), cap=n + rng.choice([0, size(1, 1000)]))
            else:
                c.update(stride=n + rng.choice([0, size(1, 1000)]))
        w = work(c)
        if all(w[k] <= max(m[k] for m in most) for k in w) and _plain_bytes(c) < 5e9:
            return c


def _plain_bytes(c):
    """What the plain form holds at once, about: fp32 scores and widened keys."""
    if c["op"] in ("kv4", "win"):
        s = c.get("seqs", 1)
        return 4 * s * (3 * c["heads"] * c["T"] * c["n_kv"] + 4 * c["kv_heads"] * c.get("cap", c["n_kv"]) * c["dim"])
    return 0


def _lens(c):
    """Lengths of the batch's sequences: the first is the full one, the others spread below it."""
    n, T = c["n_kv"], c["T"]
    return [max(T, n - (i * 2654435761 % 1009) * (n // 2) // 1009) if i else n for i in range(c["seqs"])]


def _pairs(c, n):
    """(visible pairs of one head, keys that some token sees) of a sequence of n keys."""
    T, w, s = c["T"], c["window"], c["sinks"]
    pairs = 0
    for t in range(T):
        p = n - T + t
        pairs += p + 1 if w == 0 or p + 1 <= w else w + min(s, p + 1 - w)
    first = max(0, n - T - w + 1) if w else 0
    return pairs, n - first + min(s, first)


def work(case):
    c, d = case, case["dim"]
    if c["op"] == "rope":
        v = c["seqs"] * c["T"] * (c["heads"] + c["kv_heads"]) * d
        return dict(bytes=v * ((4 if c["rows"] == "fp32" else 2) + 2), flops=10 * v)
    if c["op"] == "append":   # written to the cache, and read back from it
        v = c["seqs"] * c["T"] * c["kv_heads"] * 2 * d
        return dict(bytes=v * 4 + 2 * v * 5 // 8, flops=8 * v)
    pairs, keys = (sum(x) for x in zip(*(_pairs(c, n) for n in (_lens(c) if c["op"] == "kv4" else [c["n_kv"]]))))
    key = 2 * d * 5 // 8 if c["op"] == "kv4" else 4 * d
    return dict(bytes=keys * c["kv_heads"] * key + 4 * c.get("seqs", 1) * c["heads"] * c["T"] * d, flops=4 * d * pairs * c["heads"])


# ---- inputs ----------------------------------------------------------------------------

_DEV = "cuda"


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=torch.float32, device=_DEV).normal_(0.0, std, generator=g).to(dtype)


def _codes(x):
    """4-bit codes, scales and minima of the groups of fp16 rows: code * scale + minimum."""
    x = x.float().unflatten(-1, (-1, GROUP))
    lo = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - lo) / 15.0).half()
    f = s.float()
    c = torch.where(f > 0, torch.round((x - lo) / torch.where(f > 0, f, torch.ones_like(f))), torch.zeros_like(x)).clamp(0, 15)
    return c.to(torch.uint8).flatten(-2), torch.cat([s, lo.half()], -1)


def _layout(c):
    """Byte offsets of the cache's parts (key codes, key scales, value codes, value scales), and its size."""
    cap, d = (c["cap"] + 31) // 32 * 32, c["dim"]
    rows = c["seqs"] * c["kv_heads"] * cap
    at, parts = 0, []
    for size in (rows * d // 2, rows * d // GROUP * 4) * 2:
        parts.append((at, size))
        at = (at + size + 255) // 256 * 256
    return parts, at, cap


def _parts(c, cache):
    """The cache's parts as tensors: key codes [seq][head][key][dim/2], key (scale, minimum) [seq][head][key]
    [group][2], value codes [seq][head][key/8][dim/8][8 keys][4], value (scale, minimum) [..][key/8][group][8 keys][2]."""
    at, _, cap = _layout(c)
    S, H, d = c["seqs"], c["kv_heads"], c["dim"]
    kc, ks, vc, vs = (cache[a:a + n] for a, n in at)
    return (kc.view(S, H, cap, d // 2), ks.view(torch.float16).view(S, H, cap, d // GROUP, 2),
            vc.view(S, H, cap // 8, d // 8, 8, 4), vs.view(torch.float16).view(S, H, cap // 8, d // GROUP, 8, 2))


def _filled(c, g):
    """A cache whose every sequence holds random keys and values up to its capacity."""
    _, size, cap = _layout(c)
    cache = torch.zeros(size, dtype=torch.uint8, device=_DEV)
    kc, ks, vc, vs = _parts(c, cache)
    for s in range(c["seqs"]):
        for k in range(2):
            code, sm = _codes(_normal(g, (c["kv_heads"], cap, c["dim"]), 1.0, torch.float16))
            byte = code[..., 0::2] | code[..., 1::2] << 4
            if k == 0:
                kc[s], ks[s] = byte, sm
            else:
                vc[s] = byte.unflatten(1, (-1, 8)).unflatten(-1, (-1, 4)).transpose(2, 3)
                vs[s] = sm.unflatten(1, (-1, 8)).transpose(2, 3)
    return cache


def _inputs(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    d, T = c["dim"], c["T"]
    if c["op"] == "rope":   # fused rows: every query head, every key head, every value head
        rows, width = c["seqs"] * T, (c["heads"] + 2 * c["kv_heads"]) * d
        first = torch.randint(0, max(1, c["far"] - T), (c["seqs"], 1), generator=g, device=_DEV)
        j = torch.arange(c["rot"] // 2, device=_DEV, dtype=torch.float64)
        w = (_normal(g, (2, d), 0.2) + 1.0).half() if c["norm"] else None
        return dict(x=_normal(g, (rows, width), 1.5, torch.float16 if c["rows"] == "fp16" else torch.float32), w=w,
                    freq=(10000.0 ** (-2.0 * j / c["rot"])).float(), pos=(first + torch.arange(T, device=_DEV)).to(torch.int32).reshape(-1).contiguous())
    if c["op"] == "append":   # keys by head, values as the product's rows hold them
        H, S = c["kv_heads"], c["seqs"]
        last = torch.randint(T, c["cap"] + 1, (S,), generator=g, device=_DEV).to(torch.int32)
        if T > 1:   # a prompt stands at the front
            last.fill_(T)
        return dict(K=_normal(g, (S, H, T, d), 1.0, torch.float16), V=_normal(g, (S, T, H, d), 1.0, torch.float16), lens=last)
    if c["op"] == "kv4":
        return dict(cache=_filled(c, g), Q=_normal(g, (c["seqs"], c["heads"], T, d), 1.0, torch.float16),
                    lens=torch.tensor(_lens(c), dtype=torch.int32, device=_DEV))
    return dict(Q=_normal(g, (c["heads"], T, d), 1.0, torch.float16), K=_normal(g, (c["kv_heads"], c["stride"], d), 1.0, torch.float16),
                V=_normal(g, (c["kv_heads"], d, c["stride"]), 1.0, torch.float16))


def prepare(case, seed):
    c = dict(case)
    t = _inputs(c, seed)
    new = lambda *shape: torch.empty(shape, dtype=torch.float16, device=_DEV)  # noqa: E731
    S, T, d, H = c.get("seqs", 1), c["T"], c["dim"], c["kv_heads"]
    if c["op"] == "rope":
        t.update(q=new(S, c["heads"], T, d), k=new(S, H, T, d))
    elif c["op"] == "append":
        t.update(cache=torch.zeros(_layout(c)[1], dtype=torch.uint8, device=_DEV), k=new(S, H, T, d), v=new(S, H, T, d))
    else:
        t.update(out=new(*((S,) if c["op"] == "kv4" else ()), c["heads"], T, d))
    torch.cuda.synchronize()
    return dict(c=c, t=t)


# ---- the plain forms -------------------------------------------------------------------

def _plain_rope(c, t):
    S, T, d, nq, nk, rot = c["seqs"], c["T"], c["dim"], c["heads"], c["kv_heads"], c["rot"]
    x = t["x"][:, :(nq + nk) * d].float().view(S, T, nq + nk, d)
    if c["norm"]:
        w = torch.cat([t["w"][:1].float().expand(nq, d), t["w"][1:].float().expand(nk, d)])
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    a = t["pos"].double()[:, None] * t["freq"].double()
    cos, sin = (f(a).float().view(S, T, 1, rot // 2) for f in (torch.cos, torch.sin))
    if c["pairs"]:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    y = torch.cat([r, x[..., rot:]], -1).transpose(1, 2).half()
    return dict(q=y[:, :nq], k=y[:, nq:])


def _values(codes, sm, dtype):
    """code * scale + minimum of [..., dims] codes and [..., groups, 2] scales."""
    sm = sm.to(dtype)
    return (codes.to(dtype).unflatten(-1, (-1, GROUP)) * sm[..., :1] + sm[..., 1:]).flatten(-2)


def _plain_append(c, t):
    """The values that the tokens' codes and scales stand for."""
    codes = dict(k=_codes(t["K"]), v=_codes(t["V"].transpose(1, 2)))
    return {n: _values(code, sm, torch.float32).half() for n, (code, sm) in codes.items()}


def _unpacked(c, cache, dtype):
    """Keys and values [seq][head][key][dim] that the cache stands for."""
    kc, ks, vc, vs = _parts(c, cache)
    both = lambda b: torch.stack([b & 15, b >> 4], -1).flatten(-2)  # noqa: E731
    v = both(vc.transpose(3, 4).flatten(4)).flatten(2, 3)
    return _values(both(kc), ks, dtype), _values(v, vs.transpose(3, 4).flatten(2, 3), dtype)


def _visible(c, lens, n):
    """[seq][token][key]: whether the token sees the key."""
    p = (lens.long()[:, None] - c["T"] + torch.arange(c["T"], device=_DEV))[:, :, None]
    j = torch.arange(n, device=_DEV)
    see = j <= p
    return see & ((j > p - c["window"]) | (j < c["sinks"])) if c["window"] else see


def _attend(c, Q, K, V, see, dtype):
    """softmax over the visible keys: Q [seq][head][token][dim], K, V [seq][kv head][key][dim], see [seq][token][key]."""
    S, h, T, d = Q.shape
    H = K.shape[1]
    q = Q.to(dtype).view(S, H, h // H * T, d)
    s = torch.matmul(q, K.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    s = s.view(S, h, T, -1).masked_fill_(~see[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    o = torch.matmul(p.view(S, H, h // H * T, -1), V).view(S, h, T, -1)
    l = p.sum(-1, keepdim=True)
    return o / torch.where(l > 0, l, torch.ones_like(l))


def _plain(c, t):
    if c["op"] == "rope":
        return _plain_rope(c, t)
    if c["op"] == "append":
        return _plain_append(c, t)
    if c["op"] == "kv4":
        n = c["n_kv"]
        K, V = _unpacked(c, t["cache"], torch.float32)
        return _attend(c, t["Q"], K[:, :, :n], V[:, :, :n], _visible(c, t["lens"], n), torch.float32).half()
    n = c["n_kv"]
    see = _visible(c, torch.tensor([n], device=_DEV), n)
    return _attend(c, t["Q"][None], t["K"][None, :, :n].float(), t["V"][None, :, :, :n].float().transpose(2, 3), see, torch.float32)[0].half()


# ---- the library's calls ---------------------------------------------------------------

_lib = {}


def _session():
    """The library, a handle and the stream that its calls are queued on. It becomes torch's current stream, as in a program
    that queues its work on one stream: what reads a result, an event, a later input's allocation are all ordered with the
    calls. (A handle cannot be bound to the default stream, and its own does not wait for that one.)"""
    if not _lib:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocket-userspace_amd"))
        import rocketnpu as R
        lib, stream = R.load(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        fd = lib.rocket_open()
        assert fd >= 0, "no GPU"
        assert lib.rocket_hip_set_stream(fd, C.c_void_p(stream.cuda_stream)) == 0
        assert lib.rocket_hip_set_mode(fd, R.ROCKET_HIP_ASYNC | R.ROCKET_HIP_DEVICE_OPERANDS) == 0
        torch.cuda.set_stream(stream)
        _lib.update(R=R, lib=lib, stream=stream, fd=fd)
    return _lib


def _calls(c, t):
    """The entry points to call, with their arguments, and the outputs that they fill."""
    o = _session()
    R, lib, fd, p = o["R"], o["lib"], o["fd"], o["R"].ptr
    d, T, H = c["dim"], c["T"], c["kv_heads"]
    scale = 1.0 / math.sqrt(d)
    if c["op"] == "rope":
        fn = lib.rocket_qk_norm_rope_fp16 if c["rows"] == "fp16" else lib.rocket_qk_norm_rope_f32in
        x, w = t["x"], t["w"]
        return [(fn, (fd, c["seqs"], T, c["heads"], H, d, c["rot"], R.ROCKET_ROPE_PAIRS if c["pairs"] else R.ROCKET_ROPE_HALVES,
                      1e-6 if c["norm"] else -1.0, p(x), x.stride(0), p(x.data_ptr() + c["heads"] * d * x.element_size()), x.stride(0),
                      p(w[0]) if c["norm"] else None, p(w[1]) if c["norm"] else None, p(t["freq"]), p(t["pos"]), p(t["q"]), p(t["k"])))], dict(q=t["q"], k=t["k"])
    if c["op"] == "win":
        return [(lib.rocket_flash_attn_window_fp16, (fd, T, c["n_kv"], c["stride"], d, d, c["heads"], H, scale, c["softcap"], c["window"],
                                                     c["sinks"], p(t["Q"]), p(t["K"]), p(t["V"]), p(t["out"])))], t["out"]
    shape = R.Kv4Shape(c["seqs"], H, d, d, c["cap"])
    assert lib.rocket_kv4_bytes(C.byref(shape)) == t["cache"].numel()
    if c["op"] == "append":
        K, V = t["K"], t["V"]
        put = (fd, C.byref(shape), p(t["cache"]), 0, c["seqs"], T, p(K), K.stride(0), K.stride(1), K.stride(2),
               p(V), V.stride(0), V.stride(2), V.stride(1), p(t["lens"]))
        get = (fd, C.byref(shape), p(t["cache"]), 0, c["seqs"], T, p(t["lens"]), p(t["k"]), p(t["v"]))
        return [(lib.rocket_kv4_append_fp16, put), (lib.rocket_kv4_read_fp16, get)], dict(k=t["k"], v=t["v"])
    return [(lib.rocket_kv4_attn_fp16, (fd, C.byref(shape), p(t["cache"]), 0, c["seqs"], T, c["n_kv"], c["heads"], scale, c["softcap"],
                                        c["window"], c["sinks"], p(t["Q"]), p(t["lens"]), p(t["out"])))], t["out"]


def run(state):
    c, t = state["c"], state["t"]
    if not own:
        return _plain(c, t)
    if "calls" not in state:   # the arguments, as a program keeps them from step to step
        state["calls"], state["out"] = _calls(c, t)
        for x in t.values():   # (made on another stream, maybe: their memory is not reused before the calls are through)
            if torch.is_tensor(x):
                x.record_stream(_lib["stream"])
    for fn, args in state["calls"]:
        rc = fn(*args)
        if rc:
            raise RuntimeError("%s returned %d" % (fn.__name__, rc))
    return state["out"]


# ---- the definitions in 64 bits --------------------------------------------------------

def exact(case, seed):
    c = dict(case)
    t = _inputs(c, seed)
    S, T, d, H = c.get("seqs", 1), c["T"], c["dim"], c["kv_heads"]
    if c["op"] == "rope":
        h = c["heads"] + H
        y = t["x"].double()[:, :h * d].reshape(S, T, h, d)
        if c["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt()
            y[:, :, :c["heads"]] *= t["w"][0].double()
            y[:, :, c["heads"]:] *= t["w"][1].double()
        # a pair as a complex number, turned by its angle
        j = torch.arange(c["rot"] // 2, device=_DEV)
        a, b = (2 * j, 2 * j + 1) if c["pairs"] else (j, j + c["rot"] // 2)
        z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones((), dtype=torch.float64, device=_DEV),
                                                            t["pos"].double().view(S, T, 1, 1) * t["freq"].double())
        y[..., a], y[..., b] = z.real, z.imag
        y = y.permute(0, 2, 1, 3)
        return dict(q=y[:, :c["heads"]], k=y[:, c["heads"]:])
    if c["op"] == "append":
        r = {}
        for name, x in (("k", t["K"]), ("v", t["V"].permute(0, 2, 1, 3))):
            x = x.double().reshape(S, H, T, -1, GROUP)
            lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            s = ((hi - lo) / 15).half().double()
            q = ((x - lo) / s.clamp_min(1e-30)).round().clamp(0, 15) * (s > 0)
            r[name] = (lo + q * s).reshape(S, H, T, d)
        return r
    # one sequence and head at a time, the keys that a block of tokens sees
    if c["op"] == "kv4":
        kc, ks, vc, vs = _parts(c, t["cache"])
    outs, gqa = [], c["heads"] // H
    for i, n in enumerate(_lens(c) if c["op"] == "kv4" else [c["n_kv"]]):
        for hk in range(H):
            if c["op"] == "kv4":
                k = torch.empty((kc.shape[2], d), dtype=torch.float64, device=_DEV)
                v = torch.empty_like(k)
                k[:, 0::2], k[:, 1::2] = (kc[i, hk] & 15).double(), (kc[i, hk] >> 4).double()
                b = vc[i, hk].permute(0, 2, 1, 3).reshape(-1, d // 2)
                v[:, 0::2], v[:, 1::2] = (b & 15).double(), (b >> 4).double()
                for m, sm in ((k, ks[i, hk]), (v, vs[i, hk].permute(0, 2, 1, 3).reshape(-1, d // GROUP, 2))):
                    sm = sm.double().repeat_interleave(GROUP, 1)
                    m.mul_(sm[..., 0]).add_(sm[..., 1])
                k, v, q = k[:n], v[:n], t["Q"][i, hk * gqa:(hk + 1) * gqa].double()
            else:
                k, v, q = t["K"][hk, :n].double(), t["V"][hk, :, :n].double().t().contiguous(), t["Q"][hk * gqa:(hk + 1) * gqa].double()
            p, j = torch.arange(n - T, n, device=_DEV)[:, None], torch.arange(n, device=_DEV)[None]
            hidden = (j > p) | ((p - j >= c["window"]) & (j >= c["sinks"]) if c["window"] else j > p)
            for x in q:
                s = (x @ k.t()) * d ** -0.5
                if c["softcap"]:
                    s = c["softcap"] * (s / c["softcap"]).tanh()
                outs.append(s.masked_fill_(hidden, -math.inf).softmax(1) @ v)
    out = torch.stack(outs).view(S, c["heads"], T, d)
    return out if c["op"] == "kv4" else out[0]
