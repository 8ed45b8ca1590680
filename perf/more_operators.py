"""The feed-forward side of a serving layer in 8-bit floating point, as measurable calls: matrix products of e4m3
codes with a scale for each block of 128 (dense, and of experts whose rows the GPU counted), the quantisation that
makes their operands (rows, and gated rows), the norms before and after a block with its gate and residual scale (or
with the experts' weighted sum), and the routing of tokens to experts.

Where `own` is false, run() computes each operator in elementary torch operations, in 32 bits, with the router's
choices in 64; where it is true, it makes the library's calls."""
import ctypes as C
import math
import os
import sys

import torch

own = False

BLOCK = 128      # values of K (and rows of the weights) that share a scale
TOP = 448.0      # e4m3's largest finite value
TINY = 2.0 ** -100


def listed():
    return [
        # one token through a dense up product: a pass over the weights, latency
        dict(name="mm_token", op="mm", M=1, K=3840, N=15360, out="fp16"),
        # drafted tokens of a batch, fp32 results; no size a multiple of a tile, the last block of K a part of one
        dict(name="mm_ragged", op="mm", M=77, K=2080, N=1000, out="fp32"),
        # a prompt chunk through a dense down product: long rows, few tiles
        dict(name="mm_chunk", op="mm", M=512, K=15360, N=3840, out="fp16"),
        # a long prompt through a dense up product, the largest call
        dict(name="mm_prefill", op="mm", M=4096, K=3840, N=15360, out="fp16"),
        # a decode batch of 16 tokens, each to 6 of 64 experts: most experts have a row or two
        dict(name="moe_decode", op="moe", tokens=16, experts=64, top=6, K=2048, N=2816, gather=True, out="fp16"),
        # a long prompt's tokens to the same experts, whose shares differ
        dict(name="moe_prefill", op="moe", tokens=4096, experts=64, top=6, K=2048, N=2816, gather=True, out="fp16"),
        # fp32 rows of a prompt chunk become a down product's operand
        dict(name="quant_chunk", op="quant", M=512, K=15360, rows="fp32", act="none"),
        # gated rows of a prompt's experts become theirs
        dict(name="quant_gated", op="quant", M=24576, K=1408, rows="fp16", act="silu"),
        # behind the experts of a decode batch: weighted sum, norm, residual, the next block's norm; latency
        dict(name="norm_decode", op="norm", M=16, H=2048, rows="fp16", top=6, shared=True, post=True, gate=0, codes=True, plain=True),
        # behind a dense block of a long prompt: fp32 rows, a gate a sequence, codes for the next product
        dict(name="norm_prefill", op="norm", M=4096, H=3840, rows="fp32", top=0, shared=False, post=True, gate=1024, codes=True, plain=False),
        # the router of a decode batch: latency
        dict(name="route_decode", op="route", M=16, E=64, score="softmax", bias=False, groups=1, best=1, top_groups=1, top=6, renorm=True, off=0.0),
        # a long prompt through a router with balancing biases and groups
        dict(name="route_prefill", op="route", M=8192, E=256, score="sigmoid", bias=True, groups=8, best=2, top_groups=4, top=8, renorm=True, off=0.0),
    ]


def draw(rng):
    def size(lo, hi, step=1):   # log-uniform, a multiple of step
        return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step

    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(["mm", "mm", "mm", "moe", "moe", "quant", "norm", "norm", "route"])
        if op == "mm":
            c = dict(op=op, M=rng.choice([1, size(2, 64), size(64, 8192)]), K=size(64, 16384, 16), N=size(32, 16384, rng.choice([1, 8])),
                     out=rng.choice(["fp16", "fp32"]))
        elif op == "moe":
            E = rng.choice([8, 16, 60, 64, 128])
            c = dict(op=op, tokens=rng.choice([size(1, 64), size(64, 4096)]), experts=E, top=rng.choice([1, 2, 4, 6, 8]), K=size(256, 4096, 16),
                     N=size(256, 4096, 8), gather=rng.random() < 0.5, out=rng.choice(["fp16", "fp32"]))
        elif op == "quant":
            c = dict(op=op, M=size(1, 32768), K=size(64, 16384, 8), rows=rng.choice(["fp16", "fp32"]), act=rng.choice(["none", "silu", "gelu"]))
        elif op == "norm":
            top, M = rng.choice([0, 0, 2, 8]), size(1, 8192)
            c = dict(op=op, M=M, H=size(256, 8192, 8), rows=rng.choice(["fp16", "fp32"]), top=top, shared=top > 0 and rng.random() < 0.5,
                     post=rng.random() < 0.6, gate=rng.choice([0, 1, max(1, M // 3), M]), codes=rng.random() < 0.6, plain=True)
            c["plain"] = not c["codes"] or rng.random() < 0.5
        else:
            E, g = rng.choice([(8, 1), (60, 1), (64, 8), (128, 4), (256, 8), (257, 1), (384, 1), (512, 16)])
            tg = max(1, g // 2)
            best = 1 if g == 1 else rng.choice([1, 2])
            c = dict(op=op, M=rng.choice([size(1, 64), size(64, 16384)]), E=E, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=g,
                     best=best, top_groups=tg, top=min(rng.choice([1, 2, 6, 8]), E // g * tg), renorm=rng.random() < 0.7, off=rng.choice([0.0, 0.0, 0.3]))
        w = work(c)
        if all(w[k] <= max(m[k] for m in most) for k in w) and _plain_bytes(c) < 8e9:
            return c


def _blocks(n):
    return -(-n // BLOCK)


def _size(name):
    return 2 if name == "fp16" else 4


def _plain_bytes(c):
    """What the plain form holds at once, about: fp32 operands and their products."""
    if c["op"] == "mm":
        return 8 * (c["M"] * c["K"] + c["N"] * c["K"]) + 8 * c["M"] * c["N"]
    if c["op"] == "moe":
        rows = 4 * max(c["tokens"] * c["top"], c["experts"])
        return 12 * c["experts"] * c["N"] * c["K"] + 8 * rows * (c["K"] + c["N"])
    if c["op"] == "quant":
        return 24 * c["M"] * c["K"]
    if c["op"] == "norm":
        return 4 * c["M"] * c["H"] * (8 + 2 * c["top"])
    return 8 * c["M"] * c["E"] * 8


def work(case):
    c = case
    if c["op"] == "mm":
        M, K, N = c["M"], c["K"], c["N"]
        return dict(bytes=(M + N) * K + 4 * (M + _blocks(N)) * _blocks(K) + M * N * _size(c["out"]), flops=2 * M * N * K)
    if c["op"] == "moe":   # (experts that get a row, about: as if tokens chose evenly)
        E, K, N, rows = c["experts"], c["K"], c["N"], c["tokens"] * c["top"]
        used = E * (1.0 - (1.0 - min(1.0, c["top"] / E)) ** c["tokens"])
        read = min(rows, c["tokens"]) if c["gather"] else rows
        return dict(bytes=read * (K + 4 * _blocks(K)) + used * (N * K + 4 * _blocks(N) * _blocks(K)) + rows * N * _size(c["out"]), flops=2 * rows * N * K)
    if c["op"] == "quant":
        v = c["M"] * c["K"]
        return dict(bytes=v * _size(c["rows"]) * (1 if c["act"] == "none" else 2) + v + 4 * c["M"] * _blocks(c["K"]), flops=(3 if c["act"] == "none" else 10) * v)
    if c["op"] == "norm":
        v, e = c["M"] * c["H"], _size(c["rows"])
        gate = 2 * c["H"] * -(-c["M"] // c["gate"]) if c["gate"] else 0
        read = v * e * (1 + (c["top"] or 1) + c["shared"]) + 8 * c["M"] * c["top"] + gate + 4 * c["H"]
        return dict(bytes=read + v * e + (2 * v if c["plain"] else 0) + (v + 4 * c["M"] * _blocks(c["H"]) if c["codes"] else 0), flops=v * (10 + 2 * c["top"]))
    return dict(bytes=4 * c["M"] * c["E"] + 16 * c["M"] * c["top"] + 4 * (c["E"] + 1), flops=c["M"] * c["E"] * 12)


# ---- inputs ----------------------------------------------------------------------------

_DEV = "cuda"
_F8 = torch.float8_e4m3fn
_TYPE = dict(fp16=torch.float16, fp32=torch.float32)


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=torch.float32, device=_DEV).normal_(0.0, std, generator=g).to(dtype)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % cols, 0, -x.shape[-2] % rows))


def _quantised(x, rows):
    """Codes (as bytes) and scales of x[..., N, K], one scale for each block of rows x BLOCK values."""
    N, K = x.shape[-2:]
    b = _padded(x, rows, BLOCK).unflatten(-2, (-1, rows)).unflatten(-1, (-1, BLOCK))
    a = b.abs().amax((-3, -1)).clamp_min(TINY)
    q = (b * (TOP / a)[..., :, None, :, None]).clamp(-TOP, TOP).to(_F8).view(torch.uint8)
    return q.flatten(-2).flatten(-3, -2)[..., :N, :K].contiguous(), (a / TOP).contiguous()


def _inputs(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    op = c["op"]
    if op in ("mm", "moe"):
        K, N = c["K"], c["N"]
        lots = () if op == "mm" else (c["experts"],)
        # weights' blocks and activations' columns of unlike sizes, as trained ones have
        w = _normal(g, (*lots, N, K), 0.02) * torch.exp(_normal(g, (*lots, N, 1), 0.3))
        B, sb = _quantised(w, BLOCK)
        del w
        rows = c["M"] if op == "mm" else c["tokens"] if c["gather"] else c["tokens"] * c["top"]
        A, sa = _quantised(_normal(g, (rows, K)) * torch.exp(_normal(g, (1, K), 0.5)), 1)
        t = dict(A=A, sa=sa, B=B, sb=sb)
        if op == "moe":
            E, top = c["experts"], c["top"]
            like = _normal(g, (c["tokens"], E)) + _normal(g, (1, E), 0.5)
            ids = torch.sort(like, dim=1, descending=True, stable=True).indices[:, :top].reshape(-1)
            order = torch.sort(ids, dim=0, stable=True)
            off = torch.searchsorted(order.values, torch.arange(E + 1, device=_DEV))
            t.update(off=off.to(torch.int32), src=(order.indices // top).to(torch.int32), most=int((off[1:] - off[:-1]).max()))
        return t
    if op == "quant":
        width = c["K"] * (1 if c["act"] == "none" else 2)   # gate and up side by side, as one product writes them
        return dict(x=_normal(g, (c["M"], width), 1.5, _TYPE[c["rows"]]))
    if op == "norm":
        M, H, dt = c["M"], c["H"], _TYPE[c["rows"]]
        t = dict(h=_normal(g, (M, H), 2.0, dt), pre=(1 + _normal(g, (H,), 0.2)).half())
        t["y"] = _normal(g, (M * max(1, c["top"]), H), 1.0, dt)
        if c["top"]:
            t["slot"] = torch.randperm(M * c["top"], generator=g, device=_DEV).view(M, c["top"]).to(torch.int32)
            w = torch.rand((M, c["top"]), generator=g, device=_DEV)
            t["weight"] = w / w.sum(1, keepdim=True)
        if c["shared"]:
            t["shared"] = _normal(g, (M, H), 1.0, dt)
        if c["post"]:
            t["post"] = (1 + _normal(g, (H,), 0.2)).half()
        if c["gate"]:
            t["gate"] = _normal(g, (-(-M // c["gate"]), H), 0.5, torch.float16)
        return t
    logits = _normal(g, (c["M"], c["E"]), 1.5)
    if c["off"]:   # experts that some tokens must not take
        logits = logits.masked_fill_(torch.rand((c["M"], c["E"]), generator=g, device=_DEV) < c["off"], -math.inf)
    return dict(logits=logits, bias=_normal(g, (c["E"],), 0.05) if c["bias"] else None)


def prepare(case, seed):
    c = dict(case)
    t = _inputs(c, seed)
    new = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device=_DEV)  # noqa: E731
    op = c["op"]
    if op in ("mm", "moe"):
        t["out"] = new(c["M"] if op == "mm" else c["tokens"] * c["top"], c["N"], dtype=_TYPE[c["out"]])
    elif op == "quant":
        t.update(codes=new(c["M"], c["K"], dtype=torch.uint8), scale=new(c["M"], _blocks(c["K"]), dtype=torch.float32))
    elif op == "norm":
        M, H = c["M"], c["H"]
        t["h_out"] = new(M, H, dtype=_TYPE[c["rows"]])
        if c["plain"]:
            t["x"] = new(M, H, dtype=torch.float16)
        if c["codes"]:
            t.update(codes=new(M, H, dtype=torch.uint8), scale=new(M, _blocks(H), dtype=torch.float32))
    else:
        M, k = c["M"], c["top"]
        t.update(ids=new(M, k, dtype=torch.int32), weight=new(M, k, dtype=torch.float32), offsets=new(c["E"] + 1, dtype=torch.int32),
                 src=torch.full((M * k,), -1, dtype=torch.int32, device=_DEV), slot=new(M, k, dtype=torch.int32))
    torch.cuda.synchronize()
    return dict(c=c, t=t)


# ---- the plain forms -------------------------------------------------------------------

def _values(q, s, rows):
    """What codes q[..., N, K] with one scale for each block of rows x BLOCK stand for, in fp32."""
    N, K = q.shape[-2:]
    s = s.repeat_interleave(BLOCK, -1)[..., :K]
    s = s.repeat_interleave(rows, -2)[..., :N, :] if rows > 1 else s
    return q.view(_F8).float() * s


def _plain_moe(c, t):
    """Every expert's rows side by side, filled up to the longest, and one batched product."""
    off, rows = t["off"].long(), c["tokens"] * c["top"]
    a = _values(t["A"], t["sa"], 1)
    a = a[t["src"].long()] if c["gather"] else a
    j = torch.arange(t["most"], device=_DEV)
    x = a[(off[:-1, None] + j).clamp_max(rows - 1)]
    y = torch.bmm(x, _values(t["B"], t["sb"], BLOCK).transpose(1, 2).contiguous())
    r = torch.arange(rows, device=_DEV)
    e = torch.searchsorted(off[1:].contiguous(), r, right=True)
    return y[e, r - off[e]].to(_TYPE[c["out"]])


def _coded(x):
    """e4m3 codes and scales of the groups of BLOCK of fp32 rows."""
    K = x.shape[1]
    b = torch.nn.functional.pad(x, (0, -K % BLOCK)).unflatten(1, (-1, BLOCK))
    a = b.abs().amax(2).clamp_min(TINY)
    q = (b * (TOP / a)[..., None]).clamp(-TOP, TOP).flatten(1)[:, :K].to(_F8)
    return dict(codes=q, scale=a / TOP)


def _act(name, x):
    return x * 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) if name == "gelu" else x / (1.0 + torch.exp(-x))


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * w.float()


def _plain_norm(c, t):
    y = t["y"].float()
    if c["top"]:
        y = (y[t["slot"].long()] * t["weight"][:, :, None]).sum(1)
    if c["shared"]:
        y = y + t["shared"].float()
    if c["post"]:
        y = _rms(y, t["post"])
    if c["gate"]:
        y = y * t["gate"].float()[torch.arange(c["M"], device=_DEV) // c["gate"]]
    h = t["h"].float() + 0.75 * y
    x = _rms(h, t["pre"])
    return dict(h=h.to(t["h"].dtype), **(dict(x=x.half()) if c["plain"] else {}), **(_coded(x) if c["codes"] else {}))


def _plain_route(c, t):
    x, E, k, g = t["logits"].double(), c["E"], c["top"], c["groups"]
    can = x > -math.inf
    if c["score"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True).clamp_min(-1e300))
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    choice = (p + t["bias"].double() if c["bias"] else p).masked_fill(~can, -math.inf)
    key = choice if c["bias"] else x   # (without a bias the logits' order is the scores')
    if g > 1:
        two = torch.sort(choice.unflatten(1, (g, -1)), dim=2, descending=True).values[..., :c["best"]]
        value = two.masked_fill(two == -math.inf, 0.0).sum(2).masked_fill(two[..., 0] == -math.inf, -math.inf)
        pick = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        in_group = (pick[:, :, None] == torch.arange(g, device=_DEV)).any(1).repeat_interleave(E // g, 1)
        key = key.masked_fill(~in_group, -math.inf)
    best = torch.sort(key, dim=1, descending=True, stable=True)
    none = best.values[:, :k] == -math.inf
    ids = best.indices[:, :k].masked_fill(none, -1)
    w = torch.gather(p, 1, ids.clamp_min(0)).masked_fill(none, 0.0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    # the rows by expert, then by token
    flat = ids.masked_fill(none, E).reshape(-1)
    order = torch.sort(flat, dim=0, stable=True)
    off = torch.searchsorted(order.values, torch.arange(E + 1, device=_DEV))
    r = torch.arange(flat.numel(), device=_DEV)
    src = torch.where(order.values < E, order.indices // k, -1)
    slot = torch.empty_like(flat).scatter_(0, order.indices, r).view(-1, k).masked_fill(none, -1)
    return dict(ids=ids.to(torch.int32), weight=(2.5 * w).float(), offsets=off.to(torch.int32), src=src.to(torch.int32), slot=slot.to(torch.int32))


def _plain(c, t):
    if c["op"] == "mm":
        return torch.matmul(_values(t["A"], t["sa"], 1), _values(t["B"], t["sb"], BLOCK).t()).to(_TYPE[c["out"]])
    if c["op"] == "moe":
        return _plain_moe(c, t)
    if c["op"] == "quant":
        x, K = t["x"].float(), c["K"]
        return _coded(x if c["act"] == "none" else _act(c["act"], x[:, :K]) * x[:, K:])
    return _plain_norm(c, t) if c["op"] == "norm" else _plain_route(c, t)


# ---- the library's calls ---------------------------------------------------------------

_lib = {}


def _session():
    """The library, a handle and the stream that its calls are queued on, which becomes torch's current stream, as in a
    program that queues its work on one stream."""
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


def _call(c, t):
    """The entry point to call, with its arguments, and the outputs that it fills."""
    o = _session()
    R, lib, fd, p = o["R"], o["lib"], o["fd"], o["R"].ptr
    act = dict(silu=R.ROCKET_ACTIVATION_SILU, gelu=R.ROCKET_ACTIVATION_GELU)
    if c["op"] == "mm":
        fn = lib.rocket_matmul_fp8_block_f16out if c["out"] == "fp16" else lib.rocket_matmul_fp8_block
        return fn, (fd, c["M"], c["K"], c["N"], p(t["A"]), p(t["sa"]), p(t["B"]), p(t["sb"]), p(t["out"])), t["out"]
    if c["op"] == "moe":
        fn = lib.rocket_matmul_fp8_block_grouped_f16out if c["out"] == "fp16" else lib.rocket_matmul_fp8_block_grouped
        return fn, (fd, c["experts"], c["tokens"] * c["top"], t["A"].shape[0], c["K"], c["N"], p(t["A"]), p(t["sa"]), p(t["src"]) if c["gather"] else None,
                    p(t["off"]), p(t["B"]), p(t["sb"]), p(t["out"])), t["out"]
    if c["op"] == "quant":
        x, K, out = t["x"], c["K"], dict(codes=t["codes"].view(_F8), scale=t["scale"])
        if c["act"] == "none":
            fn = lib.rocket_quantize_rows_fp8_fp16 if c["rows"] == "fp16" else lib.rocket_quantize_rows_fp8
            return fn, (fd, c["M"], K, p(x), x.stride(0), p(t["codes"]), p(t["scale"])), out
        fn = lib.rocket_quantize_glu_fp8_fp16 if c["rows"] == "fp16" else lib.rocket_quantize_glu_fp8
        return fn, (fd, c["M"], K, p(x), p(x.data_ptr() + K * x.element_size()), x.stride(0), act[c["act"]], None, p(t["codes"]), p(t["scale"])), out
    if c["op"] == "norm":
        M, H = c["M"], c["H"]
        out = dict(h=t["h_out"], **(dict(x=t["x"]) if c["plain"] else {}), **(dict(codes=t["codes"].view(_F8), scale=t["scale"]) if c["codes"] else {}))
        tail = (p(t.get("post")), 1e-6 if c["post"] else -1.0, p(t.get("gate")), c["gate"] or 1, 0.75, p(t["pre"]), 1e-6, p(t["h_out"]), p(t.get("x")),
                p(t.get("codes")), p(t.get("scale")))
        if c["top"]:
            fn = lib.rocket_moe_add_norm_fp16 if c["rows"] == "fp16" else lib.rocket_moe_add_norm_f32
            return fn, (fd, M, H, p(t["h"]), M * c["top"], c["top"], p(t["y"]), p(t["slot"]), p(t["weight"]), p(t.get("shared")), *tail), out
        fn = lib.rocket_add_norm_fp16 if c["rows"] == "fp16" else lib.rocket_add_norm_f32
        return fn, (fd, M, H, p(t["h"]), p(t["y"]), H, *tail), out
    out = {n: t[n] for n in ("ids", "weight", "offsets", "src", "slot")}
    return lib.rocket_moe_route_f32, (fd, c["M"], c["E"], p(t["logits"]), c["E"], R.ROCKET_ROUTE_SIGMOID if c["score"] == "sigmoid" else R.ROCKET_ROUTE_SOFTMAX,
                                      p(t["bias"]), c["groups"], c["best"], c["top_groups"], c["top"], int(c["renorm"]), 2.5, None, p(t["ids"]), p(t["weight"]),
                                      p(t["offsets"]), p(t["src"]), p(t["slot"])), out


def run(state):
    c, t = state["c"], state["t"]
    if not own:
        return _plain(c, t)
    if "call" not in state:   # the arguments, as a program keeps them from step to step
        state["call"] = _call(c, t)
        for x in t.values():   # (made on another stream, maybe: their memory is not reused before the calls are through)
            if torch.is_tensor(x):
                x.record_stream(_lib["stream"])
    fn, args, out = state["call"]
    rc = fn(*args)
    if rc:
        raise RuntimeError("%s returned %d" % (fn.__name__, rc))
    return out


# ---- the definitions in 64 bits --------------------------------------------------------

def _wide(q, s, rows):
    """Codes with their blocks' scales in 64 bits, a block of K at a time."""
    v = q.view(_F8).double()
    at = torch.arange(v.shape[0], device=_DEV) // rows
    for b in range(s.shape[1]):
        v[:, b * BLOCK:(b + 1) * BLOCK] *= s[at, b].double()[:, None]
    return v


def _norm64(x, w):
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()


def _codes64(x):
    """(The codes' values, no rounding to e4m3 among them, have no 64-bit form: None.)"""
    K = x.shape[1]
    return dict(codes=None, scale=torch.stack([x[:, i:i + BLOCK].abs().amax(1).clamp_min(TINY) for i in range(0, K, BLOCK)], 1) / TOP)


def exact(case, seed):
    c = dict(case)
    t = _inputs(c, seed)
    if c["op"] == "mm":
        a = _wide(t["A"], t["sa"], 1)
        return torch.cat([a @ _wide(t["B"][i:i + 4096], t["sb"][i // BLOCK:(i + 4096) // BLOCK], BLOCK).t() for i in range(0, c["N"], 4096)], 1)
    if c["op"] == "moe":
        a, off = _wide(t["A"], t["sa"], 1), t["off"].tolist()
        out = torch.empty((c["tokens"] * c["top"], c["N"]), dtype=torch.float64, device=_DEV)
        for e in range(c["experts"]):
            i, j = off[e], off[e + 1]
            if j > i:
                out[i:j] = a[t["src"][i:j].long() if c["gather"] else slice(i, j)] @ _wide(t["B"][e], t["sb"][e], BLOCK).t()
        return out
    if c["op"] == "quant":
        x = t["x"].double()
        if c["act"] != "none":
            g, u = x.chunk(2, 1)
            x = (g * torch.special.ndtr(g) if c["act"] == "gelu" else g * torch.sigmoid(g)) * u
        return _codes64(x)
    if c["op"] == "norm":
        y = t["y"].double()
        if c["top"]:
            y = sum(y[t["slot"][:, j].long()] * t["weight"][:, j:j + 1].double() for j in range(c["top"]))
        if c["shared"]:
            y = y + t["shared"].double()
        if c["post"]:
            y = _norm64(y, t["post"])
        if c["gate"]:
            y = y * t["gate"].double().repeat_interleave(c["gate"], 0)[:c["M"]]
        h = t["h"].double() + 0.75 * y
        x = _norm64(h, t["pre"])
        return dict(h=h, **(dict(x=x) if c["plain"] else {}), **(_codes64(x) if c["codes"] else {}))
    # the weights; the choices are whole numbers, which both sides have alike
    x, ids = t["logits"].double(), _plain_route(c, t)["ids"].long()
    p = x.softmax(1).nan_to_num(0.0) if c["score"] == "softmax" else x.sigmoid()
    w = torch.gather(p, 1, ids.clamp_min(0)) * (ids >= 0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return dict(ids=None, weight=2.5 * w, offsets=None, src=None, slot=None)
