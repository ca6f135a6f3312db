"""Cases for the operators of a decoder's attention layer around ``tattn.attention``:

* ``qk_norm_rope``: norm of every query and key head with the position rotation, and its gradients;
* ``window_attention``: causal attention with a sliding window and first tokens that stay visible, and
  its gradients; ``decode_attention``: its form for one new token over a cache of keys and values;
* ``Int4Cache``: a cache held in 4 bits: appending, reading back, and the single-token attention over it.

``run`` computes them in elementary torch operations in 32 bits, or, with ``own``, by the calls a user
makes of ``tattn``; ``exact`` computes them from their definitions in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}
GROUP = 64  # head dims that share a scale and a minimum in the 4-bit cache
ODD = (1, 17, 33, 70, 1000)  # lengths that fill no block


# ------------------------------------------------------------------------------------------ cases
def _rope(name, b, h, hk, n, d, dtype, grad, interleaved, layout):
    return dict(name=name, op="rope", b=b, h=h, hk=hk, n=n, d=d, dtype=dtype, grad=grad, interleaved=interleaved, layout=layout)


def _window(name, b, h, hk, nq, nk, d, window, sinks, dtype, grad):
    return dict(name=name, op="window", b=b, h=h, hk=hk, nq=nq, nk=nk, d=d, window=window, sinks=sinks, dtype=dtype, grad=grad)


def _token(name, b, h, hk, cap, d, window, sinks, spread, dtype):
    return dict(name=name, op="token", b=b, h=h, hk=hk, cap=cap, d=d, window=window, sinks=sinks, spread=spread, dtype=dtype)


def _fill(name, b, hk, t, start, d):
    return dict(name=name, op="fill4", b=b, hk=hk, t=t, start=start, d=d)


def _attend(name, b, h, hk, cap, d, window, sinks, spread):
    return dict(name=name, op="attend4", b=b, h=h, hk=hk, cap=cap, d=d, window=window, sinks=sinks, spread=spread)


def listed():
    return [
        # One decoding step of a small batch: the new token's heads, where latency counts.
        _rope("rope_token", 8, 16, 4, 1, 128, "f16", False, False, "bnhd"),
        # A training step's queries and keys as the projections leave them ([batch, seq, heads, dim]).
        _rope("rope_train", 4, 16, 4, 4096, 64, "f16", True, False, "bnhd"),
        # 32-bit training at an odd length, neighbouring dims rotated together.
        _rope("rope_train_f32", 3, 5, 5, 1000, 32, "f32", True, True, "bhnd"),
        # Training at the benchmark's B4 H16 N4096 D64, a quarter of the keys visible.
        _window("window_train", 4, 16, 16, 4096, 4096, 64, 1024, 4, "f16", True),
        # Training with shared heads, odd length, odd window, sinks that end inside a block's neighbour.
        _window("window_train_gqa", 2, 16, 4, 2500, 2500, 128, 777, 130, "f16", True),
        # 32-bit training, small and odd.
        _window("window_train_f32", 3, 5, 5, 1000, 1000, 64, 200, 4, "f32", True),
        # A long prompt's last chunk against everything before it.
        _window("window_prompt", 1, 16, 4, 4096, 16384, 64, 4096, 4, "f16", False),
        # One new token of one sequence, window only: latency.
        _token("window_token", 1, 16, 4, 1000, 64, 512, 4, 0, "f16"),
        # One new token of each of 64 sequences of unequal lengths.
        _token("window_token_batch", 64, 16, 4, 8192, 128, 4096, 4, 4000, "f16"),
        # A prompt enters the 4-bit cache and is read back for the next chunk.
        _fill("cache4_fill", 4, 4, 4096, 0, 128),
        # One new token over a short 4-bit cache: latency.
        _attend("cache4_token", 1, 16, 4, 1000, 64, 0, 0, 0),
        # One new token of each of 16 sequences over long 4-bit caches.
        _attend("cache4_long", 16, 16, 4, 65536, 128, 0, 0, 30000),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even in the logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    return n - 1 if n == 3072 else n


def _heads(rng):
    hk = rng.choice((1, 2, 3, 4, 5, 8, 16))
    return hk * rng.choice((1, 1, 2, 3, 4, 8)), hk


def draw(rng):
    op = rng.choice(("rope", "window", "window", "token", "fill4", "attend4"))
    h, hk = _heads(rng)
    d = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("f16", "f16", "f16", "f32"))
    if op == "rope":
        b = rng.choice((1, 2, 3, 4, 8))
        n = rng.choice((rng.choice(ODD), _log(rng, 1, 4096)))
        n = max(1, min(n, 4 * 4096 * 20 * 64 // (b * (h + hk) * d)))
        c = _rope("", b, h, hk, n, d, dtype, rng.random() < 0.7, rng.random() < 0.3, rng.choice(("bnhd", "bhnd")))
    elif op == "window":
        b = rng.choice((1, 2, 3, 4))
        most = 230_000_000 * 64 // max(d, 64) if dtype == "f16" else 30_000_000
        nq = min(_log(rng, 1, 4096), int(math.sqrt(most / (b * h))))
        nk = nq if rng.random() < 0.6 else nq + _log(rng, 1, 4096)
        nk = max(nq, min(nk, most // (b * h * nq)))
        sinks = rng.choice((0, 1, 4, _log(rng, 1, 300)))
        c = _window("", b, h, hk, nq, nk, d, _log(rng, 1, 4096), sinks, dtype, rng.random() < 0.6)
    elif op == "token":
        b = rng.choice((1, 2, 7, 16, 64))
        cap = min(_log(rng, 1, 32768), 64 * 4 * 8192 * 128 // (b * hk * d))
        window = 0 if rng.random() < 0.3 else _log(rng, 1, 8192)
        c = _token("", b, h, hk, cap, d, window, rng.choice((0, 1, 4, 33)), rng.randint(0, cap - 1), dtype)
    elif op == "fill4":
        b, d = rng.choice((1, 2, 7, 16, 64)), rng.choice((64, 128))
        t = max(1, min(rng.choice((1, _log(rng, 1, 4096))), 4 * 4 * 4096 * 128 // (b * hk * d)))
        c = _fill("", b, hk, t, rng.choice((0, rng.randint(0, 2000))), d)
    else:
        b, d = rng.choice((1, 2, 7, 16, 64)), rng.choice((64, 128))
        cap = min(_log(rng, 1, 65536), 16 * 4 * 65536 * 128 // (b * hk * d))
        window = 0 if rng.random() < 0.6 else _log(rng, 1, 8192)
        c = _attend("", b, h, hk, cap, d, window, rng.choice((0, 1, 4, 33)), rng.randint(0, cap - 1))
    del c["name"]
    return c


def _lengths(c):
    """Tokens held for each sequence, the newest among them: between cap - spread and cap."""
    return [c["cap"] - (i * 7919) % (c["spread"] + 1) for i in range(c["b"])]


# ------------------------------------------------------------------------------------------ inputs
def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "rope":
        dt, b, n, d = DTYPES[c["dtype"]], c["b"], c["n"], c["d"]

        def heads(h):
            if c["layout"] == "bnhd":
                return _randn(g, (b, n, h, d), dt).transpose(1, 2)
            return _randn(g, (b, h, n, d), dt)

        s["q"], s["k"], s["dq"], s["dk"] = heads(c["h"]), heads(c["hk"]), heads(c["h"]), heads(c["hk"])
        s["wq"], s["wk"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
        # Sequences that begin at different places of the tables, as in decoding and in packed batches.
        first = torch.randint(0, 4096, (b, 1), generator=g, device="cuda", dtype=torch.int32)
        s["positions"] = first + torch.arange(n, device="cuda", dtype=torch.int32)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angle = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if c["grad"]:
            for key in ("q", "k", "wq", "wk"):
                s[key].requires_grad_()
    elif c["op"] == "window":
        dt = DTYPES[c["dtype"]]
        s["q"] = _randn(g, (c["b"], c["h"], c["nq"], c["d"]), dt)
        s["k"] = _randn(g, (c["b"], c["hk"], c["nk"], c["d"]), dt)
        s["v"] = _randn(g, (c["b"], c["hk"], c["nk"], c["d"]), dt)
        s["do"] = _randn(g, (c["b"], c["h"], c["nq"], c["d"]), dt)
        if c["grad"]:
            for key in ("q", "k", "v"):
                s[key].requires_grad_()
    elif c["op"] == "token":
        dt = DTYPES[c["dtype"]]
        s["q"] = _randn(g, (c["b"], c["h"], 1, c["d"]), dt)
        s["k"] = _randn(g, (c["b"], c["hk"], c["cap"], c["d"]), dt)
        s["v"] = _randn(g, (c["b"], c["hk"], c["cap"], c["d"]), dt)
        s["lengths"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)
    elif c["op"] == "fill4":
        shape = (c["b"], c["hk"], c["t"], c["d"])
        s["k"], s["v"] = _randn(g, shape, torch.float16), _randn(g, shape, torch.float16)
        s["start"] = torch.full((c["b"],), c["start"], device="cuda", dtype=torch.int32)
        s["cache"] = _empty_cache(c["b"], c["hk"], c["start"] + c["t"], c["d"])
    else:
        s["q"] = _randn(g, (c["b"], c["h"], 1, c["d"]), torch.float16)
        s["lengths"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)
        shape = (c["b"], c["hk"], c["cap"], c["d"])
        cache = _empty_cache(c["b"], c["hk"], c["cap"], c["d"])
        for x in ("k", "v"):
            # Codes and, around the scales of normal heads, their scales and minima.
            cache[x + "_codes"].random_(0, 256, generator=g)
            scale = 0.25 + 0.1 * torch.rand(shape[:3] + (c["d"] // GROUP,), generator=g, device="cuda")
            low = -7.5 * scale + 0.3 * torch.randn(scale.shape, generator=g, device="cuda")
            cache[x + "_params"].copy_(torch.stack((scale, low), -1))
        s["cache"] = cache
    return s


def _empty_cache(b, hk, cap, d):
    """The 4-bit cache's tensors: codes (two head dims a byte, the even one in the low half) and, for each
    group of 64 head dims of a token's head, its scale and minimum."""
    cache = {}
    for x in ("k", "v"):
        cache[x + "_codes"] = torch.zeros((b, hk, cap, d // 2), device="cuda", dtype=torch.uint8)
        cache[x + "_params"] = torch.zeros((b, hk, cap, d // GROUP, 2), device="cuda", dtype=torch.float16)
    return cache


# -------------------------------------------------------------------------------------- plain forms
def _turn(z, cos, sin, interleaved):
    if interleaved:
        a, b = z[..., 0::2], z[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = z.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_rope(x, w, cos, sin, interleaved, dy, eps=1e-6):
    x32, w32 = x.detach().float(), w.detach().float()
    r = torch.rsqrt(x32.square().mean(-1, keepdim=True) + eps)
    xr = x32 * r
    y = _turn(xr * w32, cos, sin, interleaved).to(x.dtype)
    if dy is None:
        return y, None, None
    gz = _turn(dy.float(), cos, -sin, interleaved)
    h = gz * w32
    dx = r * (h - xr * (h * xr).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (gz * xr).sum((0, 1, 2)).to(w.dtype)


def _visible(c):
    """[nq, nk]: query i stands at nk - nq + i and sees its window and the sinks, nothing ahead."""
    at = torch.arange(c["nk"] - c["nq"], c["nk"], device="cuda")[:, None]
    key = torch.arange(c["nk"], device="cuda")[None, :]
    return (key <= at) & ((key > at - c["window"]) | (key < c["sinks"]))


def _plain_window(s):
    c = s["case"]
    b, h, hk, nq, d = c["b"], c["h"], c["hk"], c["nq"], c["d"]
    scale = 1 / math.sqrt(d)
    q = s["q"].detach().float().reshape(b, hk, h // hk, nq, d)
    k, v = s["k"].detach().float()[:, :, None], s["v"].detach().float()[:, :, None]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~_visible(c), -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o32 = torch.matmul(p, v)
    out = {"o": o32.reshape(b, h, nq, d).to(s["q"].dtype)}
    if c["grad"]:
        do = s["do"].float().reshape(b, hk, h // hk, nq, d)
        dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o32).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = torch.matmul(ds, k).reshape(b, h, nq, d).to(s["q"].dtype)
        out["dk"] = torch.matmul(ds.transpose(-1, -2), q).sum(2).to(s["q"].dtype)
        out["dv"] = dv.to(s["q"].dtype)
    return out


def _plain_token(c, q, k, v, lengths, dtype):
    b, h, hk, d = c["b"], c["h"], c["hk"], c["d"]
    key = torch.arange(k.shape[2], device="cuda")[None, :]
    n = lengths[:, None].long()
    seen = key < n
    if c["window"]:
        seen = seen & ((key >= n - c["window"]) | (key < c["sinks"]))
    seen = seen[:, None, None, :]
    x = torch.matmul(q.float().reshape(b, hk, h // hk, d), k.float().transpose(-1, -2)) / math.sqrt(d)
    x = x.masked_fill(~seen, -math.inf)
    p = torch.where(seen, (x - x.amax(-1, keepdim=True)).exp(), torch.zeros_like(x))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.float()) / torch.where(total > 0, total, torch.ones_like(total))
    return o.reshape(b, h, 1, d).to(dtype)


def _plain_quantize(x):
    """[..., D] -> codes [..., D / 2] and (scale, minimum) [..., D / 64, 2]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).half().float()
    n = torch.where(scale > 0, (g - low) / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(g))
    n = n.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.cat((scale, low), -1).half()


def _plain_values(codes, params):
    """What the codes stand for, in 16 bits: scale * code + minimum."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    p = params.float()
    return (p[..., :1] * n + p[..., 1:]).flatten(-2).half()


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        at = s["positions"].long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q, dq, dwq = _plain_rope(s["q"], s["wq"], cos, sin, c["interleaved"], s["dq"] if c["grad"] else None)
        k, dk, dwk = _plain_rope(s["k"], s["wk"], cos, sin, c["interleaved"], s["dk"] if c["grad"] else None)
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if c["op"] == "window":
        return _plain_window(s)
    if c["op"] == "token":
        return {"o": _plain_token(c, s["q"], s["k"], s["v"], s["lengths"], s["q"].dtype)}
    if c["op"] == "fill4":
        cache, out = s["cache"], {}
        at = s["start"].long()[:, None] + torch.arange(c["t"], device="cuda")
        seq = torch.arange(c["b"], device="cuda")[:, None]
        kc, kp = _plain_quantize(s["k"])
        vc, vp = _plain_quantize(s["v"])
        cache["k_codes"][seq, :, at], cache["k_params"][seq, :, at] = kc.transpose(1, 2), kp.transpose(1, 2)
        cache["v_codes"][seq, :, at], cache["v_params"][seq, :, at] = vc.transpose(1, 2), vp.transpose(1, 2)
        out["k"] = _plain_values(cache["k_codes"][seq, :, at], cache["k_params"][seq, :, at]).transpose(1, 2)
        out["v"] = _plain_values(cache["v_codes"][seq, :, at], cache["v_params"][seq, :, at]).transpose(1, 2)
        return out
    cache = s["cache"]
    k = _plain_values(cache["k_codes"], cache["k_params"])
    v = _plain_values(cache["v_codes"], cache["v_params"])
    return {"o": _plain_token(c, s["q"], k, v, s["lengths"], torch.float16)}


# ------------------------------------------------------------------------------ the framework's calls
def _tattn():
    at = os.path.join(os.getcwd(), "triton-attn_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tattn

    return tattn


def _own(s):
    c, t = s["case"], _tattn()
    if c["op"] == "rope":
        q, k = t.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"], interleaved=c["interleaved"])
        out = {"q": q, "k": k}
        if c["grad"]:
            names, of = ("dq", "dk", "dwq", "dwk"), (s["q"], s["k"], s["wq"], s["wk"])
            out.update(zip(names, torch.autograd.grad((q, k), of, (s["dq"], s["dk"]))))
        return out
    if c["op"] == "window":
        o = t.window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"])
        out = {"o": o}
        if c["grad"]:
            out.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])))
        return out
    window = c.get("window") or None
    if c["op"] == "token":
        return {"o": t.decode_attention(s["q"], s["k"], s["v"], s["lengths"], window, c["sinks"])}
    cache = t.Int4Cache(**s["cache"])
    if c["op"] == "fill4":
        cache.append(s["k"], s["v"], s["start"])
        k, v = cache.read(c["t"], s["start"])
        return {"k": k, "v": v}
    return {"o": cache.attend(s["q"], s["lengths"], window, c["sinks"])}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ what it takes
def _seen(c, n):
    """Tokens of n that a query at position n - 1 sees."""
    w = c["window"] or n
    return min(n, w) + min(c["sinks"], max(0, n - w))


def work(case):
    c = case
    size = 4 if c.get("dtype") == "f32" else 2
    d = c["d"]
    if c["op"] == "rope":
        rows = c["b"] * (c["h"] + c["hk"]) * c["n"]
        tables = 4 * d * min(8192, c["b"] * c["n"])
        if c["grad"]:  # x and dy in; y and dx out
            return {"bytes": 4 * rows * d * size + tables, "flops": 22 * rows * d}
        return {"bytes": 2 * rows * d * size + tables, "flops": 9 * rows * d}
    if c["op"] == "window":
        pairs = c["b"] * c["h"] * sum(_seen(c, n) for n in range(c["nk"] - c["nq"] + 1, c["nk"] + 1))
        q, kv = c["b"] * c["h"] * c["nq"] * d * size, c["b"] * c["hk"] * c["nk"] * d * size
        if c["grad"]:  # q, do, k, v in; o, dq, dk, dv out
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + 2 * min(kv, c["b"] * c["hk"] * d * size * (c["nq"] + c["window"] + c["sinks"])), "flops": 4 * d * pairs}
    if c["op"] == "fill4":
        rows = 2 * c["b"] * c["hk"] * c["t"]
        return {"bytes": rows * (4 * d + 2 * (d // 2 + 4 * d // GROUP)), "flops": 8 * rows * d}
    rows = sum(_seen(c, n) for n in _lengths(c))
    row = d // 2 + 4 * d // GROUP if c["op"] == "attend4" else d * size
    return {"bytes": 2 * rows * c["hk"] * row + 2 * c["b"] * c["h"] * d * size, "flops": 4 * d * rows * c["h"]}


# ----------------------------------------------------------------------------------------- 64 bits
def _exact_rope(x, w, dy, positions, inv, interleaved):
    x, w, d = x.detach().double(), w.detach().double(), x.shape[-1]
    angle = positions.double()[:, None, :, None] * inv
    # The tables are inputs in 32 bits.
    co, si = angle.cos().float().double(), angle.sin().float().double()
    first = torch.arange(0, d, 2, device="cuda") if interleaved else torch.arange(d // 2, device="cuda")
    second = first + (1 if interleaved else d // 2)
    norm = ((x * x).sum(-1, keepdim=True) / d + 1e-6).sqrt()
    unit = x / norm
    z = unit * w
    y = torch.empty_like(z)
    y[..., first] = z[..., first] * co - z[..., second] * si
    y[..., second] = z[..., first] * si + z[..., second] * co
    if dy is None:
        return y, None, None
    dy = dy.double()
    dz = torch.empty_like(dy)
    dz[..., first] = dy[..., first] * co + dy[..., second] * si
    dz[..., second] = dy[..., second] * co - dy[..., first] * si
    du = dz * w
    dx = du / norm - x * (du * x).sum(-1, keepdim=True) / (d * norm**3)
    return y, dx, torch.einsum("bhnd,bhnd->d", dz, unit)


def _exact_window(s):
    c = s["case"]
    each, scale = c["h"] // c["hk"], c["d"] ** -0.5
    o, dq, dk, dv = (torch.empty(s[x].shape, device="cuda", dtype=torch.float64) for x in ("q", "q", "k", "v"))
    hidden = ~_visible(c)
    dk.zero_()
    dv.zero_()
    for b in range(c["b"]):
        for h in range(c["h"]):
            q, k, v = s["q"][b, h].detach().double(), s["k"][b, h // each].detach().double(), s["v"][b, h // each].detach().double()
            p = torch.softmax((q @ k.T * scale).masked_fill(hidden, -math.inf), -1)
            o[b, h] = p @ v
            if c["grad"]:
                g = s["do"][b, h].double()
                dp = g @ v.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dv[b, h // each] += p.T @ g
                dk[b, h // each] += ds.T @ q * scale
                dq[b, h] = ds @ k * scale
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if c["grad"] else {"o": o}


def _exact_token(c, q, k, v):
    """k(b), v(b): one sequence's keys and values in 64 bits, [heads, cap, d]."""
    o = torch.zeros((c["b"], c["h"], 1, c["d"]), device="cuda", dtype=torch.float64)
    each = c["h"] // c["hk"]
    for b, n in enumerate(_lengths(c)):
        w = c["window"] or n
        seen = sorted(set(range(min(c["sinks"], n))) | set(range(max(0, n - w), n)))
        at = torch.tensor(seen, device="cuda")
        kb, vb = k(b)[:, at].repeat_interleave(each, 0), v(b)[:, at].repeat_interleave(each, 0)
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[b, :, 0].double(), kb) * c["d"] ** -0.5, -1)
        o[b, :, 0] = torch.einsum("hn,hnd->hd", p, vb)
    return {"o": o}


def _exact_values(codes, params):
    """The fp16 values that codes stand for."""
    n = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), device="cuda", dtype=torch.float64)
    n[..., 0::2], n[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    p = params.double().repeat_interleave(GROUP, -2)
    return (n * p[..., 0] + p[..., 1]).half().double()


def _exact_round_trip(x):
    x = x.double()
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], GROUP):
        part = x[..., g : g + GROUP]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        step = ((high - low) / 15).half().double()
        code = torch.round((part - low) / step.clamp(min=1e-300)).clamp(0, 15)
        out[..., g : g + GROUP] = (low + step * code).half().double()
    return out


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "rope":
        inv = 10000.0 ** (-torch.arange(0, c["d"], 2, device="cuda", dtype=torch.float64) / c["d"])
        q, dq, dwq = _exact_rope(s["q"], s["wq"], s["dq"] if c["grad"] else None, s["positions"], inv, c["interleaved"])
        k, dk, dwk = _exact_rope(s["k"], s["wk"], s["dk"] if c["grad"] else None, s["positions"], inv, c["interleaved"])
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if c["op"] == "window":
        return _exact_window(s)
    if c["op"] == "token":
        return _exact_token(c, s["q"], lambda b: s["k"][b].double(), lambda b: s["v"][b].double())
    if c["op"] == "fill4":
        return {"k": _exact_round_trip(s["k"]), "v": _exact_round_trip(s["v"])}
    cache = s["cache"]
    return _exact_token(c, s["q"], *(lambda b, x=x: _exact_values(cache[x + "_codes"][b], cache[x + "_params"][b]) for x in ("k", "v")))
