"""Cases for the operators of a decoder that reads an encoder's states, stands at positions of several axes, and answers
one prompt many times, around ``tattn.attention``:

* ``cross_attention``: attention to an encoder's states of another length, padded to the longest of the batch, and its
  gradients;
* ``qk_rope_axes``: the rotation of query and key heads by positions on several axes (time, height, width), with the
  heads' norms or without, and its gradients;
* ``prefix_decode_attention``: one new token of each sequence where the samples of a prompt share the prompt's keys
  and values, each with tokens of its own behind it.

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
TABLE = 8192  # positions in the rotation's tables


# ------------------------------------------------------------------------------------------ cases
def _cross(name, b, h, hk, nq, nk, d, spread, dtype, grad, layout):
    """spread: sequence i holds nk - (i * 7919) % (spread + 1) states, none where that is below 0."""
    return dict(name=name, op="cross", b=b, h=h, hk=hk, nq=nq, nk=nk, d=d, spread=spread, dtype=dtype, grad=grad, layout=layout)


def _axes(name, b, h, hk, n, d, axes, mixed, norm, dtype, grad, interleaved, layout):
    """mixed: pairs take the axes in turn; else each axis has a run of pairs."""
    return dict(name=name, op="axes", b=b, h=h, hk=hk, n=n, d=d, axes=axes, mixed=mixed, norm=norm, dtype=dtype, grad=grad,
                interleaved=interleaved, layout=layout)  # fmt: skip


def _prefix(name, prompts, samples, h, hk, prefix, prefix_spread, cap, spread, d, dtype):
    return dict(name=name, op="prefix", prompts=prompts, samples=samples, h=h, hk=hk, prefix=prefix, prefix_spread=prefix_spread,
                cap=cap, spread=spread, d=d, dtype=dtype)  # fmt: skip


def listed():
    return [
        # One decoding step of 8 sequences over an encoder's 1,500 states: latency.
        _cross("cross_token", 8, 16, 16, 1, 1500, 64, 700, "f16", False, "bhnd"),
        # A few queries gather a long input: 64 rows a head, so the work has to be split along the states.
        _cross("cross_gather", 1, 16, 16, 64, 16384, 64, 0, "f16", False, "bhnd"),
        # A prompt of 2,000 tokens reads padded states, key/value heads shared by four query heads.
        _cross("cross_prompt", 2, 16, 4, 2000, 6404, 128, 900, "f16", False, "bnhd"),
        # Training an encoder-decoder: 448 tokens against up to 1,500 states, as the projections leave them.
        _cross("cross_train", 8, 16, 16, 448, 1500, 64, 1000, "f16", True, "bnhd"),
        # Training with shared heads and long inputs of unequal lengths.
        _cross("cross_train_gqa", 4, 16, 4, 2048, 4100, 128, 3600, "f16", True, "bhnd"),
        # 32-bit training, small and odd; one sequence has no states at all.
        _cross("cross_train_f32", 3, 5, 5, 200, 777, 64, 1500, "f32", True, "bhnd"),
        # One decoding step of a small batch: the new token's heads, where latency counts.
        _axes("axes_token", 8, 16, 4, 1, 128, 3, False, True, "f16", False, False, "bnhd"),
        # A training step's queries and keys as the projections leave them, axes in turn over the pairs.
        _axes("axes_train", 4, 16, 4, 4096, 128, 3, True, True, "f16", True, False, "bnhd"),
        # 32-bit training of the rotation alone at an odd length, neighbouring dims rotated together.
        _axes("axes_train_f32", 3, 5, 5, 1000, 32, 3, False, False, "f32", True, True, "bhnd"),
        # 16 samples of one short prompt, a few tokens in: latency.
        _prefix("prefix_token", 1, 16, 16, 4, 1000, 0, 256, 200, 64, "f16"),
        # 64 samples of one long prompt, each with up to 2,048 tokens of its own.
        _prefix("prefix_long", 1, 64, 16, 4, 32768, 0, 2048, 2000, 128, "f16"),
        # In 32 bits: 8 samples of each of 4 prompts of unequal length.
        _prefix("prefix_f32", 4, 8, 8, 4, 4000, 3000, 300, 299, 64, "f32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even in the logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def _heads(rng):
    hk = rng.choice((1, 2, 3, 4, 5, 8, 16))
    return hk * rng.choice((1, 1, 2, 3, 4, 8)), hk


def draw(rng):
    op = rng.choice(("cross", "cross", "cross", "axes", "axes", "prefix", "prefix"))
    h, hk = _heads(rng)
    d = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("f16", "f16", "f16", "f32"))
    layout = rng.choice(("bnhd", "bhnd"))
    size = 4 if dtype == "f32" else 2
    room = 320_000_000 // (d * size)  # rows of a head, as many as the largest listed cases read and write
    if op == "cross":
        b = rng.choice((1, 2, 3, 4, 8))
        grad = rng.random() < 0.6
        most = (400_000_000 if grad else 800_000_000) * 64 // max(d, 64) if dtype == "f16" else 30_000_000
        nk = _log(rng, 1, 16384)
        nq = rng.choice((_log(rng, 1, 16), _log(rng, 1, 4096)))
        nk = max(1, min(nk, most // (b * h), room // (4 * b * hk)))
        nq = max(1, min(nq, most // (b * h * nk), room // (4 * b * h)))
        c = _cross("", b, h, hk, nq, nk, d, rng.choice((0, rng.randint(0, nk + nk // 4))), dtype, grad, layout)
    elif op == "axes":
        b = rng.choice((1, 2, 3, 4, 8))
        n = rng.choice((1, _log(rng, 1, 4096)))
        n = max(1, min(n, room // (4 * b * (h + hk))))
        c = _axes("", b, h, hk, n, d, rng.choice((1, 2, 3, 3, 4)), rng.random() < 0.5, rng.random() < 0.6, dtype,
                  rng.random() < 0.7, rng.random() < 0.3, layout)  # fmt: skip
    else:
        prompts, samples = rng.choice((1, 1, 2, 4)), rng.choice((1, 2, 5, 8, 16, 33, 64))
        prefix, cap = _log(rng, 1, 32768), _log(rng, 1, 4096)
        most = 64 * 16 * 32768 * 128 if dtype == "f16" else 8 * 8 * 32768 * 64
        prefix = max(1, min(prefix, most // (prompts * samples * h * d), room // (4 * prompts * hk)))
        cap = max(1, min(cap, room // (2 * prompts * samples * hk)))
        c = _prefix("", prompts, samples, h, hk, prefix, rng.choice((0, rng.randint(0, prefix))), cap, rng.randint(0, cap + cap // 4), d, dtype)
    del c["name"]
    return c


def _held(count, cap, spread):
    return [max(0, cap - (i * 7919) % (spread + 1)) for i in range(count)]


def _pair_axes(c):
    """The axis of each of the d / 2 pairs."""
    pairs, a = c["d"] // 2, c["axes"]
    return [j % a if c["mixed"] else j * a // pairs for j in range(pairs)]


# ------------------------------------------------------------------------------------------ inputs
def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _rows(g, layout, b, h, n, d, dtype):
    """[b, h, n, d]: dense, or a view of a projection [b, n, h, d]."""
    if layout == "bnhd":
        return _randn(g, (b, n, h, d), dtype).transpose(1, 2)
    return _randn(g, (b, h, n, d), dtype)


def _positions(g, c):
    """[axes, b, n]: runs of text, which stand at one place on all axes, and grids of an image between them, whose
    tokens share a time and stand at their row and column."""
    b, n, a = c["b"], c["n"], c["axes"]
    start = torch.randint(0, 2000, (b, 1), generator=g, device="cuda")
    i = torch.arange(n, device="cuda")[None, :]
    wide = 24  # a grid's columns; 600 tokens of a grid follow 100 of text
    inside = torch.where(i % 700 >= 100, i % 700 - 100, torch.zeros_like(i))
    base = start + i // 700 * 125 + torch.minimum(i % 700, torch.full_like(i, 100))
    axes = [base, base + inside // wide, base + inside % wide, base + inside % 7]
    return torch.stack(axes[:a]).to(torch.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    dt, d = DTYPES[c["dtype"]], c["d"]
    if c["op"] == "cross":
        s["q"] = _rows(g, c["layout"], c["b"], c["h"], c["nq"], d, dt)
        s["k"] = _rows(g, c["layout"], c["b"], c["hk"], c["nk"], d, dt)
        s["v"] = _rows(g, c["layout"], c["b"], c["hk"], c["nk"], d, dt)
        s["lengths"] = torch.tensor(_held(c["b"], c["nk"], c["spread"]), device="cuda", dtype=torch.int32)
        if c["grad"]:
            s["do"] = _rows(g, c["layout"], c["b"], c["h"], c["nq"], d, dt)
            for key in ("q", "k", "v"):
                s[key].requires_grad_()
    elif c["op"] == "axes":
        s["q"], s["k"] = (_rows(g, c["layout"], c["b"], h, c["n"], d, dt) for h in (c["h"], c["hk"]))
        s["positions"] = _positions(g, c)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angle = torch.arange(TABLE, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["axes"] = _pair_axes(c)
        if c["norm"]:
            s["wq"], s["wk"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
        if c["grad"]:
            s["dq"], s["dk"] = (_rows(g, c["layout"], c["b"], h, c["n"], d, dt) for h in (c["h"], c["hk"]))
            for key in ("q", "k", "wq", "wk"):
                if key in s:
                    s[key].requires_grad_()
    else:
        p, b = c["prompts"], c["prompts"] * c["samples"]
        s["q"] = _randn(g, (b, c["h"], 1, d), dt)
        s["pk"], s["pv"] = (_randn(g, (p, c["hk"], c["prefix"], d), dt) for _ in range(2))
        s["k"], s["v"] = (_randn(g, (b, c["hk"], c["cap"], d), dt) for _ in range(2))
        s["prefix_lengths"] = torch.tensor(_held(p, c["prefix"], c["prefix_spread"]), device="cuda", dtype=torch.int32)
        s["lengths"] = torch.tensor(_held(b, c["cap"], c["spread"]), device="cuda", dtype=torch.int32)
    return s


# -------------------------------------------------------------------------------------- plain forms
def _softmax(x, seen):
    """Weights over the last dimension of the seen places, and zeros where there are none."""
    x = x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _plain_cross(s):
    c = s["case"]
    b, h, hk, nq, nk, d = c["b"], c["h"], c["hk"], c["nq"], c["nk"], c["d"]
    scale, dt = 1 / math.sqrt(d), s["q"].dtype
    q = s["q"].detach().float().reshape(b, hk, h // hk, nq, d)
    k, v = s["k"].detach().float()[:, :, None], s["v"].detach().float()[:, :, None]
    seen = (torch.arange(nk, device="cuda") < s["lengths"][:, None])[:, None, None, None, :]
    p = _softmax(torch.matmul(q, k.transpose(-1, -2)).mul_(scale), seen)
    o32 = torch.matmul(p, v)
    out = {"o": o32.reshape(b, h, nq, d).to(dt)}
    if c["grad"]:
        do = s["do"].float().reshape(b, hk, h // hk, nq, d)
        dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o32).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = torch.matmul(ds, k).reshape(b, h, nq, d).to(dt)
        out["dk"] = torch.matmul(ds.transpose(-1, -2), q).sum(2).to(dt)
        out["dv"] = dv.to(dt)
    return out


def _turn(z, cos, sin, interleaved):
    if interleaved:
        a, b = z[..., 0::2], z[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = z.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_heads(x, w, cos, sin, interleaved, dy, eps=1e-6):
    """(y, dx, dw) of one tensor; w None: the rotation alone."""
    z = x.detach().float()
    if w is not None:
        w32 = w.detach().float()
        r = torch.rsqrt(z.square().mean(-1, keepdim=True) + eps)
        xr = z * r
        z = xr * w32
    y = _turn(z, cos, sin, interleaved).to(x.dtype)
    if dy is None:
        return y, None, None
    gz = _turn(dy.float(), cos, -sin, interleaved)
    if w is None:
        return y, gz.to(x.dtype), None
    h = gz * w32
    dx = r * (h - xr * (h * xr).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (gz * xr).sum((0, 1, 2)).to(w.dtype)


def _plain_axes(s):
    c = s["case"]
    pairs = torch.arange(c["d"] // 2, device="cuda")
    at = s["positions"].long()[s["axes"]].permute(1, 2, 0)  # [b, n, pairs]
    cos, sin = s["cos"][at, pairs][:, None], s["sin"][at, pairs][:, None]
    q, dq, dwq = _plain_heads(s["q"], s.get("wq"), cos, sin, c["interleaved"], s.get("dq"))
    k, dk, dwk = _plain_heads(s["k"], s.get("wk"), cos, sin, c["interleaved"], s.get("dk"))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _plain_prefix(s):
    c = s["case"]
    p, n, h, hk, d = c["prompts"], c["samples"], c["h"], c["hk"], c["d"]
    q = s["q"].float().reshape(p, n, hk, h // hk, d) / math.sqrt(d)
    rows = q.transpose(1, 2).reshape(p, hk, n * (h // hk), d)  # the prompt's queries of a head, over its prefix
    shared = torch.matmul(rows, s["pk"].float().transpose(-1, -2)).reshape(p, hk, n, h // hk, c["prefix"]).transpose(1, 2)
    each = torch.matmul(q, s["k"].float().reshape(p, n, hk, c["cap"], d).transpose(-1, -2))
    seen_p = (torch.arange(c["prefix"], device="cuda") < s["prefix_lengths"][:, None]).reshape(p, 1, 1, 1, c["prefix"])
    seen = (torch.arange(c["cap"], device="cuda") < s["lengths"][:, None]).reshape(p, n, 1, 1, c["cap"])
    weights = _softmax(torch.cat((shared, each), -1), torch.cat((seen_p.expand(p, n, 1, 1, -1), seen), -1))
    of_p, of_own = weights.split((c["prefix"], c["cap"]), -1)
    o = torch.matmul(of_own, s["v"].float().reshape(p, n, hk, c["cap"], d))
    of_p = of_p.transpose(1, 2).reshape(p, hk, n * (h // hk), c["prefix"])
    o = o + torch.matmul(of_p, s["pv"].float()).reshape(p, hk, n, h // hk, d).transpose(1, 2)
    return {"o": o.reshape(p * n, h, 1, d).to(s["q"].dtype)}


# ------------------------------------------------------------------------------ the framework's calls
def _tattn():
    at = os.path.join(os.getcwd(), "triton-attn_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tattn

    return tattn


def _own(s):
    c, t = s["case"], _tattn()
    if c["op"] == "cross":
        o = t.cross_attention(s["q"], s["k"], s["v"], s["lengths"])
        out = {"o": o}
        if c["grad"]:
            out.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])))
        return out
    if c["op"] == "axes":
        q, k = t.qk_rope_axes(s["q"], s["k"], s["cos"], s["sin"], s["positions"], s["axes"], s.get("wq"), s.get("wk"),
                              interleaved=c["interleaved"])  # fmt: skip
        out = {"q": q, "k": k, "dq": None, "dk": None, "dwq": None, "dwk": None}
        if c["grad"]:
            names = ("dq", "dk", "dwq", "dwk") if c["norm"] else ("dq", "dk")
            of = (s["q"], s["k"], s["wq"], s["wk"]) if c["norm"] else (s["q"], s["k"])
            out.update(zip(names, torch.autograd.grad((q, k), of, (s["dq"], s["dk"]))))
        return out
    return {"o": t.prefix_decode_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lengths"], s["prefix_lengths"])}


def run(state):
    if own:
        return _own(state)
    return {"cross": _plain_cross, "axes": _plain_axes, "prefix": _plain_prefix}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ what it takes
def work(case):
    c = case
    size, d = 4 if c["dtype"] == "f32" else 2, c["d"]
    if c["op"] == "cross":
        held = sum(_held(c["b"], c["nk"], c["spread"]))
        q, kv = c["b"] * c["h"] * c["nq"] * d * size, held * c["hk"] * d * size
        pairs = c["h"] * c["nq"] * held
        if c["grad"]:  # q, do, k, v in; o, dq, dk, dv out, the last two over the whole length
            return {"bytes": 4 * q + 2 * kv + 2 * c["b"] * c["nk"] * c["hk"] * d * size, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * d * pairs}
    if c["op"] == "axes":
        rows = c["b"] * (c["h"] + c["hk"]) * c["n"]
        tables = 4 * d * min(TABLE, c["b"] * c["n"]) + 4 * c["axes"] * c["b"] * c["n"]
        if not c["grad"]:
            return {"bytes": 2 * rows * d * size + tables, "flops": (9 if c["norm"] else 3) * rows * d}
        # x and dy in, y and dx out
        return {"bytes": 4 * rows * d * size + tables, "flops": (22 if c["norm"] else 6) * rows * d}
    shared = sum(_held(c["prompts"], c["prefix"], c["prefix_spread"]))
    each = sum(_held(c["prompts"] * c["samples"], c["cap"], c["spread"]))
    q = c["prompts"] * c["samples"] * c["h"] * d * size
    return {"bytes": 2 * q + 2 * (shared + each) * c["hk"] * d * size, "flops": 4 * d * c["h"] * (shared * c["samples"] + each)}


# ----------------------------------------------------------------------------------------- 64 bits
def _exact_cross(s):
    c = s["case"]
    each, scale = c["h"] // c["hk"], c["d"] ** -0.5
    o, dq, dk, dv = (torch.zeros(s[x].shape, device="cuda", dtype=torch.float64) for x in ("q", "q", "k", "v"))
    for b, n in enumerate(_held(c["b"], c["nk"], c["spread"])):
        if n == 0:
            continue
        for h in range(c["h"]):
            g = h // each
            q, k, v = s["q"][b, h].detach().double(), s["k"][b, g, :n].detach().double(), s["v"][b, g, :n].detach().double()
            p = torch.softmax(q @ k.T * scale, -1)
            o[b, h] = p @ v
            if c["grad"]:
                do = s["do"][b, h].double()
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dv[b, g, :n] += p.T @ do
                dk[b, g, :n] += ds.T @ q * scale
                dq[b, h] = ds @ k * scale
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if c["grad"] else {"o": o}


def _exact_heads(x, w, dy, co, si, interleaved):
    x, d = x.detach().double(), x.shape[-1]
    first = torch.arange(0, d, 2, device="cuda") if interleaved else torch.arange(d // 2, device="cuda")
    second = first + (1 if interleaved else d // 2)
    unit = x
    if w is not None:
        norm = ((x * x).sum(-1, keepdim=True) / d + 1e-6).sqrt()
        unit = x / norm
    z = unit if w is None else unit * w.detach().double()
    turned = torch.complex(z[..., first], z[..., second]) * torch.complex(co, si)
    y = torch.empty_like(z)
    y[..., first], y[..., second] = turned.real, turned.imag
    if dy is None:
        return y, None, None
    back = torch.complex(dy.double()[..., first], dy.double()[..., second]) * torch.complex(co, -si)
    dz = torch.empty_like(z)
    dz[..., first], dz[..., second] = back.real, back.imag
    if w is None:
        return y, dz, None
    du = dz * w.detach().double()
    dx = du / norm - x * (du * x).sum(-1, keepdim=True) / (d * norm**3)
    return y, dx, torch.einsum("bhnd,bhnd->d", dz, unit)


def _exact_axes(s):
    c = s["case"]
    shape = (c["b"], 1, c["n"], c["d"] // 2)
    co, si = (torch.empty(shape, device="cuda", dtype=torch.float64) for _ in range(2))
    for j, axis in enumerate(s["axes"]):  # the tables are inputs in 32 bits
        at = s["positions"][axis].long()
        co[:, 0, :, j], si[:, 0, :, j] = s["cos"][:, j].double()[at], s["sin"][:, j].double()[at]
    q, dq, dwq = _exact_heads(s["q"], s.get("wq"), s.get("dq"), co, si, c["interleaved"])
    k, dk, dwk = _exact_heads(s["k"], s.get("wk"), s.get("dk"), co, si, c["interleaved"])
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _exact_prefix(s):
    c = s["case"]
    each = c["h"] // c["hk"]
    o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    prefix, own_lengths = _held(c["prompts"], c["prefix"], c["prefix_spread"]), _held(c["prompts"] * c["samples"], c["cap"], c["spread"])
    for b, n in enumerate(own_lengths):
        p = b // c["samples"]
        k = torch.cat((s["pk"][p, :, : prefix[p]], s["k"][b, :, :n]), 1).double()
        v = torch.cat((s["pv"][p, :, : prefix[p]], s["v"][b, :, :n]), 1).double()
        if k.shape[1] == 0:
            continue
        q = s["q"][b, :, 0].double().reshape(c["hk"], each, -1)
        w = torch.softmax(torch.einsum("ged,gnd->gen", q, k) * c["d"] ** -0.5, -1)
        o[b, :, 0] = torch.einsum("gen,gnd->ged", w, v).reshape(c["h"], -1)
    return {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    return {"cross": _exact_cross, "axes": _exact_axes, "prefix": _exact_prefix}[case["op"]](s)
