"""Attention with a window and sinks from its definition in 64 bits, with bounds for the error of kernels that
round P and dS to 16 bits (fp16) or work in 32 bits throughout (fp32)."""

from __future__ import annotations

import math

import torch


def visible(nq: int, nk: int, window: int, sinks: int, device) -> torch.Tensor:
    """[nq, nk]: does query i, at position nk - nq + i, see key j?"""
    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def window_attention64(q, k, v, do, window, sinks, scale):
    """(o, dq, dk, dv) and, of the same shapes, how far a kernel in q's dtype may be from them.

    u is the unit roundoff of the outputs. fp16: P and dS are rounded to 16 bits (u relative each), the
    forward's exponentials are within 7.5e-5, delta is taken from the rounded O; c = 1e-3 covers these
    with the 32-bit sums. fp32: c covers sums of nk + d terms. Every product's error is at most c times
    the product's magnitude, so the bounds are sums of magnitudes.
    """
    half = q.dtype == torch.float16
    nk, d = k.shape[2], k.shape[3]
    u = 2.0**-11 if half else 2.0**-24
    c = 1e-3 if half else (nk + d) * 2.0**-23 + 1e-6
    group = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    kx, vx = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    see = visible(q.shape[2], nk, window, sinks, q.device)
    p = torch.softmax((q @ kx.transpose(-1, -2) * scale).masked_fill(~see, -math.inf), -1)
    o = p @ vx
    dp = do @ vx.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq = ds @ kx * scale

    def shared(t):  # sum over the query heads of a key/value head
        return t.unflatten(1, (-1, group)).sum(2)

    dk, dv = shared(ds.transpose(-1, -2) @ q) * scale, shared(p.transpose(-1, -2) @ do)
    e_o = c * (p @ vx.abs())
    e_ds = c * p * (dp.abs() + delta.abs()) + p * (u * (do.abs() * o.abs()) + do.abs() * e_o).sum(-1, keepdim=True)
    errs = (
        e_o,
        abs(scale) * (e_ds @ kx.abs()),
        abs(scale) * shared(e_ds.transpose(-1, -2) @ q.abs()),
        c * shared(p.transpose(-1, -2) @ do.abs()),
    )
    outs = (o, dq, dk, dv)
    tiny = 2.0**-24 if half else 2.0**-126  # results below fp16's normal range round absolutely
    return outs, tuple(2 * u * x.abs() + e + tiny for x, e in zip(outs, errs, strict=True))


def assert_within(got, want, bound, name: str) -> None:
    """|got - want| <= bound everywhere, and nothing but numbers."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.detach().double() - want).abs()
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    over = off > bound
    assert not bool(over.any()), f"{name}: {int(over.sum())} values off, worst {float((off / bound).max()):.2f} of its bound"
