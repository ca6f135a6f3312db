"""``window_attention(q, k, v, window, sinks=0, sm_scale=None)``: causal attention in which a query sees the
last ``window`` keys up to its own and the first ``sinks`` ones, with autograd.

The reference has no counterpart; conventions (layout, dtypes, default scale, errors, once-differentiable
autograd) are those of ``tattn.attention``. Keys and values may have fewer heads than the queries, each
shared by a group of consecutive query heads, and more tokens: the queries are the sequence's last ones.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn.api import _dtype_code, _require_cuda, _tma_ready
from tattn.norm_rope import _dense16, _like, _rows16

INT_MAX = 2**31 - 1


def _check_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """Shapes, devices and dtypes of a call whose keys and values may have fewer heads than its queries."""
    sq, sk = q.shape, k.shape
    if len(sq) != 4 or len(sk) != 4 or v.shape != sk:
        raise ValueError(
            "expected q [batch, heads, seq, dim] and k, v of equal shape [batch, kv_heads, kv_seq, dim]; "
            f"got {sq}, {sk}, {v.shape}"
        )
    if sk[0] != sq[0] or sk[3] != sq[3]:
        raise ValueError(f"q and k must agree in batch and head dim; got {sq}, {sk}")
    if sk[1] == 0 or sq[1] % sk[1] != 0:
        raise ValueError(f"query heads must be a multiple of key/value heads; got {sq[1]} and {sk[1]}")
    if not (q.get_device() == k.get_device() == v.get_device()):
        raise ValueError(f"q, k, v must be on one device, got {q.device}, {k.device}, {v.device}")
    if sq[3] not in (16, 32, 64, 128):
        raise ValueError(f"head dim must be 16, 32, 64 or 128, got {sq[3]}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in (torch.float16, torch.float32):
        raise ValueError(f"q, k, v must share dtype float16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")


def _check_window(window: int | None, sinks: int) -> None:
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")


def _forward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, scale: float
) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns (O, M): O like q, M fp32 [Z, H, Nq] (base-2 log-sum-exp)."""
    _require_cuda(q)
    if q.dtype == torch.float16:
        q, k, v = (_tma_ready(t) for t in (q, k, v))
    (z, h, n, d), (_, hk, nk, _) = q.shape, k.shape
    o = _like(q)
    if _rows16(o) is not o:
        o = torch.empty((z, h, n, d), device=q.device, dtype=q.dtype)
    m = torch.empty((z, h, n), device=q.device, dtype=torch.float32)
    at = q.get_device()
    with _lib.on_device(at):
        rc = _lib.load().tattn_window_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), m.data_ptr(),
            _lib.strides_bytes(q.stride() + k.stride() + v.stride() + o.stride()),
            z, h, hk, n, nk, d, _dtype_code(q), window, sinks, scale, _lib.raw_stream(at),
        )  # fmt: skip
    if rc:
        _lib.check("tattn_window_fwd", rc)
    return o, m


def _backward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, m: torch.Tensor, do: torch.Tensor,
    window: int, sinks: int, scale: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """Returns contiguous (dq, dk, dv)."""
    _require_cuda(q)
    lib = _lib.load()
    (z, h, n, d), (_, hk, nk, _), code = q.shape, k.shape, _dtype_code(q)
    do = do.to(q.dtype)
    if q.dtype == torch.float16:
        q, k, v, do, o = (_tma_ready(t) for t in (q, k, v, do, o))
    else:
        do, o = _dense16(do), _dense16(o)
    delta = torch.empty((z, h, n), device=q.device, dtype=torch.float32)
    dq = torch.empty((z, h, n, d), device=q.device, dtype=q.dtype)
    dk, dv = q.new_empty((z, hk, nk, d)), q.new_empty((z, hk, nk, d))
    size = lib.tattn_window_bwd_workspace_bytes(z, h, hk, n, nk, d, code, window, sinks)
    ws = torch.empty(max(size, 0), device=q.device, dtype=torch.uint8)
    at = q.get_device()
    with _lib.on_device(at):
        rc = lib.tattn_window_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), m.data_ptr(), delta.data_ptr(), ws.data_ptr(),
            _lib.strides_bytes(q.stride() + k.stride() + v.stride() + o.stride() + do.stride()),
            z, h, hk, n, nk, d, code, window, sinks, scale, _lib.raw_stream(at),
        )  # fmt: skip
    if rc:
        _lib.check("tattn_window_bwd", rc)
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, scale: float
    ) -> torch.Tensor:
        o, m = _forward(q, k, v, window, sinks, scale)
        ctx.save_for_backward(q, k, v, o, m)
        ctx.args = window, sinks, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, do: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        return *_backward(*ctx.saved_tensors, do, *ctx.args), None, None, None


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, sm_scale: float | None = None
) -> torch.Tensor:
    """Attention over a sliding window and the first tokens, on an sm_100 GPU.

    q is [batch, heads, seq, dim]; k and v are [batch, kv_heads, kv_seq, dim] with kv_heads dividing heads and
    kv_seq >= seq. Query i stands at position p = kv_seq - seq + i and sees the keys j <= p with j > p - window
    or j < sinks. Returns a tensor like q; gradients reach q, k and v.
    """
    _check_heads(q, k, v)
    _check_window(window, sinks)
    if k.shape[2] < q.shape[2]:
        raise ValueError(f"the queries are the last of the keys' sequence; got {q.shape[2]} queries, {k.shape[2]} keys")
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(q.shape[3])
    w, s = min(int(window), INT_MAX), min(int(sinks), INT_MAX)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out: torch.Tensor = _WindowAttention.apply(q, k, v, w, s, scale)
        return out
    return _forward(q, k, v, w, s, scale)[0]
