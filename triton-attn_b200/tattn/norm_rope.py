"""``qk_norm_rope``: the norm of every query and key head with the position rotation, in one pass, with autograd.

The reference has no counterpart; conventions (layout, dtypes, errors, once-differentiable autograd) are
those of ``tattn.attention``, whose inputs this makes.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn.api import _dtype_code, _require_cuda


def _check(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
    sin: torch.Tensor, positions: torch.Tensor | None,
) -> None:  # fmt: skip
    sq, sk = q.shape, k.shape
    if len(sq) != 4 or len(sk) != 4 or sq[0] != sk[0] or sq[2:] != sk[2:]:
        raise ValueError(f"expected q [batch, heads, seq, dim] and k [batch, kv_heads, seq, dim]; got {sq}, {sk}")
    b, h, n, d = sq
    if h == 0 or sk[1] == 0:
        raise ValueError(f"q and k need at least one head; got {sq}, {sk}")
    if d not in (16, 32, 64, 128):
        raise ValueError(f"head dim must be 16, 32, 64 or 128, got {d}")
    dtype, w_dtype = q.dtype, q_weight.dtype
    if k.dtype != dtype or dtype not in (torch.float16, torch.float32):
        raise ValueError(f"q, k must share dtype float16 or float32, got {dtype}, {k.dtype}")
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError(f"weights must have shape ({d},); got {q_weight.shape}, {k_weight.shape}")
    if k_weight.dtype != w_dtype or w_dtype not in (dtype, torch.float32):
        raise ValueError(f"weights must share q's dtype or float32; got {w_dtype}, {k_weight.dtype}")
    table = cos.shape
    if len(table) != 2 or table[1] != d // 2 or sin.shape != table:
        raise ValueError(f"cos and sin must have shape [positions, {d // 2}]; got {table}, {sin.shape}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"cos and sin must be float32; got {cos.dtype}, {sin.dtype}")
    if positions is None:
        if table[0] < n:
            raise ValueError(f"the tables hold {table[0]} positions, fewer than the {n} tokens")
    else:
        if positions.dtype != torch.int32 or positions.shape not in ((n,), (b, n)):
            raise ValueError(f"positions must be int32 [{n}] or [{b}, {n}]; got {positions.dtype} {positions.shape}")
        if table[0] == 0 and b * n > 0:
            raise ValueError("the tables hold no positions")
    at = q.get_device()  # -1: not on a GPU
    for t in (k, q_weight, k_weight, cos, sin):
        if t.get_device() != at:
            raise ValueError(f"all tensors must be on one device, got {q.device} and {t.device}")
    if positions is not None and positions.get_device() != at:
        raise ValueError(f"all tensors must be on one device, got {q.device} and {positions.device}")


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` in place if its rows can be read 16 bytes at a time, else a dense copy."""
    if t.data_ptr() % 16 == 0:
        *outer, last = t.stride()
        unit = 16 // t.element_size()
        if last == 1:
            for n, s in zip(t.shape, outer):
                if s % unit and n > 1:
                    break
            else:
                return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _dense16(t: torch.Tensor) -> torch.Tensor:
    """``t`` if it is dense and 16-byte aligned, else a copy that is."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A tensor for results, dense in the order of t's dimensions."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _position_strides(positions: torch.Tensor | None) -> tuple[int, ...]:
    if positions is None:
        return 0, 0
    return (0, *positions.stride()) if positions.dim() == 1 else positions.stride()


def _forward(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
    sin: torch.Tensor, positions: torch.Tensor | None, eps: float, interleaved: bool,
) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """Of tensors that _rows16 or _dense16 left in place."""
    q_out, k_out = _like(q), _like(k)
    z, h, n, d = q.shape
    strides = q.stride() + k.stride() + q_out.stride() + k_out.stride() + _position_strides(positions)
    at = q.get_device()
    with _lib.on_device(at):
        rc = _lib.load().tattn_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
            cos.data_ptr(), sin.data_ptr(), None if positions is None else positions.data_ptr(),
            _lib.strides_bytes(strides), z, h, k.shape[1], n, d, cos.shape[0], _dtype_code(q), _dtype_code(q_weight),
            eps, interleaved, _lib.raw_stream(at),
        )  # fmt: skip
    if rc:
        _lib.check("tattn_qk_norm_rope", rc)
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
        cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None, eps: float, interleaved: bool,
    ) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = eps, interleaved
        return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, q_grad: torch.Tensor, k_grad: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        lib = _lib.load()
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        eps, interleaved = ctx.args
        q_grad, k_grad = _rows16(q_grad), _rows16(k_grad)
        dq, dk, dwq, dwk = _like(q), _like(k), torch.empty_like(q_weight), torch.empty_like(k_weight)
        z, h, n, d = q.shape
        strides = (
            q.stride() + k.stride() + q_grad.stride() + k_grad.stride() + dq.stride() + dk.stride()
            + _position_strides(positions)
        )  # fmt: skip
        at = q.get_device()
        with _lib.on_device(at):
            ws = torch.empty(lib.tattn_qk_norm_rope_bwd_workspace_bytes(d), device=q.device, dtype=torch.uint8)
            rc = lib.tattn_qk_norm_rope_bwd(
                q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), q_grad.data_ptr(),
                k_grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(), cos.data_ptr(),
                sin.data_ptr(), None if positions is None else positions.data_ptr(), ws.data_ptr(),
                _lib.strides_bytes(strides), z, h, k.shape[1], n, d, cos.shape[0], _dtype_code(q),
                _dtype_code(q_weight), eps, interleaved, _lib.raw_stream(at),
            )  # fmt: skip
        if rc:
            _lib.check("tattn_qk_norm_rope_bwd", rc)
        return dq, dk, dwq, dwk, None, None, None, None, None


def qk_norm_rope(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
    sin: torch.Tensor, positions: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """Normed and rotated queries and keys, on an sm_100 GPU.

    q is [batch, heads, seq, dim] and k [batch, kv_heads, seq, dim], fp16 or fp32, in any layout with contiguous
    rows (a transposed [batch, seq, heads, dim] projection is read in place, and the results are laid out
    alike). Each row x becomes R(p) (x / sqrt(mean(x^2) + eps) * weight), where R(p) rotates pair j by the
    angle with cosine cos[p, j] and sine sin[p, j]; cos and sin are float32 [positions, dim / 2]. The pairs
    are (j, j + dim / 2) or, interleaved, (2 j, 2 j + 1). Token n of a sequence stands at p = n, or where
    ``positions`` (int32 [seq] or [batch, seq]) says; a position outside the tables gives NaN rows and
    sets DEV_INDEX_RANGE in the device status word. Weights are [dim], of q's dtype or float32; gradients
    reach q, k and the weights.
    """
    _check(q, k, q_weight, k_weight, cos, sin, positions)
    _require_cuda(q)
    args = (
        _rows16(q), _rows16(k), _dense16(q_weight), _dense16(k_weight), _dense16(cos), _dense16(sin), positions,
        float(eps), bool(interleaved),
    )  # fmt: skip
    if torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad
    ):
        out: tuple[torch.Tensor, torch.Tensor] = _QkNormRope.apply(*args)
        return out
    return _forward(*args)
