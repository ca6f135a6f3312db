"""``window_attention(q, k, v, window, sinks=0, sm_scale=None)``: causal attention in which a query sees the
last ``window`` keys up to its own and the first ``sinks`` ones, with autograd.

The reference has no counterpart; conventions (layout, dtypes, default scale, errors, once-differentiable
autograd) are those of ``tattn.attention``. Keys and values may have fewer heads than the queries, each
shared by a group of consecutive query heads, and more tokens: the queries are the sequence's last ones.
"""

from __future__ import annotations

import torch

from tattn import _lib


def _forward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, scale: float
) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns (O, M): O like q, M fp32 [Z, H, Nq] (base-2 log-sum-exp)."""
    return _lib.torch_ext().window_forward(q, k, v, window, sinks, scale)


def _backward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, m: torch.Tensor, do: torch.Tensor,
    window: int, sinks: int, scale: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """Returns contiguous (dq, dk, dv)."""
    return _lib.torch_ext().window_backward(q, k, v, o, m, do, window, sinks, scale)


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, sm_scale: float | None = None
) -> torch.Tensor:
    """Attention over a sliding window and the first tokens, on an sm_100 GPU.

    q is [batch, heads, seq, dim]; k and v are [batch, kv_heads, kv_seq, dim] with kv_heads dividing heads and
    kv_seq >= seq. Query i stands at position p = kv_seq - seq + i and sees the keys j <= p with j > p - window
    or j < sinks. Returns a tensor like q; gradients reach q, k and v, once and in reverse mode (forward-mode
    tensors are refused). As in any masked product, a NaN or an infinity in v reaches queries near its token that
    do not see it, and in the gradients one in any input reaches tokens near its own.
    """
    return _lib.torch_ext().window_attention(q, k, v, window, sinks, sm_scale)
