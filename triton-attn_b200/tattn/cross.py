"""``cross_attention(q, k, v, lengths=None, sm_scale=None)``: attention to keys and values of another length than the
queries', such as an encoder's states, with autograd.

The reference has no counterpart; conventions (layout, dtypes, default scale, errors, once-differentiable autograd,
shared key/value heads) are those of ``tattn.window_attention``.
"""

from __future__ import annotations

import torch

from tattn import _lib


def cross_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None = None, sm_scale: float | None = None
) -> torch.Tensor:
    """Attention of every query to all keys of its sequence, on an sm_100 GPU.

    q is [batch, heads, seq, dim]; k and v are [batch, kv_heads, kv_seq, dim] with kv_heads dividing heads, of any length.
    With ``lengths`` (int32 [batch], on the device) the queries of sequence b see the first lengths[b] keys only; where
    there are none the result is zeros. A length outside [0, kv_seq] counts as the nearer end and sets DEV_INDEX_RANGE in
    the device status word. Rows of k and v past a length are never used, whatever they hold, and their gradients are
    zeros. An infinity in a row of v that is seen is one in the result, where its weight is above 0 (fp16: above 2^-25 of
    the largest). Returns a tensor like q; gradients reach q, k and v, once and in reverse mode (forward-mode tensors are
    refused), and all three are computed where any is needed. Tensors that the kernels cannot address in place are copied
    in each call: rows not contiguous or not 16-byte aligned and, in fp16, expanded ones (but k and v of single tokens).
    """
    return _lib.torch_ext().cross_attention(q, k, v, lengths, sm_scale)
