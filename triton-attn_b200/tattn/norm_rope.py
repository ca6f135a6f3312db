"""``qk_norm_rope``: the norm of every query and key head with the position rotation, in one pass, with autograd.

The reference has no counterpart; conventions (layout, dtypes, errors, once-differentiable autograd) are
those of ``tattn.attention``, whose inputs this makes.
"""

from __future__ import annotations

import torch

from tattn import _lib


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
    reach q, k and the weights, once and in reverse mode (forward-mode tensors, and tables that need gradients, are
    refused).
    """
    return _lib.torch_ext().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
