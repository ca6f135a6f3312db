"""Attention of one new token of each sequence over a cache: ``decode_attention`` over keys and values in the
queries' dtype, ``Int4Cache`` holding them in 4 bits.

The single-token form of ``tattn.window_attention``, for generation: no gradients (tensors that need them are refused
where gradients are recorded), nothing read from the device (the lengths stay there), so a step can be captured in a
CUDA graph.
"""

from __future__ import annotations

import torch

from tattn import _lib

GROUP = 64  # head dims that share a scale and a minimum in the 4-bit cache


def decode_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, window: int | None = None,
    sinks: int = 0, sm_scale: float | None = None,
) -> torch.Tensor:  # fmt: skip
    """Attention of one new token of each sequence over a cache, on an sm_100 GPU.

    q is [batch, heads, 1, dim]; k and v are [batch, kv_heads, capacity, dim] with kv_heads dividing heads. Of
    sequence b the first lengths[b] tokens are held (int32, on the device), the query's own as the last. The
    query sees the last ``window`` of them (None: all) and the first ``sinks``; where none are held the result
    is zeros. A length outside [0, capacity] counts as the nearer end and sets DEV_INDEX_RANGE in the device
    status word. Rows past a length are never used, whatever they hold. The caches are read in place:
    their rows must be contiguous and 16-byte aligned.
    """
    return _lib.torch_ext().decode_attention(q, k, v, lengths, window, sinks, sm_scale)


class Int4Cache:
    """Keys and values of a batch of sequences, held in 4 bits.

    A group of 64 head dims of a token's head is held as a scale s and a minimum m (fp16) and codes n in 0..15,
    which stand for fp16(s n + m); appending rounds to the nearest code. Of normal heads that is within a
    thirtieth of the group's range; a group with a NaN or an infinity in it reads as NaN throughout. For keys and
    values each there are the tensors ``*_codes`` uint8 [batch, kv_heads, capacity, dim / 2] (head dim 2 i in the
    low half of byte i) and ``*_params`` float16 [batch, kv_heads, capacity, dim / 64, 2] (s, m);
    ``Int4Cache.empty`` makes them. The cache holds no lengths: the caller says where rows go and how many there
    are. Head dims 64 and 128.
    """

    def __init__(
        self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor
    ) -> None:
        _lib.torch_ext().int4_check(k_codes, k_params, v_codes, v_params)
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def capacity(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k_codes.shape[3] * 2

    @classmethod
    def empty(
        cls, batch: int, kv_heads: int, capacity: int, head_dim: int, device: torch.device | str = "cuda"
    ) -> Int4Cache:
        """A cache of zeros."""
        if head_dim not in (64, 128):
            raise ValueError(f"head dim must be 64 or 128, got {head_dim}")

        def one() -> tuple[torch.Tensor, torch.Tensor]:
            shape = (batch, kv_heads, capacity)
            return (
                torch.zeros((*shape, head_dim // 2), device=device, dtype=torch.uint8),
                torch.zeros((*shape, head_dim // GROUP, 2), device=device, dtype=torch.float16),
            )

        return cls(*one(), *one())

    def append(
        self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor | None = None, counts: torch.Tensor | None = None
    ) -> None:
        """Hold the rows of k and v, fp16 [batch, kv_heads, seq, dim], from position start[b] of sequence b on (None:
        0); with ``counts`` only the first counts[b] of them. Both are int32 [batch], on the device. A row past
        the capacity is not held and sets DEV_INDEX_RANGE in the device status word. k and v that need gradients are
        refused: the cache carries none."""
        _lib.torch_ext().int4_append(self.k_codes, self.k_params, self.v_codes, self.v_params, k, v, start, counts)

    def read(self, count: int, start: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values that ``count`` rows from position start[b] of sequence b on (None: 0) stand for: k and v, fp16
        [batch, kv_heads, count, dim]. A row past the capacity reads as zeros and sets DEV_INDEX_RANGE."""
        return _lib.torch_ext().int4_read(self.k_codes, self.k_params, self.v_codes, self.v_params, count, start)

    def attend(
        self, q: torch.Tensor, lengths: torch.Tensor, window: int | None = None, sinks: int = 0,
        sm_scale: float | None = None,
    ) -> torch.Tensor:  # fmt: skip
        """``decode_attention`` over this cache: q fp16 [batch, heads, 1, dim], the query's own token already held
        (lengths[b] counts it)."""
        return _lib.torch_ext().int4_attend(
            self.k_codes, self.k_params, self.v_codes, self.v_params, q, lengths, window, sinks, sm_scale
        )
