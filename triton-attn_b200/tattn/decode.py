"""Attention of one new token of each sequence over a cache: ``decode_attention`` over keys and values in the
queries' dtype, ``Int4Cache`` holding them in 4 bits.

The single-token form of ``tattn.window_attention``, for generation: no gradients, nothing read from the device
(the lengths stay there), so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

import math

import torch

from tattn import _lib
from tattn.api import _dtype_code, _require_cuda
from tattn.norm_rope import _like, _rows16
from tattn.window import INT_MAX, _check_heads, _check_window

GROUP = 64  # head dims that share a scale and a minimum in the 4-bit cache


def _check_token(q: torch.Tensor, lengths: torch.Tensor, window: int | None, sinks: int) -> None:
    if q.shape[2] != 1:
        raise ValueError(f"q holds one token of each sequence; got {q.shape}")
    if lengths.dtype != torch.int32 or lengths.shape != (q.shape[0],):
        raise ValueError(f"lengths must be int32 [{q.shape[0]}]; got {lengths.dtype} {tuple(lengths.shape)}")
    if lengths.get_device() != q.get_device():
        raise ValueError(f"lengths must be on q's device, got {lengths.device}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError("attention over a cache has no backward pass; use window_attention, or torch.no_grad()")
    _check_window(window, sinks)


def _scale(sm_scale: float | None, d: int) -> float:
    return float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(d)


def _workspace(size: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(size, device=device, dtype=torch.uint8) if size > 0 else None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


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
    _check_heads(q, k, v)
    _check_token(q, lengths, window, sinks)
    _require_cuda(q)
    lib = _lib.load()
    (z, h, _, d), (_, hk, cap, _), code = q.shape, k.shape, _dtype_code(q)
    if _rows16(k) is not k or _rows16(v) is not v:
        raise ValueError("k and v need contiguous, 16-byte aligned rows: a cache is read in place, never copied")
    q, lengths = _rows16(q), lengths.contiguous()
    out = _like(q)
    w, s = min(int(window or 0), INT_MAX), min(int(sinks), INT_MAX)
    at = q.get_device()
    with _lib.on_device(at):
        ws = _workspace(lib.tattn_decode_workspace_bytes(z, h, hk, cap, d, code, w, s), q.device)
        rc = lib.tattn_decode(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths.data_ptr(), out.data_ptr(), _ptr(ws),
            _lib.strides_bytes(q.stride() + k.stride() + v.stride() + out.stride()),
            z, h, hk, cap, d, code, w, s, _scale(sm_scale, d), _lib.raw_stream(at),
        )  # fmt: skip
    if rc:
        _lib.check("tattn_decode", rc)
    return out


class Int4Cache:
    """Keys and values of a batch of sequences, held in 4 bits.

    A group of 64 head dims of a token's head is held as a scale s and a minimum m (fp16) and codes n in 0..15,
    which stand for fp16(s n + m); appending rounds to the nearest code. Of normal heads that is within a
    thirtieth of the group's range. For keys and values each there are the tensors
    ``*_codes`` uint8 [batch, kv_heads, capacity, dim / 2] (head dim 2 i in the low half of byte i) and
    ``*_params`` float16 [batch, kv_heads, capacity, dim / 64, 2] (s, m); ``Int4Cache.empty`` makes them. The
    cache holds no lengths: the caller says where rows go and how many there are. Head dims 64 and 128.
    """

    def __init__(
        self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor
    ) -> None:
        shape = k_codes.shape
        if len(shape) != 4 or shape[3] not in (32, 64):
            raise ValueError(f"codes must be [batch, kv_heads, capacity, dim / 2] for dim 64 or 128; got {shape}")
        params = (*shape[:3], shape[3] * 2 // GROUP, 2)
        if v_codes.shape != shape or k_params.shape != params or v_params.shape != params:
            raise ValueError(
                f"expected codes {tuple(shape)} and params {params}; got {tuple(v_codes.shape)}, "
                f"{tuple(k_params.shape)}, {tuple(v_params.shape)}"
            )
        at = k_codes.get_device()
        for t, dtype in ((k_codes, torch.uint8), (k_params, torch.float16), (v_codes, torch.uint8), (v_params, torch.float16)):
            if t.dtype != dtype or t.get_device() != at:
                raise ValueError(f"codes must be uint8 and params float16 on one device; got {t.dtype} on {t.device}")
            if not t.is_contiguous() or t.data_ptr() % 16 != 0:
                raise ValueError("the cache's tensors must be contiguous and 16-byte aligned")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.batch, self.kv_heads, self.capacity, half = shape
        self.head_dim = half * 2
        self._at = at

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

    def _check_index(self, name: str, t: torch.Tensor | None) -> torch.Tensor | None:
        if t is None:
            return None
        if t.dtype != torch.int32 or t.shape != (self.batch,) or t.get_device() != self._at:
            raise ValueError(
                f"{name} must be int32 [{self.batch}] on {self.k_codes.device}; got {t.dtype} {tuple(t.shape)} on {t.device}"
            )
        return t.contiguous()

    def append(
        self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor | None = None, counts: torch.Tensor | None = None
    ) -> None:
        """Hold the rows of k and v, fp16 [batch, kv_heads, seq, dim], from position start[b] of sequence b on (None:
        0); with ``counts`` only the first counts[b] of them. A row past the capacity is not held and sets
        DEV_INDEX_RANGE in the device status word."""
        shape = k.shape
        if len(shape) != 4 or shape != (self.batch, self.kv_heads, shape[2], self.head_dim) or v.shape != shape:
            raise ValueError(
                f"expected k, v [{self.batch}, {self.kv_heads}, seq, {self.head_dim}]; got {tuple(k.shape)}, {tuple(v.shape)}"
            )
        if k.dtype != torch.float16 or v.dtype != torch.float16:
            raise ValueError(f"k, v must be float16, got {k.dtype}, {v.dtype}")
        if not (k.get_device() == v.get_device() == self._at):
            raise ValueError(f"k, v and the cache must be on one device, got {k.device}, {v.device}")
        start, counts = self._check_index("start", start), self._check_index("counts", counts)
        _require_cuda(k)
        lib = _lib.load()
        k, v = _rows16(k), _rows16(v)
        with _lib.on_device(self._at):
            rc = lib.tattn_int4_append(
                k.data_ptr(), v.data_ptr(), self.k_codes.data_ptr(), self.k_params.data_ptr(),
                self.v_codes.data_ptr(), self.v_params.data_ptr(), _ptr(start), _ptr(counts),
                _lib.strides_bytes(k.stride() + v.stride()), self.batch, self.kv_heads, shape[2], self.capacity,
                self.head_dim, _lib.raw_stream(self._at),
            )  # fmt: skip
        if rc:
            _lib.check("tattn_int4_append", rc)

    def read(self, count: int, start: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values that ``count`` rows from position start[b] of sequence b on (None: 0) stand for: k and v, fp16
        [batch, kv_heads, count, dim]. A row past the capacity reads as zeros and sets DEV_INDEX_RANGE."""
        if count < 0:
            raise ValueError(f"count must not be negative, got {count}")
        start = self._check_index("start", start)
        _require_cuda(self.k_codes)
        lib = _lib.load()
        shape = (self.batch, self.kv_heads, count, self.head_dim)
        k, v = self.k_params.new_empty(shape), self.k_params.new_empty(shape)
        with _lib.on_device(self._at):
            rc = lib.tattn_int4_read(
                self.k_codes.data_ptr(), self.k_params.data_ptr(), self.v_codes.data_ptr(), self.v_params.data_ptr(),
                _ptr(start), k.data_ptr(), v.data_ptr(), self.batch, self.kv_heads, count, self.capacity,
                self.head_dim, _lib.raw_stream(self._at),
            )  # fmt: skip
        if rc:
            _lib.check("tattn_int4_read", rc)
        return k, v

    def attend(
        self, q: torch.Tensor, lengths: torch.Tensor, window: int | None = None, sinks: int = 0,
        sm_scale: float | None = None,
    ) -> torch.Tensor:  # fmt: skip
        """``decode_attention`` over this cache: q fp16 [batch, heads, 1, dim], the query's own token already held
        (lengths[b] counts it)."""
        shape = q.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != self.head_dim:
            raise ValueError(f"expected q [{self.batch}, heads, 1, {self.head_dim}]; got {tuple(shape)}")
        if shape[1] == 0 or self.kv_heads == 0 or shape[1] % self.kv_heads != 0:
            raise ValueError(f"query heads must be a multiple of key/value heads; got {shape[1]} and {self.kv_heads}")
        if q.dtype != torch.float16:
            raise ValueError(f"q must be float16, got {q.dtype}")
        if q.get_device() != self._at:
            raise ValueError(f"q and the cache must be on one device, got {q.device}, {self.k_codes.device}")
        _check_token(q, lengths, window, sinks)
        _require_cuda(q)
        lib = _lib.load()
        z, h, _, d = shape
        q, lengths = _rows16(q), lengths.contiguous()
        out = _like(q)
        w, s = min(int(window or 0), INT_MAX), min(int(sinks), INT_MAX)
        with _lib.on_device(self._at):
            size = lib.tattn_int4_decode_workspace_bytes(z, h, self.kv_heads, self.capacity, d, w, s)
            ws = _workspace(size, q.device)
            rc = lib.tattn_int4_decode(
                q.data_ptr(), self.k_codes.data_ptr(), self.k_params.data_ptr(), self.v_codes.data_ptr(),
                self.v_params.data_ptr(), lengths.data_ptr(), out.data_ptr(), _ptr(ws),
                _lib.strides_bytes(q.stride() + out.stride()), z, h, self.kv_heads, self.capacity, d, w, s,
                _scale(sm_scale, d), _lib.raw_stream(self._at),
            )  # fmt: skip
        if rc:
            _lib.check("tattn_int4_decode", rc)
        return out
