"""B200-native FlashAttention-2 (sm_100a CUDA behind a C ABI), drop-in for amaanmithani/triton-attn's
``tattn`` package (src/tattn/__init__.py:3-5)."""

from tattn.api import attention, cuda_available, triton_available
from tattn.decode import Int4Cache, decode_attention
from tattn.norm_rope import qk_norm_rope
from tattn.window import window_attention

__all__ = [
    "Int4Cache",
    "attention",
    "cuda_available",
    "decode_attention",
    "qk_norm_rope",
    "triton_available",
    "window_attention",
]
