"""One attention layer with head norms, rotation and a sliding window: trained on whole sequences, then generating
token by token from a 4-bit cache.

    python examples/window_layer.py

Training goes through ``tattn.qk_norm_rope`` and ``tattn.window_attention`` with their gradients. Generation takes
a prompt the same way and appends its keys and values to a ``tattn.Int4Cache``; every further token is one
captured CUDA graph of ``qk_norm_rope``, ``Int4Cache.append`` and ``Int4Cache.attend``, with the lengths
counted on the device. Prints the training loss and how far the generated outputs are from the layer's own
on the whole sequence (the 4-bit rounding of keys and values).
"""

from __future__ import annotations

import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-attn_b200"))
import tattn  # noqa: E402


class WindowLayer(nn.Module):
    """x [batch, seq, width] -> the same, in fp16 on an sm_100 GPU."""

    def __init__(
        self, width: int, heads: int, kv_heads: int, dim: int, window: int, sinks: int, positions: int = 8192
    ) -> None:
        super().__init__()
        self.heads, self.kv_heads, self.dim, self.window, self.sinks = heads, kv_heads, dim, window, sinks
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * dim, bias=False)
        self.out = nn.Linear(heads * dim, width, bias=False)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.ones(dim))
        # Angles in 64 bits (one of thousands in 32 is off by 2^-12), their cosines and sines in 32.
        inverse = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
        self.register_buffer("cos", angle.cos().float(), persistent=False)
        self.register_buffer("sin", angle.sin().float(), persistent=False)

    def _project(
        self, x: torch.Tensor, positions: torch.Tensor | None
    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q, k, v as [batch, heads, seq, dim] views of the projection; q and k normed and rotated."""
        b, n, _ = x.shape
        y = self.qkv(x).view(b, n, self.heads + 2 * self.kv_heads, self.dim).transpose(1, 2)
        q, k, v = y.split((self.heads, self.kv_heads, self.kv_heads), 1)
        q, k = tattn.qk_norm_rope(q, k, self.q_norm, self.k_norm, self.cos, self.sin, positions)
        return q, k, v

    def _merge(self, o: torch.Tensor) -> torch.Tensor:
        return self.out(o.transpose(1, 2).flatten(2))

    def forward(self, x: torch.Tensor, cache: tattn.Int4Cache | None = None) -> torch.Tensor:
        """Whole sequences; with ``cache`` their keys and values are kept there from position 0 on."""
        q, k, v = self._project(x, None)
        if cache is not None:
            cache.append(k, v)
        return self._merge(tattn.window_attention(q, k, v, self.window, self.sinks))

    def step(self, x: torch.Tensor, cache: tattn.Int4Cache, held: torch.Tensor) -> torch.Tensor:
        """One new token of each sequence, x [batch, 1, width]; held (int32 [batch]) counts the tokens in the cache
        and is raised by one."""
        q, k, v = self._project(x, held[:, None])
        cache.append(k, v, held)
        held.add_(1)
        return self._merge(cache.attend(q, held, self.window, self.sinks))


def make_layer(width: int, device: str) -> WindowLayer:
    """The projections in fp16; the norms' weights and the tables stay in fp32."""
    layer = WindowLayer(width, heads=8, kv_heads=2, dim=64, window=64, sinks=4)
    layer.qkv.half()
    layer.out.half()
    return layer.to(device)


def train(layer: WindowLayer, steps: int, batch: int, seq: int, width: int) -> list[float]:
    """Adam on one batch: each output is to be the input 7 tokens before. Returns the losses."""
    x = torch.randn((batch, seq, width), device="cuda", dtype=torch.float16)
    want = x.float().roll(7, 1)
    master = {name: p.detach().float() for name, p in layer.named_parameters()}  # fp32 weights
    adam = torch.optim.Adam(master.values(), lr=3e-3)
    losses = []
    for _ in range(steps):
        loss = (layer(x).float() - want)[:, 7:].square().mean()
        layer.zero_grad()
        (1024 * loss).backward()  # scaled: fp16 gradients of a mean over many values are small
        for name, p in layer.named_parameters():
            master[name].grad = p.grad.float() / 1024
        adam.step()
        with torch.no_grad():
            for name, p in layer.named_parameters():
                p.copy_(master[name])
        losses.append(loss.item())
    return losses


@torch.no_grad()
def generate(layer: WindowLayer, batch: int, prompt: int, tokens: int, width: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Outputs for the tokens after the prompt, by steps from the 4-bit cache and by the layer on the whole sequence."""
    x = torch.randn((batch, prompt + tokens, width), device="cuda", dtype=torch.float16)
    cache = tattn.Int4Cache.empty(batch, layer.kv_heads, prompt + tokens, layer.dim)
    layer(x[:, :prompt], cache)
    token, held = x[:, :1].clone(), torch.full((batch,), prompt, device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up outside the capture
        layer.step(token, cache, held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(token, cache, held)
    held.fill_(prompt)
    outs = []
    for i in range(tokens):
        token.copy_(x[:, prompt + i : prompt + i + 1])
        graph.replay()
        outs.append(out.clone())
    return torch.cat(outs, 1), layer(x)[:, prompt:]


def main() -> tuple[list[float], float]:
    torch.manual_seed(0)
    width = 256
    layer = make_layer(width, "cuda")
    losses = train(layer, 60, batch=4, seq=500, width=width)
    print(f"training loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    steps, whole = generate(layer, batch=3, prompt=150, tokens=40, width=width)
    off = float((steps.float() - whole.float()).norm() / whole.float().norm())
    print(f"generation from the 4-bit cache: relative difference {off:.3f}")
    return losses, off


if __name__ == "__main__":
    main()
