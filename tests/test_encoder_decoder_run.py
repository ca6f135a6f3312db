"""A decoder layer that stands at (time, row, column), attends to itself and to an encoder's states: trained, and then
answering each prompt several times from one cache of the prompt. All of it through the package's operators together, against
the same layer in 64 bits and against itself on whole sequences."""

from __future__ import annotations

import math

import pytest
import torch

from tattn import _lib, cross_attention, prefix_decode_attention, qk_rope_axes, window_attention
from tests.built import ensure_built

ensure_built()

HEADS, KV, DIM, WIDTH = 4, 2, 64, 128
AXES = [0] * 8 + [j % 2 + 1 for j in range(24)]  # a run of time, then rows and columns in turn


def _weights(seed):
    g = torch.Generator().manual_seed(seed)

    def make(*shape):
        return torch.randn(shape, generator=g) / math.sqrt(shape[0])

    w = dict(
        qkv=make(WIDTH, (HEADS + 2 * KV) * DIM), out=make(HEADS * DIM, WIDTH), q2=make(WIDTH, HEADS * DIM),
        kv2=make(WIDTH, 2 * KV * DIM), out2=make(HEADS * DIM, WIDTH),
    )  # fmt: skip
    w = {k: v.half().cuda().requires_grad_() for k, v in w.items()}
    w["nq"], w["nk"] = ((1 + 0.1 * torch.randn(DIM, generator=g)).cuda().requires_grad_() for _ in range(2))
    return w


def _tables(n):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2).double() / DIM)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def _places(b, n):
    """[3, b, n]: some text, an image of 5 columns, text again."""
    i = torch.arange(n)
    image = (i >= 7) & (i < 32)
    time = torch.where(i < 7, i, torch.where(image, torch.full_like(i, 7), i - 20))
    row, col = torch.where(image, time + (i - 7) // 5, time), torch.where(image, time + (i - 7) % 5, time)
    return torch.stack((time, row, col)).to(torch.int32)[:, None].expand(3, b, n).cuda()


def _heads(x, count):
    return x.unflatten(-1, (count, DIM)).transpose(1, 2)


def _layer(x, places, states, held, w, tables):
    q, k, v = _heads(x @ w["qkv"], HEADS + 2 * KV).split((HEADS, KV, KV), 1)
    q, k = qk_rope_axes(q, k, *tables, places, AXES, w["nq"], w["nk"])
    h = x + window_attention(q, k, v, x.shape[1]).transpose(1, 2).flatten(2) @ w["out"]
    ke, ve = _heads(states @ w["kv2"], 2 * KV).split((KV, KV), 1)
    o = cross_attention(_heads(h @ w["q2"], HEADS), ke, ve, held)
    return h + o.transpose(1, 2).flatten(2) @ w["out2"], (k, v, ke, ve)


def _layer64(x, places, states, held, w, tables):
    """The same in 64 bits and plain products."""
    w = {k: t.double() for k, t in w.items()}
    q, k, v = _heads(x @ w["qkv"], HEADS + 2 * KV).split((HEADS, KV, KV), 1)
    co, si = (t.double()[places.long()[AXES].permute(1, 2, 0), torch.arange(DIM // 2, device="cuda")][:, None] for t in tables)

    def turn(z, weight):
        z = z * (z.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight
        a, b = z.chunk(2, -1)
        return torch.cat((a * co - b * si, b * co + a * si), -1)

    def attend(q, k, v, hidden):
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        p = torch.softmax((q @ k.transpose(-1, -2) / math.sqrt(DIM)).masked_fill(hidden, -math.inf), -1)
        return (p @ v).transpose(1, 2).flatten(2)

    n = x.shape[1]
    ahead = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    h = x + attend(turn(q, w["nq"]), turn(k, w["nk"]), v, ahead) @ w["out"]
    ke, ve = _heads(states @ w["kv2"], 2 * KV).split((KV, KV), 1)
    past = torch.arange(states.shape[1], device="cuda") >= held[:, None]
    return h + attend(_heads(h @ w["q2"], HEADS), ke, ve, past[:, None, None]) @ w["out2"]


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_gradients(gpu) -> None:
    """Of every weight and both inputs, against 64 bits. Each of some ten steps rounds its 16-bit results, and sums of
    independent roundings of 2^-11 each are far below 1 % of a gradient's norm."""
    g = torch.Generator().manual_seed(1)
    x, states, dy = (torch.randn((3, n, WIDTH), generator=g).half().cuda() for n in (50, 90, 50))
    held = torch.tensor([90, 17, 64], dtype=torch.int32, device="cuda")
    w, tables, places = _weights(2), _tables(64), _places(3, 50)
    inputs = [x.requires_grad_(), states.requires_grad_(), *w.values()]
    y, _ = _layer(x, places, states, held, w, tables)
    grads = torch.autograd.grad(y, inputs, dy)
    w64 = {k: t.detach().double().requires_grad_() for k, t in w.items()}
    inputs64 = [x.detach().double().requires_grad_(), states.detach().double().requires_grad_(), *w64.values()]
    y64 = _layer64(inputs64[0], places, inputs64[1], held, w64, tables)
    want = torch.autograd.grad(y64, inputs64, dy.double())
    for name, a, b in zip(("y", "x", "states", *w), (y.detach(), *grads), (y64.detach(), *want), strict=True):
        assert float((a.double() - b).norm()) <= 1e-2 * float(b.norm()), name
    assert not bool(grads[1][1, 17:].any()) and not bool(grads[1][2, 64:].any())


@pytest.mark.gpu
def test_samples_of_prompts(gpu) -> None:
    """Two prompts of 41 tokens, three samples of each, ten tokens a sample by one captured step, against the layer on
    whole sequences; fp16 throughout on both sides, so 1 % of the norm again."""
    prompts, samples, prompt, tokens = 2, 3, 41, 10
    g = torch.Generator().manual_seed(3)
    b = prompts * samples
    states = torch.randn((prompts, 90, WIDTH), generator=g).half().cuda()
    held = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    x = torch.randn((prompts, prompt, WIDTH), generator=g).half().cuda()
    own = torch.randn((b, tokens, WIDTH), generator=g).half().cuda()
    w, tables = {k: t.detach() for k, t in _weights(4).items()}, _tables(64)
    places = _places(b, prompt + tokens)
    with torch.no_grad():
        _, (pk, pv, ke, ve) = _layer(x, places[:, :prompts, :prompt], states, held, w, tables)
        ke, ve, held_b = (t.repeat_interleave(samples, 0) for t in (ke, ve, held))
        k_cache, v_cache = (torch.zeros((b, KV, tokens, DIM), device="cuda", dtype=torch.float16) for _ in range(2))
        token, at = own[:, :1].clone(), places[:, :, prompt : prompt + 1].clone()
        step = torch.zeros(1, dtype=torch.long, device="cuda")
        lengths = torch.zeros(b, dtype=torch.int32, device="cuda")

        def one():
            q, k, v = _heads(token @ w["qkv"], HEADS + 2 * KV).split((HEADS, KV, KV), 1)
            q, k = qk_rope_axes(q, k, *tables, at, AXES, w["nq"], w["nk"])
            k_cache.index_copy_(2, step, k)
            v_cache.index_copy_(2, step, v)
            step.add_(1)
            lengths.add_(1)
            o = prefix_decode_attention(q, pk, pv, k_cache, v_cache, lengths)
            h = token + o.transpose(1, 2).flatten(2) @ w["out"]
            o = cross_attention(_heads(h @ w["q2"], HEADS), ke, ve, held_b)
            return h + o.transpose(1, 2).flatten(2) @ w["out2"]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = one()
        step.zero_()
        lengths.zero_()
        outs = []
        for i in range(tokens):
            token.copy_(own[:, i : i + 1])
            at.copy_(places[:, :, prompt + i : prompt + i + 1])
            graph.replay()
            outs.append(y.clone())
        whole = torch.cat((x.repeat_interleave(samples, 0), own), 1)
        want, _ = _layer(whole, places, states.repeat_interleave(samples, 0), held_b, w, tables)
    got, want = torch.cat(outs, 1).double(), want[:, prompt:].double()
    assert float((got - want).norm()) <= 1e-2 * float(want.norm())
