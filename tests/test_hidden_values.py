"""What lies past a length at every head dim of ``tattn.cross_attention`` and ``tattn.prefix_decode_attention``, rows without
a softmax beside rows that have one, and sizes past 65,535 heads and 2^32 bytes (``tattn.qk_rope_axes`` too)."""

from __future__ import annotations

import math

import pytest
import torch

from tattn import _lib, cross_attention, prefix_decode_attention, qk_rope_axes
from tests.built import ensure_built
from tests.plain64 import assert_within, cross_attention64

ensure_built()

F16_F32 = pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
DIMS = pytest.mark.parametrize("d", [16, 32, 64, 128])


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0
    torch.cuda.empty_cache()


def _rand(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _int(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@F16_F32
@DIMS
@pytest.mark.parametrize("value", [math.nan, -math.inf])
@pytest.mark.parametrize("nq, nk, held", [(1, 300, 223), (3, 300, 1), (20, 2000, 1923), (90, 300, 223), (300, 700, 577)])
def test_past_a_length(gpu, nq, nk, held, value, d, dtype) -> None:
    """Results and gradients are the definition's, which looks at the held rows alone; gradients past a length are zeros.
    Lengths end inside a block of 64 and of 128 keys; 2 nq rows share a head, so the largest fill two tiles of 128."""
    q, do = _rand(3, 4, nq, d, dtype=dtype, seed=1), _rand(3, 4, nq, d, dtype=dtype, seed=2)
    k, v = _rand(3, 2, nk, d, dtype=dtype, seed=3), _rand(3, 2, nk, d, dtype=dtype, seed=4)
    lengths = _int(held, 0, max(held - 128, 0))
    past = (torch.arange(nk, device="cuda") >= lengths[:, None])[:, None, :, None]
    k, v = (t.masked_fill(past, value) for t in (k, v))
    want, bounds = cross_attention64(q, k, v, do, lengths, d**-0.5)
    with torch.no_grad():
        assert_within(cross_attention(q, k, v, lengths), want[0], bounds[0], "o alone")
    args = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*args, lengths)
    for got, w, e, name in zip((o, *torch.autograd.grad(o, args, do)), want, bounds, ("o", "dq", "dk", "dv"), strict=True):
        assert_within(got, w, e, name)
        if name in ("dk", "dv"):
            assert not bool(got.masked_select(past).any())


@pytest.mark.gpu
@F16_F32
@DIMS
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("samples", [1, 8, 16, 30, 70])
def test_past_a_prefix_and_own_lengths(gpu, samples, value, d, dtype) -> None:
    q = _rand(2 * samples, 8, 1, d, dtype=dtype, seed=1)
    pk, pv = _rand(2, 2, 500, d, dtype=dtype, seed=2), _rand(2, 2, 500, d, dtype=dtype, seed=3)
    k, v = _rand(2 * samples, 2, 90, d, dtype=dtype, seed=4), _rand(2 * samples, 2, 90, d, dtype=dtype, seed=5)
    prefix_lengths, lengths = [423, 0], [(13 * i) % 91 for i in range(2 * samples)]
    for p, n in enumerate(prefix_lengths):
        pk[p, :, n:], pv[p, :, n:] = value, value
    for b, n in enumerate(lengths):
        k[b, :, n:], v[b, :, n:] = value, value
    got = prefix_decode_attention(q, pk, pv, k, v, _int(*lengths), _int(*prefix_lengths))
    for b, n in enumerate(lengths):
        p = b // samples
        m = prefix_lengths[p]
        one = [torch.cat([x[p : p + 1, :, :m], y[b : b + 1, :, :n]], 2) for x, y in ((pk, k), (pv, v))]
        want, bounds = cross_attention64(q[b : b + 1], *one, q[b : b + 1], None, d**-0.5)
        assert_within(got[b : b + 1], want[0], bounds[0], "o")


@pytest.mark.gpu
@F16_F32
@DIMS
@pytest.mark.parametrize("nq, nk", [(1, 300), (20, 2000), (90, 300), (300, 700)])
def test_scores_without_a_softmax_and_the_rows_beside_them(gpu, nq, nk, d, dtype) -> None:
    """A NaN among the scores of some queries, infinite ones, and none but -infinity: NaN rows there, the definition's
    everywhere else, in the same head, the same group and the other sequence."""
    q, k, v = _rand(2, 6, nq, d, dtype=dtype, seed=1), _rand(2, 3, nk, d, dtype=dtype, seed=2), _rand(2, 3, nk, d, dtype=dtype, seed=3)
    dead = torch.zeros((2, 6, nq), dtype=torch.bool, device="cuda")
    q[0, 0, nq // 2, 3], dead[0, 0, nq // 2] = math.nan, True  # one query
    k[0, 1, nk - 1, 1], dead[0, 2:4] = math.nan, True  # a key: all queries of the group
    q[1, 0, nq - 1, 2], dead[1, 0, nq - 1] = math.inf, True  # scores of both infinities
    k[1, 2, :, 5], q[1, 4:, :, 5] = -math.inf, 1.0  # every key: nothing above -infinity
    dead[1, 4:] = True
    k[1, 1, : nk - 1, 4], q[1, 2:4, :, 4] = -math.inf, 1.0  # every key but one: its value
    o = cross_attention(q, k, v)
    assert bool(o[dead].isnan().all())
    want, bounds = cross_attention64(q, k.clone(), v, q, None, d**-0.5)
    rest = ~dead
    rest[1, 2:4] = False
    assert_within(o[rest], want[0][rest], bounds[0][rest], "o")
    one = v[1, 1, nk - 1].double().expand(2, nq, d)
    assert_within(o[1, 2:4], one, 2.0**-10 * one.abs(), "the only key above -infinity")


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("h, hk", [(1, 1), (2, 1)])
def test_more_heads_than_a_grid_dimension(gpu, h, hk, dtype) -> None:
    b, nq, nk, d = 70001, 3, 5, 16
    q, do = _rand(b, h, nq, d, dtype=dtype, seed=1), _rand(b, h, nq, d, dtype=dtype, seed=2)
    k, v = _rand(b, hk, nk, d, dtype=dtype, seed=3), _rand(b, hk, nk, d, dtype=dtype, seed=4)
    lengths = torch.arange(b, device="cuda", dtype=torch.int32) % (nk + 1)
    want, bounds = cross_attention64(q, k, v, do, lengths, d**-0.5)
    with torch.no_grad():
        assert_within(cross_attention(q, k, v, lengths), want[0], bounds[0], "o alone")
        one, e = cross_attention64(q[:, :, :1], k, v, q[:, :, :1], lengths, d**-0.5)
        assert_within(cross_attention(q[:, :, :1], k, v, lengths), one[0], e[0], "one token")
    args = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*args, lengths)
    for got, w, e, name in zip((o, *torch.autograd.grad(o, args, do)), want, bounds, ("o", "dq", "dk", "dv"), strict=True):
        assert_within(got, w, e, name)
    pk, pv = _rand(b, hk, 2, d, dtype=dtype, seed=5), _rand(b, hk, 2, d, dtype=dtype, seed=6)
    got = prefix_decode_attention(q[:, :, :1], pk, pv, k, v, torch.full_like(lengths, nk))
    want, bounds = cross_attention64(q[:, :, :1], torch.cat([pk, k], 2), torch.cat([pv, v], 2), q[:, :, :1], None, d**-0.5)
    assert_within(got, want[0], bounds[0], "over a prefix")


@pytest.mark.gpu
@F16_F32
def test_gradients_past_32_bits(gpu, dtype) -> None:
    """Q of more than 2^32 bytes over few keys, and few queries over K and V of that size each: of all but the last head
    everything is zeros, and so must its gradients be."""
    n, d = (1 << 18) if dtype == torch.float16 else 1 << 17, 128
    for nq, nk in ((n, 130), (70, n)):
        q, do = (torch.zeros((9, 8, nq, d), device="cuda", dtype=dtype) for _ in range(2))
        k, v = (torch.zeros((9, 8, nk, d), device="cuda", dtype=dtype) for _ in range(2))
        for i, t in enumerate((q, do, k, v)):
            t[-1, -1].normal_(generator=torch.Generator(device="cuda").manual_seed(i))
        args = [t.requires_grad_() for t in (q, k, v)]
        lengths = torch.full((9,), nk, dtype=torch.int32, device="cuda")
        lengths[-1] = nk - 3
        o = cross_attention(*args, lengths)
        grads = torch.autograd.grad(o, args, do)
        held = nk - 3
        for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv"), strict=True):
            assert not bool(got[:-1].any()) and not bool(got[-1, :-1].any()), name
        last = [t.detach()[-1:, -1:] for t in (q, k, v)]
        parts = range(0, nq, 1 << 14)  # of the queries: the definition's scores fit, and its sums are over parts
        want = None
        for i in parts:
            rows = slice(i, i + (1 << 14))
            w, e = cross_attention64(last[0][:, :, rows], last[1][:, :, :held], last[2][:, :, :held], do[-1:, -1:, rows], None, d**-0.5)
            assert_within(o[-1:, -1:, rows], w[0], e[0], "o")
            assert_within(grads[0][-1:, -1:, rows], w[1], e[1], "dq")
            want = [*w[2:], *e[2:]] if want is None else [a + b for a, b in zip(want, (*w[2:], *e[2:]), strict=True)]
        assert_within(grads[1][-1:, -1:, :held], want[0], want[2], "dk")
        assert_within(grads[2][-1:, -1:, :held], want[1], want[3], "dv")
        assert not bool(grads[1][-1, -1, held:].any()) and not bool(grads[2][-1, -1, held:].any())
        del q, k, v, do, o, grads, args, last, got
        torch.cuda.empty_cache()


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_rotation_past_32_bits(gpu, layout, norm, dtype) -> None:
    """Bitwise the results of the last tokens by themselves: of more than 2^31 values, fp16, and 2^32 bytes, fp32."""
    n, h, d = (1 << 17) + 5, 136 if dtype == torch.float16 else 68, 128
    g = torch.Generator(device="cuda").manual_seed(1)

    def make():
        shape = (1, h, n, d) if layout == "bhnd" else (1, n, h, d)
        t = torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g)
        return t if layout == "bhnd" else t.transpose(1, 2)

    q, dq = make(), make()
    k, dk = (t[:, -1:].clone() for t in (q, dq))
    angle = torch.rand((64, d // 2), generator=g, device="cuda") * 6
    positions = torch.randint(0, 64, (3, n), generator=g, device="cuda", dtype=torch.int32)
    weights = [1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2)] if norm else []
    axes = [j % 3 for j in range(d // 2)]

    def run(x, y, gx, gy, at):
        x, y = (t.detach().requires_grad_() for t in (x, y))
        outs = qk_rope_axes(x, y, angle.cos(), angle.sin(), at, axes, *weights)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, (x, y), (gx, gy)))

    whole = run(q, k, dq, dk, positions)
    last = slice(n - 300, n)
    part = run(*(t[:, :, last] for t in (q, k, dq, dk)), positions[:, last])
    for a, b, name in zip(whole, part, ("q", "k", "dq", "dk"), strict=True):
        assert torch.equal(a[:, :, last], b), name
    if not norm:  # the key head is the last query head
        assert torch.equal(whole[0][:, -1], whole[1][:, 0])
