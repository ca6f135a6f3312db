"""``tattn.window_attention``: refusals and host arithmetic without a GPU; outputs and gradients on a B200
against the definition in 64 bits, against differences, and against ``tattn.attention`` where both apply."""

from __future__ import annotations

import math

import pytest
import torch

import tattn
from tattn import _lib, attention, window_attention
from tattn.window import _backward, _forward
from tests.built import ensure_built
from tests.plain64 import assert_within, window_attention64

ensure_built()


def _qkv(b, h, hk, nq, nk, d, dtype, seed, layout="bhnd", device="cuda"):
    g = torch.Generator().manual_seed(seed)

    def make(heads, n):
        if layout == "bnhd":
            return torch.randn((b, n, heads, d), generator=g).to(dtype).to(device).transpose(1, 2)
        return torch.randn((b, heads, n, d), generator=g).to(dtype).to(device)

    return make(h, nq), make(hk, nk), make(hk, nk), make(h, nq)


# ------------------------------------------------------------------------------------ without a GPU
def _cpu(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize(
    "q, k, v, window, sinks, message",
    [
        (_cpu(1, 4, 8), _cpu(1, 2, 8, 16), _cpu(1, 2, 8, 16), 4, 0, "expected q"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 9, 16), 4, 0, "expected q"),
        (_cpu(2, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 8, 16), 4, 0, "agree in batch"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 32), _cpu(1, 2, 8, 32), 4, 0, "agree in batch"),
        (_cpu(1, 4, 8, 16), _cpu(1, 3, 8, 16), _cpu(1, 3, 8, 16), 4, 0, "multiple"),
        (_cpu(1, 4, 8, 16), _cpu(1, 0, 8, 16), _cpu(1, 0, 8, 16), 4, 0, "multiple"),
        (_cpu(1, 4, 8, 48), _cpu(1, 2, 8, 48), _cpu(1, 2, 8, 48), 4, 0, "head dim"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 8, 16, dtype=torch.float32), 4, 0, "dtype"),
        (*[_cpu(1, 2, 8, 16, dtype=torch.bfloat16)] * 3, 4, 0, "dtype"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 8, 16), 0, 0, "window"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 8, 16), 4, -1, "sinks"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 7, 16), _cpu(1, 2, 7, 16), 4, 0, "last of the keys"),
    ],
)
def test_refusals(q, k, v, window, sinks, message) -> None:
    with pytest.raises(ValueError, match=message):
        window_attention(q, k, v, window, sinks)


def test_no_cpu_path() -> None:
    x = _cpu(1, 2, 8, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        window_attention(x, x, x, 4)


def test_abi_refuses_before_any_device_call() -> None:
    lib = _lib.load()
    s = _lib.strides_array(*[(8 * 16, 8 * 16, 16, 1)] * 5)
    dims = dict(z=1, h=2, hk=2, nq=8, nk=8, d=16, dtype=0, window=4, sinks=0)
    for bad in (dict(d=24), dict(hk=0), dict(hk=3), dict(nk=7), dict(window=0), dict(sinks=-1), dict(dtype=2), dict(z=-1)):
        a = (dims | bad).values()
        assert lib.tattn_window_fwd(*[16] * 6, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_window_bwd(*[16] * 12, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_window_bwd_workspace_bytes(*a) == -1
    # No queries of no batch: nothing to do.
    assert lib.tattn_window_fwd(*[None] * 6, s, *(dims | dict(z=0)).values(), 0.1, None) == 0


def test_workspace_size() -> None:
    """The fp32 dQ rows and 16 bytes, and partial dV and dK of the key tiles that are several units' work: units of
    what a tile without sinks costs or, where that is more, of 8 blocks (a CTA's share is small here)."""
    size = _lib.load().tattn_window_bwd_workspace_bytes
    dq = 2 * 4 * 1000 * 64 * 4 + 16
    part = 2 * 2 * 2 * 128 * 64 * 4  # of one unit of each of the 2 * 2 key/value heads
    # A window of 100 meets ceil(227 / 128) + 1 = 3 of the 8 query blocks, of 2 heads: one unit a tile.
    assert size(2, 4, 2, 1000, 1000, 64, 0, 100, 0) == dq
    # The sink tile meets all 8, of 2 heads: 3 units of 6.
    assert size(2, 4, 2, 1000, 1000, 64, 0, 100, 4) == dq + 3 * part
    # A window of everything: 2 units for each of the 8 tiles.
    assert size(2, 4, 2, 1000, 1000, 64, 0, 1000, 4) == dq + 16 * part
    # fp32: tiles of 32 here and blocks of 64, no dQ rows; 4 and 16 blocks of 2 heads.
    assert size(2, 4, 2, 1000, 1000, 64, 1, 100, 0) == 0
    assert size(2, 4, 2, 1000, 1000, 64, 1, 100, 4) == 2 * 2 * 4 * 2 * 32 * 64 * 4


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0  # no bounded wait ran out


def _check(b, h, hk, nq, nk, d, window, sinks, dtype, seed=0, layout="bhnd", scale=None):
    q, k, v, do = _qkv(b, h, hk, nq, nk, d, dtype, seed, layout)
    for t in (q, k, v):
        t.requires_grad_()
    o = window_attention(q, k, v, window, sinks, scale)
    got = (o, *torch.autograd.grad(o, (q, k, v), do))
    want, bounds = window_attention64(q, k, v, do, window, sinks, 1 / math.sqrt(d) if scale is None else scale)
    for g, w, e, name in zip(got, want, bounds, ("o", "dq", "dk", "dv"), strict=True):
        assert g.dtype == dtype
        assert_within(g, w, e, name)


SHAPES = [
    # b, h, hk, nq, nk, window, sinks
    (1, 1, 1, 1, 1, 1, 0),
    (2, 2, 1, 1, 40, 7, 3),
    (1, 2, 2, 17, 17, 1, 0),  # every query sees itself alone
    (1, 2, 2, 33, 33, 1, 1),
    (2, 6, 2, 70, 70, 16, 4),
    (1, 3, 3, 128, 128, 128, 0),
    (1, 2, 1, 129, 129, 128, 1),
    (1, 4, 2, 300, 300, 64, 4),
    (1, 2, 2, 300, 300, 129, 128),
    (1, 2, 2, 700, 700, 100, 130),  # sinks end in the second tile, cut into chunks
    (1, 2, 2, 700, 700, 100, 600),  # sinks past most windows
    (2, 5, 1, 260, 515, 127, 2),  # queries begin inside a block
    (1, 2, 1, 40, 700, 50, 4),  # keys that no query sees
    (1, 2, 1, 100, 1000, 300, 200),
    (1, 2, 2, 200, 200, 10**9, 10**9),  # longer than the keys
    (3, 5, 5, 1000, 1000, 200, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(gpu, shape, d, dtype) -> None:
    b, h, hk, nq, nk, window, sinks = shape
    _check(b, h, hk, nq, nk, d, window, sinks, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("window, sinks", [(512, 4), (777, 130), (1500, 0), (64, 33)])
def test_longer_sequences(gpu, window, sinks, d) -> None:
    _check(1, 4, 2, 2500, 2500, d, window, sinks, torch.float16)
    _check(1, 4, 2, 1100, 2500, d, window, sinks, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("hk", [12, 4])
def test_many_tiles_in_fp32(gpu, hk, d) -> None:
    """96 query heads of 8 tiles of 64 rows fill the GPU five times: tiles of 64 rows, for 12 key heads also of keys."""
    _check(8, 12, hk, 500, 510, d, 90, 70, torch.float32)


@pytest.mark.gpu
def test_heads_in_sets(gpu) -> None:
    """fp16: 66 heads of 1,100 tokens, of which 59 with their tiles cut short by the ends are taken at once."""
    _check(6, 11, 11, 1100, 1100, 128, 1100, 4, torch.float16)
    _check(6, 11, 11, 1100, 1300, 128, 1200, 0, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(gpu, scale, dtype) -> None:
    _check(1, 4, 2, 300, 333, 64, 90, 4, dtype, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_transposed_layout_is_read_in_place(gpu, dtype) -> None:
    _check(2, 6, 3, 200, 290, 64, 70, 5, dtype, layout="bnhd")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_layouts_that_need_a_copy(gpu, dtype) -> None:
    """Odd strides, a base that no 16-byte load reaches and a broadcast dO give the dense tensors' results."""
    b, h, hk, n, d = 1, 4, 2, 150, 64
    q, k, v, _ = _qkv(b, h, hk, n, n, d, dtype, 3)
    odd = torch.empty((b, h, n, d + 1), device="cuda", dtype=dtype)[..., 1:].copy_(q)
    do = torch.randn((b, h, 1, d), device="cuda").to(dtype).expand(b, h, n, d)
    args = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    want = window_attention(*args, 40, 4)
    want_g = torch.autograd.grad(want, args, do.contiguous())
    odd.requires_grad_()
    got = window_attention(odd, args[1], args[2], 40, 4)
    assert torch.equal(got, want)
    got_g = torch.autograd.grad(got, (odd, args[1], args[2]), do)
    assert torch.equal(got_g[1], want_g[1]) and torch.equal(got_g[2], want_g[2])
    torch.testing.assert_close(got_g[0], want_g[0], atol=2e-3, rtol=2e-3)  # fp16 dQ sums in varying order


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_a_window_of_everything_is_causal_attention(gpu, d) -> None:
    q, k, v, do = _qkv(1, 3, 3, 400, 400, d, torch.float16, 5)
    ref = [t.clone().requires_grad_() for t in (q, k, v)]
    own = [t.clone().requires_grad_() for t in (q, k, v)]
    a, b = attention(*ref, causal=True), window_attention(*own, 400)
    torch.testing.assert_close(a, b, atol=2e-3, rtol=2e-3)
    for x, y in zip(torch.autograd.grad(a, ref, do), torch.autograd.grad(b, own, do), strict=True):
        torch.testing.assert_close(x, y, atol=2e-3, rtol=2e-3)


@pytest.mark.gpu
def test_gradients_against_differences(gpu) -> None:
    """fp32: d/de of sum(O * dO) along random directions by central differences. With e = 2e-3 the third
    derivative's part is of the order e^2 and the rounding of O about 2^-24 / e, both below 1e-3 of the
    slope's scale (the root of the number of summed products)."""
    q, k, v, do = _qkv(1, 4, 2, 90, 120, 32, torch.float32, 9)
    args = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*args, 30, 3), args, do)
    e = 2e-3
    for i, t in enumerate((q, k, v)):
        direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).cuda()
        values = []
        for sign in (1, -1):
            moved = [x + sign * e * direction if j == i else x for j, x in enumerate((q, k, v))]
            values.append((window_attention(*moved, 30, 3).double() * do.double()).sum())
        slope = float((values[0] - values[1]) / (2 * e))
        want = float((grads[i].double() * direction.double()).sum())
        size = float(grads[i].double().norm())
        assert abs(slope - want) <= 1e-3 * max(size, abs(want)), (i, slope, want, size)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_dk_and_dv_do_not_vary(gpu, d) -> None:
    """Cut sink tiles are summed in a fixed order: dK and dV are bitwise the same each time."""
    q, k, v, do = _qkv(2, 4, 2, 900, 900, d, torch.float16, 11)
    o, m = _forward(q, k, v, 100, 130, 0.125)
    first = _backward(q, k, v, o, m, do, 100, 130, 0.125)
    for _ in range(3):
        again = _backward(q, k, v, o, m, do, 100, 130, 0.125)
        assert torch.equal(first[1], again[1]) and torch.equal(first[2], again[2])


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 3, 8, 200])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_gradients_with_few_keys(gpu, window, d) -> None:
    """Rounding to fp16 is off by 2.1e-4 of a value in the root mean square (a last place of 2^-11 to 2^-10 of it). A
    gradient has that of itself, that of dS and some of that of P in O, and not that of O in delta, which with few
    keys is larger than the others: sqrt(3) 2.1e-4 bounds it. (At window 1 only dV is not zero.)"""
    q, k, v, do = _qkv(2, 4, 2, 500, 500, d, torch.float16, 21)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    window_attention(*leaves, window).backward(do)
    (_, *exact), _ = window_attention64(q, k, v, do, window, 0, 1 / math.sqrt(d))
    for x, want in list(zip(leaves, exact))[2 if window == 1 else 0 :]:
        assert (x.grad.double() - want).norm() <= math.sqrt(3) * 2.1e-4 * want.norm()


@pytest.mark.gpu
def test_log_sum_exp(gpu) -> None:
    q, k, v, _ = _qkv(1, 2, 1, 200, 330, 64, torch.float16, 12)
    _, m = _forward(q, k, v, 50, 3, 0.125)
    x = q.double() @ k.repeat_interleave(2, 1).double().transpose(-1, -2) * 0.125
    from tests.plain64 import visible

    x = x.masked_fill(~visible(200, 330, 50, 3, "cuda"), -math.inf)
    want = torch.logsumexp(x, -1) / math.log(2)
    torch.testing.assert_close(m.double(), want, atol=1e-3, rtol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_large_scores(gpu, dtype) -> None:
    """Scores of some hundreds: one key takes nearly all the weight, and the first block that a row sees may
    hold none of its keys. The output is a convex combination of rows of V."""
    q, k, v, _ = _qkv(1, 2, 1, 300, 300, 64, dtype, 13)
    o = window_attention(20 * q, k, v, 30, 2)
    assert bool(torch.isfinite(o).all())
    want, _ = window_attention64(20 * q, k, v, torch.zeros_like(q), 30, 2, 0.125)
    # 20 q doubles the exponent's size about 20 times over: its error, 2^-21 of some 300, is below 2e-4.
    torch.testing.assert_close(o.double(), want[0], atol=4e-3, rtol=4e-3)


@pytest.mark.gpu
def test_no_queries(gpu) -> None:
    q, k, v, do = _qkv(2, 2, 1, 0, 50, 64, torch.float16, 14)
    for t in (q, k, v):
        t.requires_grad_()
    o = window_attention(q, k, v, 8, 2)
    assert o.shape == q.shape
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    assert dq.shape == q.shape and not bool(dk.any()) and not bool(dv.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_nothing_to_attend_with(gpu, dtype) -> None:
    """No batch, or no query heads: empty results, and zeros for keys and values that no query sees."""
    for b, h in ((0, 2), (3, 0)):
        q, k, v, do = _qkv(b, h, 2, 5, 9, 32, dtype, 16)
        for t in (q, k, v):
            t.requires_grad_()
        o = window_attention(q, k, v, 4, 1)
        grads = torch.autograd.grad(o, (q, k, v), do)
        assert o.shape == q.shape and all(g.shape == t.shape for g, t in zip(grads, (q, k, v), strict=True))
        assert not bool(grads[1].any()) and not bool(grads[2].any())


@pytest.mark.gpu
def test_more_heads_than_a_grid_dimension(gpu) -> None:
    for dtype in (torch.float16, torch.float32):
        q, k, v, do = _qkv(66000, 1, 1, 3, 5, 16, dtype, 17)
        for t in (q, k, v):
            t.requires_grad_()
        o = window_attention(q, k, v, 2, 1)
        got = (o, *torch.autograd.grad(o, (q, k, v), do))
        want, bounds = window_attention64(q, k, v, do, 2, 1, 0.25)
        for g, w, e, name in zip(got, want, bounds, ("o", "dq", "dk", "dv"), strict=True):
            assert_within(g, w, e, name)


@pytest.mark.gpu
def test_side_stream_and_once_differentiable(gpu) -> None:
    q, k, v, do = _qkv(1, 4, 2, 500, 500, 64, torch.float16, 15)
    want = window_attention(q, k, v, 100, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = window_attention(q, k, v, 100, 4)
    side.synchronize()
    assert torch.equal(got, want)
    args = [t.clone().requires_grad_() for t in (q, k, v)]
    (g,) = torch.autograd.grad(window_attention(*args, 100, 4), args[:1], do.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    # ... and where the gradient is only a part of what is differentiated.
    args = [t.clone().requires_grad_() for t in (q, k, v)]
    (g,) = torch.autograd.grad(window_attention(*args, 100, 4), args[:1], do, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (g.sum() + args[0].sum()).backward()


def test_public_name() -> None:
    assert tattn.window_attention is window_attention and "window_attention" in tattn.__all__


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("how", ["window", "causal", "full"])
def test_a_key_that_is_not_a_number_shows(gpu, how, d, dtype) -> None:
    """Head i has a NaN in key i, i + 100 or 299 - i: the queries that see it give NaN and every other one what it
    gives without, wherever in a block the key lies."""
    n, heads = 300, 48
    q, k, v, _ = _qkv(1, heads, heads, n, n, d, dtype, 31)

    def call(k):
        return window_attention(q, k, v, 70, 9) if how == "window" else attention(q, k, v, causal=how == "causal")

    clean = call(k)
    p, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
    see = {"window": (j <= p) & ((j > p - 70) | (j < 9)), "causal": j <= p, "full": (j >= 0).expand(n, n)}[how]
    for at in (lambda i: i, lambda i: i + 100, lambda i: 299 - i):
        bad, keys = k.clone(), torch.tensor([at(i) for i in range(heads)], device="cuda")
        bad[0, torch.arange(heads, device="cuda"), keys, 5] = math.nan
        o, shows = call(bad), see[:, keys].T  # [heads, n]
        assert bool(o[0][shows].isnan().all()) and torch.equal(o[0][~shows], clean[0][~shows])
    if how == "window":
        m, clean_m = _forward(q, bad, v, 70, 9, 0.1)[1][0], _forward(q, k, v, 70, 9, 0.1)[1][0]
        assert bool(m[shows].isnan().all()) and torch.equal(m[~shows], clean_m[~shows])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("how", ["window", "causal", "full"])
def test_a_query_that_is_not_a_number_shows_in_the_gradients(gpu, how, d, dtype) -> None:
    """Head i has a NaN in query i, i + 100 or 299 - i: its weights are NaN, so dV and dK of the keys that it sees are no
    numbers, nor is its own dQ. In each of another head's gradients all is finite."""
    n, heads = 300, 48
    q, k, v, do = _qkv(1, heads, heads, n, n, d, dtype, 32)
    p, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
    see = {"window": (j <= p) & ((j > p - 70) | (j < 9)), "causal": j <= p, "full": (j >= 0).expand(n, n)}[how]
    for at in (lambda i: i, lambda i: i + 100, lambda i: 299 - i):
        bad, rows = q.clone(), torch.tensor([at(i) for i in range(heads)], device="cuda")
        every = torch.arange(0, heads, 2, device="cuda")  # the even heads
        bad[0, every, rows[every], 5] = math.nan
        args = [t.clone().requires_grad_() for t in (bad, k, v)]
        o = window_attention(*args, 70, 9) if how == "window" else attention(*args, causal=how == "causal")
        dq, dk, dv = torch.autograd.grad(o, args, do)
        shows = see[rows[every]]  # [heads, keys]
        assert not bool(torch.isfinite(dq[0, every, rows[every]]).any())
        for g in (dk, dv):
            assert not bool(torch.isfinite(g[0, every][shows]).any())
        for g in (dq, dk, dv):
            assert bool(torch.isfinite(g[0, 1::2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_scores_of_minus_infinity(gpu, d, dtype) -> None:
    """Keys with an infinity that makes their scores -infinity weigh nothing; a query that sees no others has no result
    and a log-sum-exp of -infinity."""
    n = 300
    q, k, v, _ = _qkv(1, 4, 2, n, n, d, dtype, 33)
    q[..., 3] = 1.0
    for first, last in ((0, 150), (0, 290), (130, 300)):
        bad = k.clone()
        bad[:, :, first:last, 3] = -math.inf
        o, m = _forward(q, bad, v, 70, 0, 0.2)
        p, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
        see = (j <= p) & (j > p - 70) & ((j < first) | (j >= last))
        none = ~see.any(1)
        assert bool(o[:, :, none].isnan().all()) and bool((m[:, :, none] == -math.inf).all())
        x = (q.double() @ k.repeat_interleave(2, 1).double().transpose(-1, -2) * 0.2).masked_fill(~see, -math.inf)
        w = torch.softmax(x, -1)[:, :, ~none]
        vx = v.repeat_interleave(2, 1).double()
        # As plain64: each weight is off by c of it, the result by its rounding.
        c, u = (1e-3, 2.0**-11) if dtype == torch.float16 else ((n + d) * 2.0**-23 + 1e-6, 2.0**-24)
        assert_within(o[:, :, ~none], w @ vx, c * (w @ vx.abs()) + 2 * u * (w @ vx).abs() + 2.0**-24, "o")


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(which) -> None:
    """As tattn.attention refuses them: not a result without a tangent. (Without a GPU: before the device check.)"""
    with torch.autograd.forward_ad.dual_level():
        args = [_cpu(1, 2, 8, 16) for _ in range(3)]
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for take in (torch.enable_grad, torch.no_grad):
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                window_attention(*args, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_forward_and_backward_on_side_streams(gpu, dtype) -> None:
    """Two streams work on different inputs at the same time, forward and backward (whose kernel has its workspace and a
    barrier over its few CTAs): each gets its own inputs' results."""
    b, h, hk, n, d, window, sinks = 1, 4, 2, 500, 64, 100, 130
    inputs = [_qkv(b, h, hk, n, n, d, dtype, 40 + i) for i in range(2)]
    want = [window_attention64(*x, window, sinks, d**-0.5) for x in inputs]
    args = [[t.detach().clone().requires_grad_() for t in x[:3]] for x in inputs]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                o = window_attention(*args[i], window, sinks)
                got[i].append((o, *torch.autograd.grad(o, args[i], inputs[i][3])))
    for side in sides:
        side.synchronize()
    for results, (outs, bounds) in zip(got, want, strict=True):
        for result in results:
            for g, w, e, name in zip(result, outs, bounds, ("o", "dq", "dk", "dv"), strict=True):
                assert_within(g, w, e, name)
                if dtype == torch.float32 or name != "dq":  # (its sums vary in order in fp16)
                    assert torch.equal(g, results[0][("o", "dq", "dk", "dv").index(name)])
