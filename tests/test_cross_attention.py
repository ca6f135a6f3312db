"""``tattn.cross_attention``: refusals and host arithmetic without a GPU; outputs and gradients on a B200 against the
definition in 64 bits, against differences, and against ``tattn.attention`` where both apply."""

from __future__ import annotations

import math

import pytest
import torch

import tattn
from tattn import _lib, attention, cross_attention
from tests.built import ensure_built
from tests.plain64 import assert_within, cross_attention64

ensure_built()

F16_F32 = pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])


def _qkv(b, h, hk, nq, nk, d, dtype, seed, layout="bhnd"):
    g = torch.Generator().manual_seed(seed)

    def make(heads, n):
        if layout == "bnhd":
            return torch.randn((b, n, heads, d), generator=g).to(dtype).cuda().transpose(1, 2)
        return torch.randn((b, heads, n, d), generator=g).to(dtype).cuda()

    return make(h, nq), make(hk, nk), make(hk, nk), make(h, nq)


def _int(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------ without a GPU
def _cpu(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize(
    "q, k, v, lengths, message",
    [
        (_cpu(1, 4, 8), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16), None, "expected q"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 8, 16), _cpu(1, 2, 9, 16), None, "expected q"),
        (_cpu(2, 4, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16), None, "agree in batch"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 9, 32), _cpu(1, 2, 9, 32), None, "agree in batch"),
        (_cpu(1, 4, 8, 16), _cpu(1, 3, 9, 16), _cpu(1, 3, 9, 16), None, "multiple"),
        (_cpu(1, 4, 8, 16), _cpu(1, 0, 9, 16), _cpu(1, 0, 9, 16), None, "multiple"),
        (_cpu(1, 4, 8, 48), _cpu(1, 2, 9, 48), _cpu(1, 2, 9, 48), None, "head dim"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16, dtype=torch.float32), None, "dtype"),
        (_cpu(1, 2, 8, 16, dtype=torch.bfloat16), *[_cpu(1, 2, 9, 16, dtype=torch.bfloat16)] * 2, None, "dtype"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16), torch.zeros(1), "lengths must be int32"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16), torch.zeros(2, dtype=torch.int32), "lengths must be int32"),
        (_cpu(1, 4, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16), torch.zeros((), dtype=torch.int32), "lengths must be int32"),
    ],
)
def test_refusals(q, k, v, lengths, message) -> None:
    with pytest.raises(ValueError, match=message):
        cross_attention(q, k, v, lengths)


def test_no_cpu_path() -> None:
    with pytest.raises(RuntimeError, match="no CPU path"):
        cross_attention(_cpu(1, 2, 8, 16), _cpu(1, 2, 9, 16), _cpu(1, 2, 9, 16))
    assert "cross_attention" in tattn.__all__


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_derivatives_are_refused(which) -> None:
    with torch.autograd.forward_ad.dual_level():
        args = [torch.zeros(1, 2, 8, 16) for _ in range(3)]
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for take in (torch.enable_grad, torch.no_grad):
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                cross_attention(*args)


def test_abi_refuses_before_any_device_call() -> None:
    lib = _lib.load()
    s = _lib.strides_array(*[(8 * 16, 8 * 16, 16, 1)] * 5)
    dims = dict(z=1, h=2, hk=2, nq=8, nk=9, d=16, dtype=0)
    for bad in (dict(d=24), dict(hk=0), dict(h=3), dict(nk=-1), dict(nq=-1), dict(dtype=2), dict(z=-1), dict(nk=(1 << 29) + 1)):
        a = (dims | bad).values()
        assert lib.tattn_cross_fwd(*[16] * 8, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_cross_bwd(*[16] * 13, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_cross_fwd_workspace_bytes(*a) == lib.tattn_cross_bwd_workspace_bytes(*a) == -1
    large = (dims | dict(z=1 << 20, nq=1 << 10)).values()
    assert lib.tattn_cross_fwd(*[16] * 8, s, *large, 0.1, None) == _lib.ERR_TOO_LARGE
    assert lib.tattn_cross_bwd(*[16] * 13, s, *large, 0.1, None) == _lib.ERR_TOO_LARGE
    # No batch: nothing to do. A pointer that 16-byte loads do not reach, and none at all.
    assert lib.tattn_cross_fwd(*[None] * 8, s, *(dims | dict(z=0)).values(), 0.1, None) == 0
    assert lib.tattn_cross_fwd(17, *[16] * 7, s, *dims.values(), 0.1, None) == _lib.ERR_LAYOUT
    assert lib.tattn_cross_fwd(None, *[16] * 7, s, *dims.values(), 0.1, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.tattn_cross_bwd(*[16] * 4, None, *[16] * 8, s, *dims.values(), 0.1, None) == _lib.ERR_INVALID_ARGUMENT


def test_workspace_size() -> None:
    """By the sizes alone: partial rows of a row tile whose keys are cut, none where the tiles fill the GPU (148 SMs are
    assumed without one)."""
    size = _lib.load().tattn_cross_fwd_workspace_bytes
    assert size(8, 16, 16, 2048, 1500, 64, 0) == 0
    part = size(1, 16, 16, 64, 16384, 64, 0)
    assert part > 0 and part % (16 * 64 * (64 + 2) * 4) == 0
    assert size(0, 16, 16, 64, 16384, 64, 0) == 0
    back = _lib.load().tattn_cross_bwd_workspace_bytes
    assert back(1, 2, 2, 8, 0, 64, 0) == 2 * 8 * 64 * 4 + 16 and back(1, 2, 2, 0, 8, 64, 0) == 0


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0  # no bounded wait ran out


def _compare(q, k, v, do, lengths, scale=None):
    """Forward, forward for a backward, and backward against the definition."""
    with torch.no_grad():
        alone = cross_attention(q, k, v, lengths, scale)
    args = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*args, lengths, scale)
    grads = torch.autograd.grad(o, args, do)
    want, bounds = cross_attention64(q, k, v, do, lengths, 1 / math.sqrt(q.shape[3]) if scale is None else scale)
    for g, w, e, name in zip((alone, o, *grads), (want[0], *want), (bounds[0], *bounds), ("o alone", "o", "dq", "dk", "dv"), strict=True):
        assert g.dtype == q.dtype
        assert_within(g, w, e, name)


SHAPES = [
    # b, h, hk, nq, nk, lengths
    (1, 1, 1, 1, 1, None),
    (2, 2, 1, 1, 40, (40, 0)),
    (3, 4, 2, 1, 300, (300, 1, 129)),
    (2, 6, 2, 3, 70, (33, 64)),
    (1, 2, 2, 17, 5, None),
    (2, 2, 2, 40, 128, (127, 128)),
    (2, 2, 1, 128, 129, (129, 128)),
    (3, 5, 5, 129, 65, (0, 1, 65)),
    (2, 8, 2, 70, 515, (515, 257)),
    (1, 3, 3, 300, 300, None),
    (2, 4, 1, 257, 1000, (1000, 385)),
    (1, 2, 2, 700, 33, (32,)),
    (4, 2, 2, 5, 2000, (2000, 0, 64, 1999)),  # few rows: the keys are cut into parts, some without any
]


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(gpu, shape, d, dtype) -> None:
    b, h, hk, nq, nk, lengths = shape
    _compare(*_qkv(b, h, hk, nq, nk, d, dtype, nq + nk), None if lengths is None else _int(*lengths))


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_longer_sequences(gpu, d, layout, dtype) -> None:
    _compare(*_qkv(2, 4, 2, 1100, 2500, d, dtype, 1, layout), _int(2500, 1201))
    _compare(*_qkv(1, 8, 2, 45, 5000, d, dtype, 2, layout), _int(4999))
    _compare(*_qkv(9, 16, 4, 10, 130, d, dtype, 3, layout), _int(*[15 * i for i in range(9)]))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_tiles(gpu, d) -> None:
    """More tiles than the GPU holds at a time, fp32 tiles of 64 rows among them."""
    _compare(*_qkv(8, 12, 12, 500, 510, d, torch.float32, 1), _int(*[510 - 60 * i for i in range(8)]))
    _compare(*_qkv(8, 12, 12, 500, 510, d, torch.float16, 1), _int(*[510 - 60 * i for i in range(8)]))
    _compare(*_qkv(30, 12, 4, 130, 140, d, torch.float16, 1), _int(*[min(i * 5, 140) for i in range(30)]))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("b, h, hk, nq, nk", [(1, 1, 1, 2000, 100), (2, 8, 2, 300, 1300), (70, 2, 1, 130, 400), (40, 4, 4, 260, 250)])
def test_tiles_cut_between_ctas(gpu, b, h, hk, nq, nk, d) -> None:
    """fp16 backward: a last round of few key tiles is cut into runs of pairs; batches of more than 32 sequences, with and
    without lengths (every third none)."""
    inputs = _qkv(b, h, hk, nq, nk, d, torch.float16, 2)
    _compare(*inputs, None)
    _compare(*inputs, _int(*[(i * 53) % (nk + 1) if i % 3 else 0 for i in range(1, b + 1)]))


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("nq", [1, 4, 300])
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(gpu, scale, nq, dtype) -> None:
    _compare(*_qkv(1, 4, 2, nq, 333, 64, dtype, 1), _int(301), scale)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nq, nk", [(1, 300), (3, 300), (40, 2000), (300, 300)])
def test_what_lies_past_a_length_is_never_used(gpu, nq, nk, value, dtype) -> None:
    """Bitwise the results with zeros there, but for fp16 dQ, whose sums' order varies; gradients there are zeros."""
    q, k, v, do = _qkv(2, 4, 2, nq, nk, 64, dtype, 5)
    held = _int(nk - 77, 0)
    past = (torch.arange(nk, device="cuda") >= held[:, None])[:, None, :, None]
    results = []
    for fill in (0.0, value):
        args = [q.clone().requires_grad_(), *(torch.where(past, fill, t).to(dtype).requires_grad_() for t in (k, v))]
        with torch.no_grad():
            alone = cross_attention(*args, held)
        o = cross_attention(*args, held)
        results.append((alone, o, *torch.autograd.grad(o, args, do)))
    for name, a, b in zip(("alone", "o", "dq", "dk", "dv"), *results, strict=True):
        if name == "dq" and dtype == torch.float16:
            torch.testing.assert_close(a, b, atol=2e-3, rtol=2e-3)
        else:
            assert torch.equal(a, b), name
    for g in results[1][3:]:
        assert not bool(g.masked_select(past).any())


@pytest.mark.gpu
@F16_F32
def test_gradients_past_a_length_are_zeros_whatever_the_rest_is(gpu, dtype) -> None:
    """A NaN in one query and an infinity in dO reach the keys that are seen (as a NaN or an infinity: fp16's exponentials
    make either of a NaN), not those behind them."""
    q, k, v, do = _qkv(2, 4, 2, 50, 300, 64, dtype, 6)
    q[0, 0, 3, 5] = math.nan
    do[1, 1, 7, 9] = math.inf
    args = [t.requires_grad_() for t in (q, k, v)]
    held = _int(200, 130)
    dq, dk, dv = torch.autograd.grad(cross_attention(*args, held), args, do)
    for g in (dk, dv):
        assert not bool(g[0, :, 200:].any()) and not bool(g[1, :, 130:].any())
        assert not bool(g[0, 0, :200].isfinite().all()) and bool(g[1, 1, :130].isfinite().all())
    assert bool(dq[0, 2:].isfinite().all())


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("nq, nk", [(1, 300), (40, 2000), (300, 300)])
def test_scores_that_have_no_softmax(gpu, nq, nk, dtype) -> None:
    """A NaN among a query's scores, an infinite one, and all of them -infinity make its row NaN and no other's."""
    q, k, v, _ = _qkv(1, 3, 3, nq, nk, 64, dtype, 7)
    k[0, 0, nk // 2, 0] = math.nan
    k[0, 1, nk // 3, 1], q[0, 1, :, 1] = math.inf, 1.0
    k[0, 2, :, 2], q[0, 2, 0, 2] = -math.inf, 1.0
    q[0, 2, 1:, 2] = -1.0
    o = cross_attention(q, k, v)
    assert bool(o.isnan().all())
    k[0, 2, : nk - 1, 2] = -math.inf
    k[0, 2, nk - 1, 2] = 1.0
    o = cross_attention(q[:, 2:, :1].contiguous(), k[:, 2:], v[:, 2:])
    torch.testing.assert_close(o[0, 0, 0], v[0, 2, nk - 1], atol=0, rtol=2.0**-10)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("nq", [1, 5, 200])
def test_lengths_outside_their_range(gpu, nq, dtype) -> None:
    q, k, v, _ = _qkv(3, 4, 2, nq, 100, 64, dtype, 8)
    got = cross_attention(q, k, v, _int(-1, 101, 2**31 - 1))
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    assert torch.equal(got, cross_attention(q, k, v, _int(0, 100, 100)))
    assert not bool(got[0].any())


@pytest.mark.gpu
@F16_F32
def test_no_keys_no_queries_no_batch(gpu, dtype) -> None:
    for b, h, nq, nk in ((2, 4, 3, 0), (2, 4, 1, 0), (2, 4, 40, 0), (2, 4, 0, 7), (0, 4, 3, 7), (2, 0, 3, 7)):
        q, k, v, do = _qkv(b, h, 2, nq, nk, 64, dtype, 9)
        for lengths in (None, torch.zeros(b, dtype=torch.int32, device="cuda")):
            args = [t.detach().requires_grad_() for t in (q, k, v)]
            o = cross_attention(*args, lengths)
            if nk == 0 or lengths is not None:
                assert not bool(o.any())
            grads = torch.autograd.grad(o, args, do)
            assert all(g.shape == t.shape for g, t in zip(grads, args, strict=True))
            assert nk > 0 and lengths is None and nq > 0 or not any(bool(g.any()) for g in grads)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("nq", [1, 3, 150])
def test_layouts_that_need_a_copy(gpu, nq, dtype) -> None:
    """Odd strides, a base that no 16-byte load reaches, a broadcast batch and a broadcast dO."""
    q, k, v, _ = _qkv(2, 4, 2, nq, 333, 64, dtype, 3)
    held = _int(300, 7)
    odd = torch.empty((2, 4, nq, 65), device="cuda", dtype=dtype)[..., 1:].copy_(q)
    strided = torch.zeros((4, 4), dtype=torch.int32, device="cuda")[::2, 1].copy_(held)
    k1, v1 = k[:1].expand_as(k), v[:1].expand_as(v)
    do = torch.randn((2, 4, 1, 64), device="cuda").to(dtype).expand(2, 4, nq, 64)
    args = [t.detach().clone().requires_grad_() for t in (q, k1, v1)]
    want = cross_attention(*args, held)
    want_g = torch.autograd.grad(want, args, do.contiguous())
    odd.requires_grad_()
    got = cross_attention(odd, k1.requires_grad_(), v1.requires_grad_(), strided)
    assert torch.equal(got, want)
    got_g = torch.autograd.grad(got, (odd, k1, v1), do)
    assert torch.equal(got_g[1], want_g[1]) and torch.equal(got_g[2], want_g[2])
    torch.testing.assert_close(got_g[0], want_g[0], atol=2e-3, rtol=2e-3)  # fp16 dQ sums in varying order


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("nq, nk", [(1, 1), (200, 1), (300, 129), (40, 2000)])
def test_one_key_has_no_gradient_through_its_score(gpu, nq, nk, d, dtype) -> None:
    """Its weight is 1 whatever its score: exact zeros for Q and K."""
    q, k, v, do = _qkv(3, 4, 2, nq, nk, d, dtype, seed=nq)
    lengths = torch.tensor([1, nk, 1], dtype=torch.int32, device="cuda")
    out = cross_attention(q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), lengths)
    out.backward(do)
    for z in (0, 2):
        assert not q.grad[z].any() and not k.grad[z].any()
    assert bool(q.grad[1].any()) == (nk > 1)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_equal_lengths_are_attention(gpu, d) -> None:
    """fp16: the same mathematics in another kernel; both are within the bound of the definition."""
    q, k, v, do = _qkv(1, 4, 4, 500, 500, d, torch.float16, 4)
    want, bounds = cross_attention64(q, k, v, do, None, 1 / math.sqrt(d))
    off = (cross_attention(q, k, v).double() - attention(q, k, v).double()).abs()
    assert bool((off <= 2 * bounds[0]).all())


@pytest.mark.gpu
def test_gradients_against_differences(gpu) -> None:
    """fp32, central differences with e = 4e-3: the third derivative's part is of the order e^2, the rounding of the
    results about 2^-22 / e; both are far below 2e-3 of the gradient's norm."""
    q, k, v, do = _qkv(2, 4, 2, 9, 23, 32, torch.float32, 4)
    held = _int(23, 11)
    args = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*args, held), args, do)
    e = 4e-3
    for i, t in enumerate((q, k, v)):
        direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).cuda()
        values = []
        for sign in (1, -1):
            moved = [x + sign * e * direction if j == i else x for j, x in enumerate((q, k, v))]
            values.append(float((cross_attention(*moved, held).double() * do).sum()))
        want = float((grads[i].double() * direction).sum())
        assert abs((values[0] - values[1]) / (2 * e) - want) <= 2e-3 * max(float(grads[i].norm()), abs(want)), i


@pytest.mark.gpu
@F16_F32
def test_reproducible_on_two_streams_and_once_differentiable(gpu, dtype) -> None:
    inputs = [_qkv(2, 8, 2, 60, 1500, 64, dtype, 20 + i) for i in range(2)]
    held = _int(1500, 800)
    args = [[t.detach().requires_grad_() for t in x[:3]] for x in inputs]

    def both(i):
        o = cross_attention(*args[i], held)
        with torch.no_grad():
            alone = cross_attention(*args[i], held)
        _, dk, dv = torch.autograd.grad(o, args[i], inputs[i][3])
        return o, alone, dk, dv

    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(both(i))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i], strict=True))
    grads = torch.autograd.grad(cross_attention(*args[0], held), args[0], inputs[0][3], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].sum().backward()


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("nq", [1, 3, 70])
def test_captured_with_lengths_that_change(gpu, nq, dtype) -> None:
    """Two graphs of one pool, replayed in turn, forward and backward."""
    q, k, v, do = _qkv(2, 8, 2, nq, 1500, 64, dtype, 30)
    held = _int(1500, 0)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        args = [t.detach().requires_grad_() for t in (q, k, v)]
        torch.autograd.grad(cross_attention(*args, held), args, do)
        pool = None
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool, stream=side):
                o = cross_attention(*args, held)
                _, dk, dv = torch.autograd.grad(o, args, do)
                with torch.no_grad():
                    alone = cross_attention(*args, held)
            pool = graph.pool()
            graphs.append(graph)
            outs.append((o, dk, dv, alone))
    torch.cuda.current_stream().wait_stream(side)
    for lengths in ((7, 1500), (1500, 1), (0, 0)):
        held.copy_(_int(*lengths))
        o = cross_attention(*args, held)
        _, dk, dv = torch.autograd.grad(o, args, do)
        with torch.no_grad():
            want = (o, dk, dv, cross_attention(*args, held))
        for graph, got in zip(graphs, outs, strict=True):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu) -> None:
    """Keys and values of more than 2^32 bytes each, fp16: the last sequence's lie behind that."""
    b, hk, nk, d = 9, 8, 1 << 18, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros((b, hk, nk, d), device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    for t in (k, v):
        t[-1, -1].normal_(generator=g)
    q = torch.randn((b, hk, 20, d), generator=g, device="cuda").half()
    held = torch.full((b,), nk, dtype=torch.int32, device="cuda")
    for rows in (q, q[:, :, :1].contiguous()):
        o = cross_attention(rows, k, v, held)
        assert not bool(o[:, :-1].any()) and not bool(o[:-1].any())
        want, bounds = cross_attention64(*(t[-1:, -1:] for t in (rows, k, v, rows)), None, d**-0.5)
        assert_within(o[-1:, -1:], want[0], bounds[0], "o")
