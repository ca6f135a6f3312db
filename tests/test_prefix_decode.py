"""``tattn.prefix_decode_attention``: refusals without a GPU; results on a B200 against the definition in 64 bits and
against ``tattn.decode_attention`` over the joined cache."""

from __future__ import annotations

import math

import pytest
import torch

import tattn
from tattn import _lib, decode_attention, prefix_decode_attention
from tests.built import ensure_built
from tests.plain64 import assert_within, cross_attention64

ensure_built()

F16_F32 = pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])


def _inputs(prompts, samples, h, hk, prefix, cap, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def make(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    b = prompts * samples
    return (make(b, h, 1, d), make(prompts, hk, prefix, d), make(prompts, hk, prefix, d), make(b, hk, cap, d), make(b, hk, cap, d))


def _int(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _joined(pk, k, prefix_lengths, lengths):
    """Each sequence's keys in one tensor, its prompt's first, and their number."""
    prompts, hk, prefix, d = pk.shape
    b, cap = k.shape[0], k.shape[2]
    out = torch.zeros((b, hk, prefix + cap, d), device="cuda", dtype=k.dtype)
    held = []
    for i in range(b):
        p = i * prompts // b
        n, m = prefix_lengths[p], lengths[i]
        out[i, :, :n], out[i, :, n : n + m] = pk[p, :, :n], k[i, :, :m]
        held.append(n + m)
    return out, held


def _check(prompts, samples, h, hk, prefix, cap, d, dtype, prefix_lengths=None, lengths=None, scale=None, seed=0):
    q, pk, pv, k, v = _inputs(prompts, samples, h, hk, prefix, cap, d, dtype, seed)
    lengths = [cap - (7 * i) % (cap + 1) for i in range(prompts * samples)] if lengths is None else lengths
    given = None if prefix_lengths is None else _int(prefix_lengths)
    got = prefix_decode_attention(q, pk, pv, k, v, _int(lengths), given, scale)
    assert got.dtype == dtype and got.shape == q.shape
    prefix_lengths = [prefix] * prompts if prefix_lengths is None else prefix_lengths
    (jk, held), (jv, _) = _joined(pk, k, prefix_lengths, lengths), _joined(pv, v, prefix_lengths, lengths)
    want, bounds = cross_attention64(q, jk, jv, q, _int(held), 1 / math.sqrt(d) if scale is None else scale)
    assert_within(got, want[0], bounds[0], "o")
    return got, (q, jk, jv, _int(held))


# ------------------------------------------------------------------------------------ without a GPU
def _good(**other):
    a = dict(
        q=torch.zeros(6, 4, 1, 16), prefix_k=torch.zeros(2, 2, 9, 16), prefix_v=torch.zeros(2, 2, 9, 16),
        k=torch.zeros(6, 2, 5, 16), v=torch.zeros(6, 2, 5, 16), lengths=torch.zeros(6, dtype=torch.int32),
        prefix_lengths=torch.zeros(2, dtype=torch.int32),
    )  # fmt: skip
    return a | other


@pytest.mark.parametrize(
    "other, message",
    [
        (dict(q=torch.zeros(6, 4, 16)), "expected q"),
        (dict(q=torch.zeros(6, 4, 2, 16)), "one token"),
        (dict(v=torch.zeros(6, 2, 6, 16)), "expected q"),
        (dict(k=torch.zeros(5, 2, 5, 16), v=torch.zeros(5, 2, 5, 16)), "agree in batch"),
        (dict(k=torch.zeros(6, 3, 5, 16), v=torch.zeros(6, 3, 5, 16)), "multiple of key/value heads"),
        (dict(prefix_k=torch.zeros(2, 2, 9), prefix_v=torch.zeros(2, 2, 9)), "expected prefix_k"),
        (dict(prefix_v=torch.zeros(2, 2, 8, 16)), "expected prefix_k"),
        (dict(prefix_k=torch.zeros(2, 4, 9, 16), prefix_v=torch.zeros(2, 4, 9, 16)), "expected prefix_k"),
        (dict(prefix_k=torch.zeros(2, 2, 9, 32), prefix_v=torch.zeros(2, 2, 9, 32)), "expected prefix_k"),
        (dict(prefix_k=torch.zeros(2, 2, 9, 16).half()), "prefix must have q's dtype"),
        (dict(prefix_k=torch.zeros(4, 2, 9, 16), prefix_v=torch.zeros(4, 2, 9, 16)), "multiple of the prompts"),
        (dict(prefix_k=torch.zeros(0, 2, 9, 16), prefix_v=torch.zeros(0, 2, 9, 16)), "multiple of the prompts"),
        (dict(lengths=torch.zeros(6)), "lengths must be int32"),
        (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths must be int32"),
        (dict(prefix_lengths=torch.zeros(6, dtype=torch.int32)), "prefix_lengths must be int32"),
        (dict(prefix_lengths=torch.zeros(2)), "prefix_lengths must be int32"),
    ],
)
def test_refusals(other, message) -> None:
    with pytest.raises(ValueError, match=message):
        prefix_decode_attention(**_good(**other))


def test_no_cpu_path_and_no_gradients() -> None:
    with pytest.raises(RuntimeError, match="no CPU path"):
        prefix_decode_attention(**_good())
    for name in ("q", "prefix_k", "prefix_v", "k", "v"):
        args = _good()
        args[name] = args[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            prefix_decode_attention(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            prefix_decode_attention(**args)
    assert "prefix_decode_attention" in tattn.__all__


@pytest.mark.parametrize("name", ["q", "prefix_k", "prefix_v", "k", "v"])
def test_forward_mode_derivatives_are_refused(name) -> None:
    with torch.autograd.forward_ad.dual_level():
        args = _good()
        args[name] = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            prefix_decode_attention(**args)


def test_abi_refuses_before_any_device_call() -> None:
    lib = _lib.load()
    s = _lib.strides_array(*[(8 * 16, 8 * 16, 16, 1)] * 6)
    dims = dict(prompts=2, samples=3, h=2, hk=2, p=8, c=8, d=16, dtype=0)
    for bad in (dict(d=24), dict(hk=0), dict(h=3), dict(h=0), dict(p=-1), dict(c=-1), dict(dtype=2), dict(prompts=-1), dict(samples=0)):
        a = (dims | bad).values()
        assert lib.tattn_prefix_decode(*[16] * 9, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_prefix_decode_workspace_bytes(*a) == -1
    assert lib.tattn_prefix_decode(*[16] * 9, s, *(dims | dict(prompts=1 << 15, samples=1 << 15)).values(), 0.1, None) == _lib.ERR_TOO_LARGE
    assert lib.tattn_prefix_decode(*[None] * 9, s, *(dims | dict(prompts=0)).values(), 0.1, None) == 0
    assert lib.tattn_prefix_decode(17, *[16] * 8, s, *dims.values(), 0.1, None) == _lib.ERR_LAYOUT
    assert lib.tattn_prefix_decode(*[16] * 8, None, s, *dims.values(), 0.1, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.tattn_prefix_decode_workspace_bytes(*dims.values()) >= 2 * 3 * 2 * 2 * (16 + 2) * 4


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


SHAPES = [
    # prompts, samples, h, hk, prefix, cap, prefix lengths, lengths
    (1, 1, 1, 1, 1, 1, None, [1]),
    (1, 4, 4, 2, 70, 33, None, [33, 1, 0, 17]),
    (2, 3, 6, 2, 129, 40, [129, 0], [40, 0, 7, 0, 1, 40]),  # a sequence with nothing at all
    (3, 5, 5, 5, 300, 9, [1, 128, 257], None),
    (1, 64, 8, 2, 1000, 20, [999], None),
    (1, 33, 5, 1, 515, 300, [300], None),  # 165 rows: two tiles, the second partly filled
    (2, 70, 4, 4, 65, 2, [64, 65], None),
    (1, 2, 16, 1, 4000, 1500, [3999], [1500, 3]),
    (4, 1, 4, 2, 200, 100, [0, 1, 199, 200], [0, 100, 50, 1]),
]


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(gpu, shape, d, dtype) -> None:
    prompts, samples, h, hk, prefix, cap, prefix_lengths, lengths = shape
    _check(prompts, samples, h, hk, prefix, cap, d, dtype, prefix_lengths, lengths)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(gpu, scale, dtype) -> None:
    _check(2, 5, 8, 2, 300, 40, 64, dtype, [300, 77], scale=scale)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [64, 128])
def test_long_ones_are_decode_attention_over_the_joined_cache(gpu, d, dtype) -> None:
    """Both are within the bound of the definition, which _check holds this one to."""
    got, joined = _check(1, 16, 8, 2, 9000, 3000, d, dtype, [8999])
    want, bounds = cross_attention64(joined[0], joined[1], joined[2], joined[0], joined[3], d**-0.5)
    assert bool(((got.double() - decode_attention(*joined).double()).abs() <= 2 * bounds[0]).all())


@pytest.mark.gpu
@F16_F32
def test_without_a_prefix_or_own_tokens(gpu, dtype) -> None:
    _check(2, 3, 4, 2, 0, 40, 64, dtype)
    _check(2, 3, 4, 2, 40, 0, 64, dtype)
    _check(2, 3, 3, 1, 0, 40, 64, dtype)
    _check(1, 3, 3, 1, 40, 0, 64, dtype)
    q, pk, pv, k, v = _inputs(2, 3, 4, 2, 0, 0, 64, dtype)
    assert not bool(prefix_decode_attention(q, pk, pv, k, v, _int([0] * 6)).any())
    q, pk, pv, k, v = (t[:0] for t in _inputs(2, 3, 4, 2, 7, 5, 64, dtype))
    assert prefix_decode_attention(q, pk, pv, k, v, _int([])).shape == (0, 4, 1, 64)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_lies_past_a_length_is_never_used(gpu, value, dtype) -> None:
    q, pk, pv, k, v = _inputs(2, 5, 8, 2, 300, 50, 64, dtype)
    n, m = [301 - 100, 0], [50 - 5 * i for i in range(10)]
    results = []
    for fill in (0.0, value):
        for p in range(2):
            pk[p, :, n[p] :], pv[p, :, n[p] :] = fill, fill
        for b in range(10):
            k[b, :, m[b] :], v[b, :, m[b] :] = fill, fill
        results.append(prefix_decode_attention(q, pk, pv, k, v, _int(m), _int(n)))
    assert torch.equal(*results) and bool(results[0].isfinite().all())


@pytest.mark.gpu
@F16_F32
def test_scores_that_have_no_softmax(gpu, dtype) -> None:
    """A NaN or an infinite score in the prefix makes the rows that share its head NaN, one among a sequence's own tokens
    that sequence's; scores of -infinity weigh nothing beside others, and alone leave no result."""
    q, pk, pv, k, v = _inputs(1, 3, 4, 2, 300, 50, 64, dtype)
    q[:, :, 0, 0] = 1.0
    pk[0, 0, 200, 0] = math.nan
    k[1, 1, 7, 0] = math.inf
    o = prefix_decode_attention(q, pk, pv, k, v, _int([50, 50, 50]))
    assert bool(o[:, :2].isnan().all()) and bool(o[1, 2:].isnan().all())
    assert bool(o[0, 2:].isfinite().all()) and bool(o[2, 2:].isfinite().all())
    pk[0, 0, 200, 0] = 0.0
    k[1, 1, 7, 0] = 0.0
    pk[..., 0] = -math.inf  # the whole prefix
    o = prefix_decode_attention(q, pk, pv, k, v, _int([50, 1, 0]))
    want = decode_attention(q, k, v, _int([50, 1, 0]))
    torch.testing.assert_close(o[:2], want[:2], atol=1e-2, rtol=0)  # each within 1e-3 of weighted values of up to 5
    assert bool(o[2].isnan().all())


@pytest.mark.gpu
@F16_F32
def test_lengths_outside_their_range(gpu, dtype) -> None:
    q, pk, pv, k, v = _inputs(2, 2, 4, 2, 100, 30, 64, dtype)
    got = prefix_decode_attention(q, pk, pv, k, v, _int([31, -1, 5, 6]), _int([-7, 101]))
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    assert torch.equal(got, prefix_decode_attention(q, pk, pv, k, v, _int([30, 0, 5, 6]), _int([0, 100])))


@pytest.mark.gpu
@F16_F32
def test_caches_in_place_and_refused_layouts(gpu, dtype) -> None:
    """Slices of larger caches are read in place; rows that 16-byte loads do not reach are refused; q may lie anyhow."""
    q, pk, pv, k, v = _inputs(2, 3, 4, 2, 100, 30, 64, dtype)
    lengths = _int(range(24, 30))
    want = prefix_decode_attention(q, pk, pv, k, v, lengths)

    def wider(t):
        big = torch.full((t.shape[0], t.shape[2] + 9, t.shape[1], 64), math.nan, device="cuda", dtype=dtype).transpose(1, 2)
        big[:, :, : t.shape[2]] = t
        return big[:, :, : t.shape[2]]

    odd = torch.empty((6, 4, 1, 65), device="cuda", dtype=dtype)[..., 1:].copy_(q)
    assert torch.equal(prefix_decode_attention(odd, *(wider(t) for t in (pk, pv, k, v)), lengths), want)
    for i in range(4):
        args = [pk, pv, k, v]
        args[i] = torch.empty((*args[i].shape[:3], 65), device="cuda", dtype=dtype)[..., 1:].copy_(args[i])
        with pytest.raises(ValueError, match="in place"):
            prefix_decode_attention(q, *args, lengths)


@pytest.mark.gpu
@F16_F32
def test_captured_steps_with_lengths_that_change_and_two_streams(gpu, dtype) -> None:
    q, pk, pv, k, v = _inputs(2, 8, 8, 2, 3000, 500, 64, dtype)
    lengths, prefix_lengths = _int([1] * 16), _int([3000, 100])
    call = (q, pk, pv, k, v, lengths, prefix_lengths)
    prefix_decode_attention(*call)
    graphs, outs, pool = [], [], None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(prefix_decode_attention(*call))
        pool = graph.pool()
        graphs.append(graph)
    for step in range(3):
        lengths.add_(150)
        prefix_lengths.sub_(30)
        want = prefix_decode_attention(*call)
        for graph, out in zip(graphs, outs, strict=True):
            graph.replay()
            assert torch.equal(out, want)
    sides, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for side in sides:
            with torch.cuda.stream(side):
                got.append(prefix_decode_attention(*call))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("dim", [0, 1])
def test_an_expanded_prefix(gpu, dim, dtype) -> None:
    """Over prompts or heads: fp32 reads it in place; fp16 refuses it, and says why (its own tokens may be expanded)."""
    q, pk, pv, k, v = _inputs(2, 3, 4, 2, 100, 30, 64, dtype)
    pk, pv, k, v = (t.narrow(dim, 0, 1).expand_as(t) for t in (pk, pv, k, v))
    lengths = _int([30, 1, 0, 7, 30, 5])
    want = prefix_decode_attention(q, *(t.contiguous() for t in (pk, pv, k, v)), lengths)
    assert torch.equal(prefix_decode_attention(q, pk.contiguous(), pv.contiguous(), k, v, lengths), want)
    if dtype == torch.float32:
        assert torch.equal(prefix_decode_attention(q, pk, pv, k, v, lengths), want)
        return
    for args in ((pk, pv.contiguous()), (pk.contiguous(), pv)):
        with pytest.raises(ValueError, match="a prefix in float16 cannot be expanded"):
            prefix_decode_attention(q, *args, k, v, lengths)
