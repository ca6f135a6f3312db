"""Infinities among the values that queries see (``tattn.cross_attention``, ``tattn.prefix_decode_attention``): an infinity
times a weight above 0 is an infinity, whichever kernel the number of rows selects, and reaches nothing else.

Scores are of the order of 1, so no weight falls to 2^-24 of the largest, where one rounds to 0 in 16 bits."""

from __future__ import annotations

import math

import pytest
import torch

from tattn import _lib, cross_attention, prefix_decode_attention
from tests.built import ensure_built
from tests.plain64 import assert_within, cross_attention64

ensure_built()

F16_F32 = pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


def _rows(*shape, dtype, seed):
    """Values in (-1, 1), of variance 1/3: scores have a standard deviation of 1/3 at the default scale."""
    return (torch.rand(shape, generator=torch.Generator().manual_seed(seed)) * 2 - 1).to(dtype).cuda()


def _same(got, want, bound, name) -> None:
    """The definition's infinities and NaN where it has them, within the bound elsewhere."""
    finite = want.isfinite()
    assert bool(finite.any())
    rest = got[~finite].double()
    assert torch.equal(rest.nan_to_num(7.0, 8.0, 9.0), want[~finite].nan_to_num(7.0, 8.0, 9.0)), f"{name}: {rest[:8]} for {want[~finite][:8]}"
    assert_within(got[finite], want[finite], bound[finite], name)


def _plant(v, first, last) -> None:
    """Into the second head of the first sequence: an infinity of either sign at a key of its own, and both in one dim."""
    v[0, 1, first, 2] = math.inf
    v[0, 1, last, 3] = -math.inf
    v[0, 1, first, 5], v[0, 1, last, 5] = math.inf, -math.inf


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("nk, held", [(300, 289), (3000, 2900)])
@pytest.mark.parametrize("nq", [1, 2, 9, 16, 17, 20, 32, 33, 65, 129])
def test_cross_attention(gpu, nq, nk, held, d, dtype) -> None:
    """2 nq rows share a key/value head: up to 64 of them stand in an fp16 tile several times, and up to 16 without
    gradients take the single-token kernel."""
    q, do = _rows(2, 4, nq, d, dtype=dtype, seed=1), _rows(2, 4, nq, d, dtype=dtype, seed=2)
    k, v = _rows(2, 2, nk, d, dtype=dtype, seed=3), _rows(2, 2, nk, d, dtype=dtype, seed=4)
    _plant(v, 70, held - 1)
    lengths = torch.tensor([held, nk], dtype=torch.int32, device="cuda")
    want, bounds = cross_attention64(q, k, v, do, lengths, d**-0.5)
    with torch.no_grad():
        _same(cross_attention(q, k, v, lengths), want[0], bounds[0], "o alone")
    args = [t.detach().requires_grad_() for t in (q, k, v)]
    _same(cross_attention(*args, lengths), want[0], bounds[0], "o")


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("where", ["v", "do"])
@pytest.mark.parametrize("nq, nk, held", [(1, 300, 289), (20, 3000, 2900), (33, 300, 289), (129, 300, 289), (300, 1300, 1200)])
def test_cross_attention_gradients(gpu, nq, nk, held, where, d, dtype) -> None:
    """dV does not read V, and a dim of it reads that dim of dO alone; the other heads and sequences have finite gradients
    throughout."""
    q, do = _rows(2, 4, nq, d, dtype=dtype, seed=1), _rows(2, 4, nq, d, dtype=dtype, seed=2)
    k, v = _rows(2, 2, nk, d, dtype=dtype, seed=3), _rows(2, 2, nk, d, dtype=dtype, seed=4)
    if where == "v":
        _plant(v, 70, held - 1)
    else:  # (of a query head of the second key/value head)
        do[0, 3, nq // 2, 2], do[0, 3, nq // 2, 3] = math.inf, -math.inf
    lengths = torch.tensor([held, nk], dtype=torch.int32, device="cuda")
    want, bounds = cross_attention64(q, k, v, do, lengths, d**-0.5)
    args = [t.detach().requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(cross_attention(*args, lengths), args, do)
    seen = torch.arange(nk, device="cuda") < lengths[:, None]
    want_dv = torch.where(seen[:, None, :, None], want[3], torch.zeros_like(want[3]))  # (0 x infinity in the definition's sum)
    _same(dv, want_dv, bounds[3], "dv")
    for got, i, heads in ((dq, 1, 2), (dk, 2, 1)):
        assert_within(got[0, :heads], want[i][0, :heads], bounds[i][0, :heads], "dq, dk of the other heads")
        assert_within(got[1], want[i][1], bounds[i][1], "dq, dk of the other sequence")


@pytest.mark.gpu
@F16_F32
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("samples", [1, 3, 16, 20, 32, 33, 70])
def test_prefix_decode_attention(gpu, samples, where, d, dtype) -> None:
    """2 x samples rows share a prompt's head."""
    prefix, cap = 900, 40
    q = _rows(samples, 4, 1, d, dtype=dtype, seed=1)
    pk, pv = _rows(1, 2, prefix, d, dtype=dtype, seed=2), _rows(1, 2, prefix, d, dtype=dtype, seed=3)
    k, v = _rows(samples, 2, cap, d, dtype=dtype, seed=4), _rows(samples, 2, cap, d, dtype=dtype, seed=5)
    _plant(*((pv, 70, prefix - 1) if where == "prefix" else (v, 7, cap - 1)))
    got = prefix_decode_attention(q, pk, pv, k, v, torch.full((samples,), cap, dtype=torch.int32, device="cuda"))
    jk, jv = (torch.cat([p.expand(samples, -1, -1, -1), t], 2) for p, t in ((pk, k), (pv, v)))
    want, bounds = cross_attention64(q, jk, jv, q, None, d**-0.5)
    _same(got, want[0], bounds[0], "o")
