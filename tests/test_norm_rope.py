"""``tattn.qk_norm_rope``: refusals without a GPU; results and gradients on a B200 against the definition in 64
bits and against differences."""

from __future__ import annotations

import pytest
import torch

import tattn
from tattn import _lib, qk_norm_rope
from tests.built import ensure_built
from tests.plain64 import assert_within

ensure_built()

EPS = 1e-6


def _tables(positions, d, device="cuda"):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2).double() / d)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _inputs(b, h, hk, n, d, dtype, seed=0, layout="bhnd", w_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)

    def heads(k):
        if layout == "bnhd":
            return torch.randn((b, n, k, d), generator=g).to(dtype).cuda().transpose(1, 2)
        if layout == "packed":  # a slice of a wider projection
            return torch.randn((b, n, k, 2 * d), generator=g).to(dtype).cuda()[..., d:].transpose(1, 2)
        return torch.randn((b, k, n, d), generator=g).to(dtype).cuda()

    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(w_dtype).cuda() for _ in range(2)]
    return heads(h), heads(hk), *w, heads(h), heads(hk)


def _definition(x, w, dy, cos, sin, interleaved, dtype):
    """(y, dx, dw) in 64 bits and bounds: the result's rounding, and for everything in 32 bits c of the summed
    magnitudes (c covers a sum of 128 squares, its root and a handful of products)."""
    u = 2.0**-11 if dtype == torch.float16 else 2.0**-24
    c = 2e-5
    x, w, dy = x.double(), w.double(), dy.double()
    d = x.shape[-1]
    first = torch.arange(0, d, 2) if interleaved else torch.arange(d // 2)
    second = first + 1 if interleaved else first + d // 2
    co, si = cos.double()[:, None], sin.double()[:, None]
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()

    def turn(a, sign, mags=False):
        out = torch.empty_like(a)
        a1, a2 = a[..., first], a[..., second]
        if mags:
            out[..., first], out[..., second] = a1 * co.abs() + a2 * si.abs(), a2 * co.abs() + a1 * si.abs()
        else:
            out[..., first], out[..., second] = a1 * co - sign * a2 * si, a2 * co + sign * a1 * si
        return out

    y = turn(x * r * w, 1)
    e_y = c * turn((x * r * w).abs(), 1, True)
    g = turn(dy, -1)
    gm = turn(dy.abs(), 1, True)
    hm = gm * w.abs()
    dx = r * (g * w - x * r * (g * w * x * r).mean(-1, keepdim=True))
    e_dx = c * r * (hm + (x * r).abs() * (hm * (x * r).abs()).mean(-1, keepdim=True))
    dw = (g * x * r).sum((0, 1, 2))
    rows = x.numel() // d
    e_dw = (c + rows * 2.0**-24) * (gm * (x * r).abs()).sum((0, 1, 2))
    return (y, 2 * u * y.abs() + e_y + 2.0**-24), (dx, 2 * u * dx.abs() + e_dx + 2.0**-24), (dw, e_dw)


def _check(b, h, hk, n, d, dtype, interleaved=False, layout="bhnd", w_dtype=torch.float32, positions=None, P=512):
    q, k, wq, wk, dyq, dyk = _inputs(b, h, hk, n, d, dtype, n + d, layout, w_dtype)
    cos, sin = _tables(P, d)
    at = torch.arange(n, device="cuda").expand(b, n) if positions is None else positions.long().expand(b, n)
    args = [t.requires_grad_() for t in (q, k, wq, wk)]
    outs = qk_norm_rope(*args, cos, sin, positions, EPS, interleaved)
    grads = torch.autograd.grad(outs, args, (dyq, dyk))
    for x, w, dy, y, dx, dw, name in (
        (q, wq, dyq, outs[0], grads[0], grads[2], "q"),
        (k, wk, dyk, outs[1], grads[1], grads[3], "k"),
    ):
        want = _definition(x.detach(), w.detach(), dy, cos[at], sin[at], interleaved, dtype)
        assert y.dtype == dx.dtype == dtype and dw.dtype == w_dtype
        assert_within(y, *want[0], name)
        assert_within(dx, *want[1], "d" + name)
        e = want[2][1] + (want[2][0].abs() * 2.0**-10 if w_dtype == torch.float16 else 0)
        assert_within(dw, want[2][0], e, "dw" + name)


# ------------------------------------------------------------------------------------ without a GPU
def _good(**other):
    a = dict(
        q=torch.zeros(2, 4, 8, 16), k=torch.zeros(2, 2, 8, 16), q_weight=torch.zeros(16), k_weight=torch.zeros(16),
        cos=torch.zeros(8, 8), sin=torch.zeros(8, 8), positions=None,
    )  # fmt: skip
    return a | other


@pytest.mark.parametrize(
    "other, message",
    [
        (dict(q=torch.zeros(2, 4, 16)), "expected q"),
        (dict(k=torch.zeros(2, 2, 7, 16)), "expected q"),
        (dict(k=torch.zeros(1, 2, 8, 16)), "expected q"),
        (dict(k=torch.zeros(2, 0, 8, 16)), "at least one head"),
        (dict(q=torch.zeros(2, 4, 8, 24), k=torch.zeros(2, 2, 8, 24)), "head dim"),
        (dict(k=torch.zeros(2, 2, 8, 16).half()), "dtype"),
        (dict(q=torch.zeros(2, 4, 8, 16).bfloat16(), k=torch.zeros(2, 2, 8, 16).bfloat16()), "dtype"),
        (dict(q_weight=torch.zeros(8)), "weights must have shape"),
        (dict(q_weight=torch.zeros(16).half()), "weights must share"),
        (dict(cos=torch.zeros(8, 16)), "cos and sin must have shape"),
        (dict(sin=torch.zeros(9, 8)), "cos and sin must have shape"),
        (dict(cos=torch.zeros(8, 8).double(), sin=torch.zeros(8, 8).double()), "float32"),
        (dict(cos=torch.zeros(7, 8), sin=torch.zeros(7, 8)), "fewer than"),
        (dict(positions=torch.zeros(2, 8)), "positions must be int32"),
        (dict(positions=torch.zeros(2, 7, dtype=torch.int32)), "positions must be int32"),
    ],
)
def test_refusals(other, message) -> None:
    with pytest.raises(ValueError, match=message):
        qk_norm_rope(**_good(**other))


def test_no_cpu_path() -> None:
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_norm_rope(**_good())
    assert "qk_norm_rope" in tattn.__all__


def test_abi_refuses_before_any_device_call() -> None:
    lib = _lib.load()
    s = _lib.strides_array(*[(512, 128, 16, 1)] * 6, (8, 1))
    dims = dict(z=1, h=2, hk=2, n=8, d=16, p=8, dtype=0, w=1)

    def forward(**o):
        return lib.tattn_qk_norm_rope(*[16] * 9, s, *(dims | o).values(), 1e-6, 0, None)

    def backward(**o):
        return lib.tattn_qk_norm_rope_bwd(*[16] * 14, s, *(dims | o).values(), 1e-6, 0, None)

    for bad in (dict(d=24), dict(h=0), dict(hk=0), dict(z=-1), dict(dtype=2), dict(dtype=1, w=0), dict(p=-1), dict(p=0)):
        assert forward(**bad) == backward(**bad) == _lib.ERR_INVALID_ARGUMENT
    assert forward(z=1 << 20, n=1 << 10) == backward(z=1 << 20, n=1 << 10) == _lib.ERR_TOO_LARGE
    assert forward(z=0) == 0
    assert lib.tattn_qk_norm_rope(17, *[16] * 8, s, *dims.values(), 1e-6, 0, None) == _lib.ERR_LAYOUT
    assert lib.tattn_qk_norm_rope_bwd_workspace_bytes(24) == -1


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["split", "interleaved"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("b, h, hk, n", [(1, 1, 1, 1), (3, 5, 1, 17), (2, 6, 2, 70)])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "packed"])
def test_against_the_definition(gpu, b, h, hk, n, d, interleaved, dtype, layout) -> None:
    _check(b, h, hk, n, d, dtype, interleaved, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_many_rows(gpu, d, dtype) -> None:
    """Enough rows for several heads an item and several items a thread, in head counts that 4 does not divide."""
    _check(3, 13, 3, 2500, d, dtype, layout="bnhd", P=2500)
    _check(2, 5, 5, 4001, d, dtype, True, P=4001)


@pytest.mark.gpu
def test_weights_of_the_tensors_type(gpu) -> None:
    _check(2, 6, 2, 70, 64, torch.float16, w_dtype=torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["each", "shared", "strided"])
def test_positions(gpu, shape) -> None:
    g = torch.Generator().manual_seed(2)
    if shape == "each":
        at = torch.randint(0, 512, (3, 40), generator=g, dtype=torch.int32).cuda()
    elif shape == "shared":
        at = torch.randint(0, 512, (40,), generator=g, dtype=torch.int32).cuda()
    else:
        at = torch.randint(0, 512, (40, 6), generator=g, dtype=torch.int32).cuda().t()[::2]
    _check(3, 4, 2, 40, 64, torch.float16, positions=at)


@pytest.mark.gpu
def test_a_position_outside_the_tables(gpu) -> None:
    """Its rows are NaN, all others as without it, and the status word says so."""
    q, k, wq, wk, *_ = _inputs(1, 2, 1, 6, 64, torch.float16)
    cos, sin = _tables(100, 64)
    at = torch.tensor([5, 99, 100, -1, 0, 7], dtype=torch.int32, device="cuda")
    out = qk_norm_rope(q, k, wq, wk, cos, sin, at)
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    want = qk_norm_rope(q, k, wq, wk, cos, sin, at.clamp(0, 99))
    outside = [2, 3]
    inside = [0, 1, 4, 5]
    for o, w in zip(out, want, strict=True):
        assert bool(o[:, :, outside].isnan().all())
        assert torch.equal(o[:, :, inside], w[:, :, inside])


@pytest.mark.gpu
def test_layouts_that_need_a_copy(gpu) -> None:
    q, k, wq, wk, dyq, dyk = _inputs(2, 4, 2, 30, 64, torch.float16)
    cos, sin = _tables(64, 64)
    want = qk_norm_rope(q, k, wq, wk, cos, sin)
    odd = torch.empty((2, 4, 30, 65), device="cuda", dtype=torch.float16)[..., 1:].copy_(q)
    wide = torch.cat((cos, sin), 1)
    shifted = torch.empty(65, device="cuda")[1:].copy_(wq)
    got = qk_norm_rope(odd, k, shifted, wk, wide[:, :32], wide[:, 32:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # A gradient that is one row for all, and a permuted one.
    args = [t.clone().requires_grad_() for t in (q, k)]
    outs = qk_norm_rope(*args, wq, wk, cos, sin)
    one = dyq[:, :, :1].expand_as(dyq)
    turned = dyk.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    a = torch.autograd.grad(outs, args, (one, turned), retain_graph=True)
    b = torch.autograd.grad(outs, args, (one.contiguous(), turned.contiguous()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, size", [(torch.float16, 2e4), (torch.float32, 1e15), (torch.float32, 1e-12)])
def test_extreme_rows(gpu, dtype, size) -> None:
    """Rows whose squares are far from 1 (fp16: whose squares overflow 16 bits), and rows of zeros."""
    q, k, wq, wk, dyq, dyk = _inputs(1, 2, 2, 9, 64, dtype)
    q = (q * size).clamp(-6e4, 6e4) if dtype == torch.float16 else q * size
    k = torch.zeros_like(k)
    cos, sin = _tables(9, 64)
    out = qk_norm_rope(q, k, wq, wk, cos, sin)
    at = torch.arange(9).expand(1, 9)
    want = _definition(q, wq, dyq, cos[at], sin[at], False, dtype)[0]
    assert_within(out[0], *want, "q")
    assert not bool(out[1].any())


@pytest.mark.gpu
def test_gradients_against_differences(gpu) -> None:
    """fp32, central differences with e = 2e-3: the third derivative's part is of the order e^2, the rounding of
    the results about 2^-24 / e; both are far below 1e-3 of the gradient's norm."""
    q, k, wq, wk, dyq, dyk = _inputs(2, 3, 1, 11, 32, torch.float32, 4)
    cos, sin = _tables(11, 32)
    args = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(qk_norm_rope(*args, cos, sin), args, (dyq, dyk))
    e = 2e-3
    for i, t in enumerate((q, k, wq, wk)):
        direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).cuda()
        values = []
        for sign in (1, -1):
            moved = [x + sign * e * direction if j == i else x for j, x in enumerate((q, k, wq, wk))]
            yq, yk = qk_norm_rope(*moved, cos, sin)
            values.append(float((yq.double() * dyq).sum() + (yk.double() * dyk).sum()))
        want = float((grads[i].double() * direction).sum())
        assert abs((values[0] - values[1]) / (2 * e) - want) <= 1e-3 * max(float(grads[i].norm()), abs(want)), i


@pytest.mark.gpu
def test_reproducible_empty_and_streams(gpu) -> None:
    q, k, wq, wk, dyq, dyk = _inputs(4, 16, 4, 1000, 64, torch.float16)
    cos, sin = _tables(1000, 64)
    args = [t.requires_grad_() for t in (q, k, wq, wk)]
    outs = qk_norm_rope(*args, cos, sin)
    first = torch.autograd.grad(outs, args, (dyq, dyk), retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(outs, args, (dyq, dyk))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again, strict=True))
    none = [t.detach()[:, :, :0].requires_grad_() for t in (q, k)]
    outs = qk_norm_rope(*none, *args[2:], cos, sin)
    grads = torch.autograd.grad(outs, (*none, *args[2:]), outs)
    assert outs[0].shape == none[0].shape and not bool(grads[2].any()) and not bool(grads[3].any())


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_derivatives_are_refused(which) -> None:
    """For each tensor that could carry a tangent. (Without a GPU: before the device check.)"""
    with torch.autograd.forward_ad.dual_level():
        args = [torch.zeros(1, 2, 8, 16), torch.zeros(1, 1, 8, 16), *[torch.ones(16)] * 2, *[torch.ones(8, 8)] * 2]
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for take in (torch.enable_grad, torch.no_grad):
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                qk_norm_rope(*args)


@pytest.mark.parametrize("which", [4, 5])
def test_tables_that_need_gradients_are_refused(which) -> None:
    """Gradients reach q, k and the weights; a table would get none. (Without a GPU: before the device check.)"""
    args = [torch.zeros(1, 2, 8, 16), torch.zeros(1, 1, 8, 16), *[torch.ones(16)] * 2, *[torch.ones(8, 8)] * 2]
    args[which] = args[which].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        qk_norm_rope(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        qk_norm_rope(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_forward_and_backward_on_side_streams(gpu, dtype) -> None:
    """Two streams work on different inputs at the same time, forward and backward: each gets what its inputs give alone
    (the results are bitwise reproducible)."""
    cos, sin = _tables(1000, 64)
    inputs = [_inputs(2, 16, 4, 1000, 64, dtype, 50 + i) for i in range(2)]
    args = [[t.clone().requires_grad_() for t in x[:4]] for x in inputs]

    def both(i):
        outs = qk_norm_rope(*args[i], cos, sin)
        return (*outs, *torch.autograd.grad(outs, args[i], inputs[i][4:]))

    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(both(i))
    for side in sides:
        side.synchronize()
    for results, first in zip(got, want, strict=True):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, first, strict=True))
