"""``tattn.qk_rope_axes``: refusals without a GPU; results and gradients on a B200 against the definition in 64 bits,
against differences, and against ``tattn.qk_norm_rope`` where both apply."""

from __future__ import annotations

import pytest
import torch

import tattn
from tattn import _lib, qk_norm_rope, qk_rope_axes
from tests.built import ensure_built
from tests.plain64 import assert_within
from tests.test_norm_rope import EPS, _definition, _inputs, _tables

ensure_built()


def _pair_axes(d, count, mixed):
    return [j % count if mixed else j * count // (d // 2) for j in range(d // 2)]


def _positions(count, b, n, P, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, P, (count, b, n), generator=g, dtype=torch.int32).cuda()


def _rotation(x, dy, cos, sin, interleaved, dtype):
    """(y, dx) of the rotation alone in 64 bits, and bounds: two products and a sum in 32 bits, and the rounding."""
    u = 2.0**-11 if dtype == torch.float16 else 2.0**-24
    d = x.shape[-1]
    first = torch.arange(0, d, 2) if interleaved else torch.arange(d // 2)
    second = first + 1 if interleaved else first + d // 2
    co, si = cos.double()[:, None], sin.double()[:, None]
    out = []
    for a, sign in ((x.double(), 1), (dy.double(), -1)):
        y, m = torch.empty_like(a), torch.empty_like(a)
        y[..., first] = a[..., first] * co - sign * a[..., second] * si
        y[..., second] = a[..., second] * co + sign * a[..., first] * si
        m[..., first] = (a[..., first] * co).abs() + (a[..., second] * si).abs()
        m[..., second] = (a[..., second] * co).abs() + (a[..., first] * si).abs()
        out.append((y, u * y.abs() + 3 * 2.0**-24 * m + 2.0**-24))
    return out


def _check(b, h, hk, n, d, dtype, count=3, mixed=False, norm=True, interleaved=False, layout="bhnd", P=512, positions=None):
    q, k, wq, wk, dyq, dyk = _inputs(b, h, hk, n, d, dtype, n + d, layout)
    cos, sin = _tables(P, d)
    axes = _pair_axes(d, count, mixed)
    at = _positions(count, b, n, P, n) if positions is None else positions
    wide = at if at.dim() == 3 else at[:, None].expand(count, b, n)
    rows, pairs = wide.long()[axes].permute(1, 2, 0), torch.arange(d // 2, device="cuda")
    co, si = cos[rows, pairs], sin[rows, pairs]
    args = [t.requires_grad_() for t in ((q, k, wq, wk) if norm else (q, k))]
    outs = qk_rope_axes(*args[:2], cos, sin, at, axes, *args[2:], eps=EPS, interleaved=interleaved)
    grads = torch.autograd.grad(outs, args, (dyq, dyk))
    for i, (x, w, dy, name) in enumerate(((q, wq, dyq, "q"), (k, wk, dyk, "k"))):
        assert outs[i].dtype == grads[i].dtype == dtype
        if not norm:
            y, dx = _rotation(x.detach(), dy, co, si, interleaved, dtype)
        else:
            y, dx, (dw, e_dw) = _definition(x.detach(), w.detach(), dy, co, si, interleaved, dtype)
            assert_within(grads[2 + i], dw, e_dw, "dw" + name)
        assert_within(outs[i], *y, name)
        assert_within(grads[i], *dx, "d" + name)


# ------------------------------------------------------------------------------------ without a GPU
def _good(**other):
    a = dict(
        q=torch.zeros(2, 4, 8, 16), k=torch.zeros(2, 2, 8, 16), cos=torch.zeros(8, 8), sin=torch.zeros(8, 8),
        positions=torch.zeros(3, 2, 8, dtype=torch.int32), axes=[0, 1, 2] * 2 + [0, 0],
        q_weight=torch.zeros(16), k_weight=torch.zeros(16),
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
        (dict(q_weight=torch.zeros(8)), "weights must have shape"),
        (dict(q_weight=torch.zeros(16).half()), "weights must share"),
        (dict(q_weight=None), "for both"),
        (dict(k_weight=None), "for both"),
        (dict(cos=torch.zeros(8, 16)), "cos and sin must have shape"),
        (dict(sin=torch.zeros(9, 8)), "cos and sin must have shape"),
        (dict(cos=torch.zeros(8, 8).double(), sin=torch.zeros(8, 8).double()), "float32"),
        (dict(cos=torch.zeros(0, 8), sin=torch.zeros(0, 8)), "no positions"),
        (dict(positions=torch.zeros(3, 2, 8)), "positions must be int32"),
        (dict(positions=torch.zeros(8, dtype=torch.int32)), "positions must be int32"),
        (dict(positions=torch.zeros(3, 2, 7, dtype=torch.int32)), "positions must be int32"),
        (dict(positions=torch.zeros(3, 1, 8, dtype=torch.int32)), "positions must be int32"),
        (dict(positions=torch.zeros(5, 2, 8, dtype=torch.int32)), "1 to 4 axes"),
        (dict(positions=torch.zeros(0, 2, 8, dtype=torch.int32)), "1 to 4 axes"),
        (dict(axes=[0] * 7), "one axis for each of the 8 pairs"),
        (dict(axes=[0] * 7 + [3]), r"axes must lie in \[0, 3\)"),
        (dict(axes=[0] * 7 + [-1]), r"axes must lie in \[0, 3\)"),
    ],
)
def test_refusals(other, message) -> None:
    with pytest.raises(ValueError, match=message):
        qk_rope_axes(**_good(**other))


def test_no_cpu_path() -> None:
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_rope_axes(**_good())
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_rope_axes(**_good(q_weight=None, k_weight=None, positions=torch.zeros(3, 8, dtype=torch.int32)))
    assert "qk_rope_axes" in tattn.__all__


@pytest.mark.parametrize("name", ["q", "k", "cos", "sin", "q_weight", "k_weight"])
def test_forward_mode_derivatives_are_refused(name) -> None:
    with torch.autograd.forward_ad.dual_level():
        args = _good()
        args[name] = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        for take in (torch.enable_grad, torch.no_grad):
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                qk_rope_axes(**args)


@pytest.mark.parametrize("name", ["cos", "sin"])
def test_tables_that_need_gradients_are_refused(name) -> None:
    args = _good()
    args[name] = args[name].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        qk_rope_axes(**args)


def test_abi_refuses_before_any_device_call() -> None:
    import ctypes

    lib = _lib.load()
    s = _lib.strides_array(*[(512, 128, 16, 1)] * 6, (8, 8, 1))
    dims = dict(z=1, h=2, hk=2, n=8, d=16, p=8, a=2, dtype=0, w=1)

    def both(axes=(0, 1) * 4, weights=(16, 16), **o):
        ax = (ctypes.c_int32 * 64)(*axes)
        of = (dims | o).values()
        f = lib.tattn_qk_rope_axes(16, 16, *weights, *[16] * 5, ax, s, *of, 1e-6, 0, None)
        b = lib.tattn_qk_rope_axes_bwd(16, 16, *weights, *[16] * 9, ax, 16, s, *of, 1e-6, 0, None)
        assert f == b
        return f

    for bad in (dict(d=24), dict(h=0), dict(hk=0), dict(z=-1), dict(dtype=2), dict(dtype=1, w=0), dict(p=-1), dict(p=0),
                dict(a=0), dict(a=5), dict(a=1), dict(axes=(0, 1) * 3 + (0, -1)), dict(weights=(None, 16)),
                dict(weights=(16, None))):  # fmt: skip
        assert both(**bad) == _lib.ERR_INVALID_ARGUMENT
    assert both(z=1 << 20, n=1 << 10) == _lib.ERR_TOO_LARGE
    ax = (ctypes.c_int32 * 8)(*[0] * 8)
    assert lib.tattn_qk_rope_axes(None, 16, None, None, *[16] * 5, ax, s, *dims.values(), 1e-6, 0, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.tattn_qk_rope_axes(17, 16, None, None, *[16] * 5, ax, s, *dims.values(), 1e-6, 0, None) == _lib.ERR_LAYOUT
    assert lib.tattn_qk_rope_axes(16, 16, None, None, *[16] * 4, None, ax, s, *dims.values(), 1e-6, 0, None) == _lib.ERR_INVALID_ARGUMENT


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["split", "interleaved"])
@pytest.mark.parametrize("mixed", [False, True], ids=["runs", "mixed"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_against_the_definition(gpu, d, mixed, interleaved, norm, dtype) -> None:
    for (b, h, hk, n), layout, count in (((1, 1, 1, 1), "bhnd", 4), ((3, 5, 1, 17), "packed", 2), ((2, 6, 2, 70), "bnhd", 3)):
        _check(b, h, hk, n, d, dtype, count, mixed, norm, interleaved, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_many_rows(gpu, d, norm, dtype) -> None:
    """Enough rows for several heads an item and several items a thread, in head counts that 4 does not divide."""
    _check(3, 13, 3, 2500, d, dtype, 3, True, norm, layout="bnhd", P=2500)
    _check(2, 5, 5, 4001, d, dtype, 4, False, norm, interleaved=True, P=4001)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["shared", "strided", "permuted", "broadcast"])
def test_positions(gpu, shape) -> None:
    if shape == "shared":
        at = _positions(3, 1, 40, 512)[:, 0]
    elif shape == "strided":
        at = _positions(3, 6, 80, 512)[:, ::2, ::2]
    elif shape == "permuted":
        at = _positions(40, 3, 3, 512).permute(1, 2, 0)
    else:
        at = _positions(1, 3, 40, 512).expand(3, 3, 40)
    _check(3, 4, 2, 40, 64, torch.float16, positions=at)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["split", "interleaved"])
def test_one_axis_and_equal_axes_are_qk_norm_rope(gpu, interleaved, dtype) -> None:
    q, k, wq, wk, *_ = _inputs(2, 6, 2, 70, 64, dtype)
    cos, sin = _tables(512, 64)
    at = _positions(1, 2, 70, 512)
    want = qk_norm_rope(q, k, wq, wk, cos, sin, at[0], interleaved=interleaved)
    for count, mixed in ((1, False), (3, False), (4, True)):
        got = qk_rope_axes(q, k, cos, sin, at.expand(count, 2, 70), _pair_axes(64, count, mixed), wq, wk, interleaved=interleaved)
        for g, w in zip(got, want, strict=True):  # the same sums in another order: 16-bit results a rounding apart
            torch.testing.assert_close(g, w, atol=2e-6, rtol=2.0**-10 if dtype == torch.float16 else 2e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_a_position_outside_the_tables(gpu, axis, norm) -> None:
    """Whichever axis it is on, also one that no pair turns by: the token's rows are NaN, and its rows of the gradients;
    all others are as without it."""
    q, k, wq, wk, dyq, dyk = _inputs(1, 2, 1, 6, 64, torch.float16)
    cos, sin = _tables(100, 64)
    at = torch.full((3, 1, 6), 7, dtype=torch.int32, device="cuda")
    at[axis, 0] = torch.tensor([5, 99, 100, -1, 0, 2**31 - 1], dtype=torch.int32)
    axes = [j % 2 for j in range(32)]
    args = [t.requires_grad_() for t in (q, k)]
    w = (wq, wk) if norm else ()

    def both(positions):
        outs = qk_rope_axes(*args, cos, sin, positions, axes, *w)
        return (*outs, *torch.autograd.grad(outs, args, (dyq, dyk)))

    got = both(at)
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    want = both(at.clamp(0, 99))
    outside, inside = [2, 3, 5], [0, 1, 4]
    for o, w in zip(got, want, strict=True):
        assert bool(o[:, :, outside].isnan().all())
        assert torch.equal(o[:, :, inside], w[:, :, inside])


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
def test_layouts_that_need_a_copy(gpu, norm) -> None:
    q, k, wq, wk, dyq, dyk = _inputs(2, 4, 2, 30, 64, torch.float16)
    w = (wq, wk) if norm else ()
    cos, sin = _tables(64, 64)
    at, axes = _positions(3, 2, 30, 64), _pair_axes(64, 3, True)
    want = qk_rope_axes(q, k, cos, sin, at, axes, *w)
    odd = torch.empty((2, 4, 30, 65), device="cuda", dtype=torch.float16)[..., 1:].copy_(q)
    wide = torch.cat((cos, sin), 1)
    got = qk_rope_axes(odd, k, wide[:, :32], wide[:, 32:], at, tuple(axes), *w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    args = [t.clone().requires_grad_() for t in (q, k)]
    outs = qk_rope_axes(*args, cos, sin, at, axes, *w)
    one, turned = dyq[:, :, :1].expand_as(dyq), dyk.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    a = torch.autograd.grad(outs, args, (one, turned), retain_graph=True)
    b = torch.autograd.grad(outs, args, (one.contiguous(), turned.contiguous()), retain_graph=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # Only one of the results is used: the other's gradient is zeros.
    c = torch.autograd.grad(outs[0], args, dyq)
    assert not bool(c[1].any()) and bool(c[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
def test_gradients_against_differences(gpu, norm) -> None:
    """fp32, central differences with e = 2e-3 (as for qk_norm_rope: both errors are far below 1e-3 of the norm)."""
    q, k, wq, wk, dyq, dyk = _inputs(2, 3, 1, 11, 32, torch.float32, 4)
    cos, sin = _tables(64, 32)
    at, axes = _positions(3, 2, 11, 64), _pair_axes(32, 3, True)
    of = (q, k, wq, wk) if norm else (q, k)
    args = [t.clone().requires_grad_() for t in of]
    grads = torch.autograd.grad(qk_rope_axes(*args[:2], cos, sin, at, axes, *args[2:]), args, (dyq, dyk))
    e = 2e-3
    for i, t in enumerate(of):
        direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).cuda()
        values = []
        for sign in (1, -1):
            moved = [x + sign * e * direction if j == i else x for j, x in enumerate(of)]
            yq, yk = qk_rope_axes(*moved[:2], cos, sin, at, axes, *moved[2:])
            values.append(float((yq.double() * dyq).sum() + (yk.double() * dyk).sum()))
        want = float((grads[i].double() * direction).sum())
        assert abs((values[0] - values[1]) / (2 * e) - want) <= 1e-3 * max(float(grads[i].norm()), abs(want)), i


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
def test_empty_twice_and_streams(gpu, norm) -> None:
    q, k, wq, wk, dyq, dyk = _inputs(4, 16, 4, 1000, 64, torch.float16)
    cos, sin = _tables(1000, 64)
    at, axes = _positions(3, 4, 1000, 1000), _pair_axes(64, 3, True)
    args = [t.requires_grad_() for t in ((q, k, wq, wk) if norm else (q, k))]
    outs = qk_rope_axes(*args[:2], cos, sin, at, axes, *args[2:])
    first = torch.autograd.grad(outs, args, (dyq, dyk), retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(outs, args, (dyq, dyk), create_graph=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again, strict=True))
    with pytest.raises(RuntimeError, match="twice"):
        again[0].sum().backward()
    none = [t.detach()[:, :, :0].requires_grad_() for t in (q, k)]
    outs = qk_rope_axes(*none, cos, sin, at[:, :, :0], axes, *args[2:])
    grads = torch.autograd.grad(outs, (*none, *args[2:]), outs)
    assert outs[0].shape == none[0].shape and all(not bool(g.any()) for g in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "alone"])
def test_a_captured_step_reads_new_positions(gpu, norm) -> None:
    q, k, wq, wk, *_ = _inputs(2, 4, 2, 5, 64, torch.float16)
    w = (wq, wk) if norm else ()
    cos, sin = _tables(64, 64)
    at, axes = _positions(3, 2, 5, 64), _pair_axes(64, 3, False)
    qk_rope_axes(q, k, cos, sin, at, axes, *w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = qk_rope_axes(q, k, cos, sin, at, axes, *w)
    at.copy_(_positions(3, 2, 5, 64, 9))
    graph.replay()
    want = qk_rope_axes(q, k, cos, sin, at, axes, *w)
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
