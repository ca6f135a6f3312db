"""``tattn.decode_attention`` and ``tattn.Int4Cache``: refusals without a GPU; results on a B200 against the
definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import tattn
from tattn import Int4Cache, _lib, decode_attention, window_attention
from tests.built import ensure_built
from tests.plain64 import assert_within

ensure_built()


def _decode64(q, k, v, lengths, window, sinks, scale, c, u):
    """(o, bound): each weight and each value of a product may be off by c of it, the result by u of itself."""
    b, h, _, d = q.shape
    group = h // k.shape[1]
    o = torch.zeros((b, h, 1, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    for z in range(b):
        n = max(0, min(int(lengths[z]), k.shape[2]))
        w = n if window is None else window
        at = [j for j in range(n) if j >= n - w or j < sinks]
        if not at:
            continue
        kz, vz = (t[z][:, at].double().repeat_interleave(group, 0) for t in (k, v))
        p = torch.softmax((kz @ q[z, :, 0].double()[:, :, None])[:, :, 0] * scale, -1)[:, None]
        o[z], bound[z] = p @ vz, c * (p @ vz.abs())
    return o, bound + 2 * u * o.abs() + 2.0**-24


# fp16: P is rounded (2^-11) and scores and sums are fp32 (with exponentials to about 2^-21 of the largest
# score's size): 1e-3 of the products' magnitudes. fp32: sums of as many terms as keys or dims.
def _c(dtype, keys):
    return (1e-3, 2.0**-11) if dtype == torch.float16 else ((keys + 128) * 2.0**-23 + 2e-6, 2.0**-24)


def _inputs(b, h, hk, cap, d, dtype, seed=0, layout="bhnd", device="cuda"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((b, h, 1, d), generator=g).to(dtype).to(device)
    if layout == "bnhd":
        k, v = (torch.randn((b, cap, hk, d), generator=g).to(dtype).to(device).transpose(1, 2) for _ in range(2))
    else:
        k, v = (torch.randn((b, hk, cap, d), generator=g).to(dtype).to(device) for _ in range(2))
    return q, k, v


def _lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------ without a GPU
def _cpu(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def _len(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize(
    "q, k, lengths, window, sinks, message",
    [
        (_cpu(2, 4, 2, 16), _cpu(2, 2, 8, 16), _len(2), None, 0, "one token"),
        (_cpu(2, 4, 1, 16), _cpu(2, 3, 8, 16), _len(2), None, 0, "multiple"),
        (_cpu(2, 4, 1, 16), _cpu(1, 2, 8, 16), _len(2), None, 0, "agree"),
        (_cpu(2, 4, 1, 48), _cpu(2, 2, 8, 48), _len(2), None, 0, "head dim"),
        (_cpu(2, 4, 1, 16), _cpu(2, 2, 8, 16), _len(3), None, 0, "lengths must be int32"),
        (_cpu(2, 4, 1, 16), _cpu(2, 2, 8, 16), _len(2, dtype=torch.int64), None, 0, "lengths must be int32"),
        (_cpu(2, 4, 1, 16), _cpu(2, 2, 8, 16), _len(2), 0, 0, "window"),
        (_cpu(2, 4, 1, 16), _cpu(2, 2, 8, 16), _len(2), 4, -1, "sinks"),
    ],
)
def test_refusals(q, k, lengths, window, sinks, message) -> None:
    with pytest.raises(ValueError, match=message):
        decode_attention(q, k, k, lengths, window, sinks)


def test_no_gradients_and_no_cpu_path() -> None:
    q, k = _cpu(2, 4, 1, 16), _cpu(2, 2, 8, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        decode_attention(q, k, k, _len(2))
    with pytest.raises(RuntimeError, match="no backward"):
        decode_attention(q.requires_grad_(), k, k, _len(2))


def _cache(b=2, hk=2, cap=8, d=64):
    return Int4Cache.empty(b, hk, cap, d, device="cpu")


def test_cache_refusals() -> None:
    with pytest.raises(ValueError, match="head dim"):
        Int4Cache.empty(1, 1, 1, 32, device="cpu")
    c = _cache()
    with pytest.raises(ValueError, match="codes must be"):
        Int4Cache(c.k_codes[..., :8], c.k_params, c.v_codes, c.v_params)
    with pytest.raises(ValueError, match="expected codes"):
        Int4Cache(c.k_codes, c.k_params[:1], c.v_codes, c.v_params)
    with pytest.raises(ValueError, match="uint8"):
        Int4Cache(c.k_codes, c.k_params.float(), c.v_codes, c.v_params)
    wide = torch.zeros((2, 2, 8, 64), dtype=torch.uint8)[..., ::2]
    with pytest.raises(ValueError, match="contiguous"):
        Int4Cache(wide, c.k_params, c.v_codes, c.v_params)
    rows = _cpu(2, 2, 3, 64)
    for k, v, start, message in (
        (_cpu(2, 2, 3, 128), _cpu(2, 2, 3, 128), None, "expected k"),
        (rows, _cpu(2, 2, 4, 64), None, "expected k"),
        (rows.float(), rows.float(), None, "float16"),
        (rows, rows, _len(3), "start must be"),
        (rows, rows, _len(2, dtype=torch.int64), "start must be"),
    ):
        with pytest.raises(ValueError, match=message):
            c.append(k, v, start)
    with pytest.raises(ValueError, match="counts must be"):
        c.append(rows, rows, None, _len(1))
    with pytest.raises(ValueError, match="negative"):
        c.read(-1)
    for q, message in (
        (_cpu(1, 4, 1, 64), "expected q"), (_cpu(2, 3, 1, 64), "multiple"), (_cpu(2, 4, 2, 64), "one token"),
        (_cpu(2, 4, 1, 64).float(), "float16"),
    ):  # fmt: skip
        with pytest.raises(ValueError, match=message):
            c.attend(q, _len(2))
    for call in (lambda: c.append(rows, rows), lambda: c.read(1), lambda: c.attend(_cpu(2, 4, 1, 64), _len(2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_abi_refuses_before_any_device_call() -> None:
    lib = _lib.load()
    s = _lib.strides_array(*[(128, 64, 64, 1)] * 4)
    dims = dict(z=1, h=2, hk=2, c=8, d=64, dtype=0, w=0, s=0)
    for bad in (dict(z=-1), dict(h=3), dict(hk=0), dict(c=-1), dict(d=24), dict(dtype=2), dict(s=-1)):
        a = (dims | bad).values()
        assert lib.tattn_decode(*[16] * 6, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_decode_workspace_bytes(*a) == -1
    assert lib.tattn_decode(17, *[16] * 5, s, *dims.values(), 0.1, None) == _lib.ERR_LAYOUT
    assert lib.tattn_decode(None, None, None, None, None, None, s, 0, *list(dims.values())[1:], 0.1, None) == 0
    del dims["dtype"]
    for bad in (dict(d=32), dict(h=3), dict(c=-1)):
        a = (dims | bad).values()
        assert lib.tattn_int4_decode(*[16] * 8, s, *a, 0.1, None) == _lib.ERR_INVALID_ARGUMENT
        assert lib.tattn_int4_decode_workspace_bytes(*a) == -1
    assert lib.tattn_int4_append(*[16] * 8, s, 1, 2, 3, 8, 32, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.tattn_int4_append(18, *[16] * 7, s, 1, 2, 3, 8, 64, None) == _lib.ERR_LAYOUT
    assert lib.tattn_int4_append(*[None] * 8, s, 1, 2, 0, 8, 64, None) == 0
    assert lib.tattn_int4_read(*[16] * 7, 1, -1, 3, 8, 64, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.tattn_int4_read(*[16] * 6, 8, 1, 1, 3, 8, 64, None) == _lib.ERR_LAYOUT


def test_public_names() -> None:
    assert {"decode_attention", "Int4Cache"} <= set(tattn.__all__)


# -------------------------------------------------------------------------------------- on a B200
@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    assert _lib.device_status() == 0


CASES = [
    # h, hk, cap, lengths, window, sinks
    (1, 1, 1, (1,), None, 0),
    (4, 2, 40, (0, 1, 2, 40), None, 0),  # empty and full
    (6, 2, 70, (16, 17, 33, 70), None, 0),
    (5, 5, 130, (64, 65, 128, 130), 1, 0),
    (5, 1, 130, (64, 65, 128, 130), 64, 4),
    (8, 1, 300, (300, 5, 299, 130), 100, 130),  # sinks past the window
    (24, 2, 300, (300, 0, 77, 200), 128, 1),  # 12 heads of one: two matrix tiles
    (40, 1, 200, (200, 3), 50, 2),  # 40 heads of one: three CTAs
    (16, 4, 5000, (5000, 4999, 1, 2500), None, 0),
    (16, 4, 5000, (5000, 4999, 1, 2500), 1024, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(gpu, case, layout, d, dtype) -> None:
    h, hk, cap, lengths, window, sinks = case
    q, k, v = _inputs(len(lengths), h, hk, cap, d, dtype, 1, layout)
    o = decode_attention(q, k, v, _lens(*lengths), window, sinks)
    assert o.shape == q.shape and o.dtype == dtype
    assert_within(o, *_decode64(q, k, v, lengths, window, sinks, 1 / math.sqrt(d), *_c(dtype, cap)), "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_rows_past_a_length_are_never_used(gpu, dtype) -> None:
    q, k, v = _inputs(3, 4, 2, 200, 64, dtype, 2)
    lengths = _lens(0, 37, 128)
    want = decode_attention(q, k, v, lengths, 50, 4)
    for z, n in enumerate(lengths.tolist()):
        seen = torch.zeros(200, dtype=torch.bool, device="cuda")
        seen[max(0, n - 50) : n] = True
        seen[: min(n, 4)] = True
        k[z, :, ~seen], v[z, :, ~seen] = math.nan, math.inf
    got = decode_attention(q, k, v, lengths, 50, 4)
    assert torch.equal(got, want) and not bool(got[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_values_that_are_not_numbers_show(gpu, dtype) -> None:
    q, k, v = _inputs(2, 2, 2, 100, 64, dtype, 3)
    k[0, 0, 70, 3] = math.nan
    o = decode_attention(q, k, v, _lens(100, 100))
    assert bool(o[0, 0].isnan().all()) and bool(torch.isfinite(o[0, 1]).all()) and bool(torch.isfinite(o[1]).all())


@pytest.mark.gpu
def test_a_length_outside_the_cache(gpu) -> None:
    q, k, v = _inputs(3, 2, 1, 50, 64, torch.float16, 4)
    o = decode_attention(q, k, v, _lens(-5, 51, 2**31 - 1))
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    assert torch.equal(o, decode_attention(q, k, v, _lens(0, 50, 50)))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.4, -0.3, 0.0])
def test_scales(gpu, scale) -> None:
    for dtype in (torch.float16, torch.float32):
        q, k, v = _inputs(2, 4, 2, 333, 64, dtype, 5)
        o = decode_attention(q, k, v, _lens(333, 100), sm_scale=scale)
        assert_within(o, *_decode64(q, k, v, (333, 100), None, 0, scale, *_c(dtype, 333)), "o")


@pytest.mark.gpu
def test_large_scores(gpu) -> None:
    """Scores of hundreds: their fp32 rounding (2^-23 of 500) in the exponent adds 1e-4 to c."""
    q, k, v = _inputs(2, 4, 2, 500, 128, torch.float16, 6)
    o = decode_attention(30 * q, k, v, _lens(500, 499))
    assert_within(o, *_decode64(30 * q, k, v, (500, 499), None, 0, 128**-0.5, 1.2e-3, 2.0**-11), "o")


@pytest.mark.gpu
def test_agrees_with_window_attention(gpu) -> None:
    """The last query of a window_attention call and the token form see the same."""
    q, k, v = _inputs(2, 6, 3, 400, 64, torch.float16, 7)
    want = window_attention(q, k, v, 100, 4)
    torch.testing.assert_close(decode_attention(q, k, v, _lens(400, 400), 100, 4), want, atol=2e-3, rtol=2e-3)


@pytest.mark.gpu
def test_layouts(gpu) -> None:
    q, k, v = _inputs(2, 4, 2, 60, 64, torch.float16, 8)
    want = decode_attention(q, k, v, _lens(60, 31))
    odd = torch.empty((2, 4, 1, 65), device="cuda", dtype=torch.float16)[..., 1:].copy_(q)
    strided = torch.stack((_lens(60, 31), _lens(0, 0)), 1)[:, 0]
    assert torch.equal(decode_attention(odd, k, v, strided), want)
    part = torch.empty((2, 2, 100, 128), device="cuda", dtype=torch.float16)
    part[:, :, 20:80, 64:] = k
    assert torch.equal(decode_attention(q, part[:, :, 20:80, 64:], v, _lens(60, 31)), want)
    with pytest.raises(ValueError, match="read in place"):
        decode_attention(q, part[:, :, 20:80, 1:65], v, _lens(60, 31))


@pytest.mark.gpu
def test_nothing_to_attend_with(gpu) -> None:
    q, k, v = _inputs(2, 0, 1, 50, 64, torch.float16, 4)
    assert decode_attention(q, k, v, _lens(3, 4)).shape == q.shape
    q, k, v = _inputs(0, 2, 1, 50, 64, torch.float16, 4)
    assert decode_attention(q, k, v, _lens()).shape == q.shape
    q, k, v = _inputs(2, 2, 1, 0, 64, torch.float16, 4)
    assert not bool(decode_attention(q, k, v, _lens(0, 0)).any())
    cache = Int4Cache.empty(2, 1, 0, 64)
    assert not bool(cache.attend(q, _lens(0, 0)).any())
    cache.append(k, v)
    assert cache.read(0)[0].shape == (2, 1, 0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1000, 4000, 40000])
def test_every_way_of_joining_parts(gpu, cap) -> None:
    """One sequence of few heads is cut into as many parts as its capacity allows: a cluster or a second kernel;
    with parts that hold nothing (a short length) in both."""
    for d, h in ((64, 1), (128, 12)):
        q, k, v = _inputs(2, h, 1, cap, d, torch.float16, 23)
        cache = Int4Cache.empty(2, 1, cap, d)
        cache.append(k, v)
        for lengths in ((cap, cap - 1), (1, 40), (0, 700)):
            o = decode_attention(q, k, v, _lens(*lengths))
            assert_within(o, *_decode64(q, k, v, lengths, None, 0, d**-0.5, 1e-3, 2.0**-11), "o")
            o = cache.attend(q, _lens(*lengths))
            assert_within(o, *_decode64(q, *_exact_values(cache), lengths, None, 0, d**-0.5, 2e-3, 2.0**-11), "4 bits")


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu) -> None:
    """The last sequence's rows begin past 2^32 elements of a cache and 2^32 bytes of codes."""
    b, cap, d = 3, 1 << 24, 128
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    k, v = (torch.empty((b, 1, cap, d), device="cuda", dtype=torch.float16) for _ in range(2))
    q, rows, _ = _inputs(b, 2, 1, 300, d, torch.float16, 9)
    n = cap - 5
    k[2, 0, n - 300 : n], v[2, 0, n - 300 : n] = rows[2, 0], rows[1, 0]
    o = decode_attention(q, k, v, _lens(0, 0, n), 300)
    want = _decode64(q[2:], rows[2:], rows[1:2], (300,), None, 0, d**-0.5, 1e-3, 2.0**-11)
    assert_within(o[2:], *want, "o")
    del k, v
    cache = Int4Cache.empty(5, 1, cap, d)
    start = _lens(0, 0, 0, 0, n - 300)
    cache.append(rows[:1].expand(5, 1, 300, d), rows[1:2].expand(5, 1, 300, d), start)
    ck, cv = cache.read(300, start)
    q5 = q[:1].expand(5, 2, 1, d)
    o = cache.attend(q5, _lens(0, 0, 0, 0, n), 300)
    want = _decode64(q5[4:], ck[4:], cv[4:], (300,), None, 0, d**-0.5, 1e-3, 2.0**-11)
    assert_within(o[4:], *want, "o")
    assert torch.equal(ck[4], ck[0]) and torch.equal(cv[4], cv[0])


# ------------------------------------------------------------------------------------- 4-bit cache
def _quantized(x):
    """Codes, scales and minima of fp16 rows by the format's definition."""
    g = x.double().unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    span = (high - low).float()
    s = (span / torch.full_like(span, 15)).half().double()  # (a division; by a number torch multiplies with 1 / 15)
    n = torch.where(s > 0, ((g - low).float() / s.float()).double().round(), 0.0).clamp(0, 15)
    return n.flatten(-2).to(torch.uint8), torch.stack((s.squeeze(-1), low.squeeze(-1)), -1).half()


def _codes(cache):
    return [torch.stack((c & 15, c >> 4), -1).flatten(-2) for c in (cache.k_codes, cache.v_codes)]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("t", [1, 33])
def test_append_and_read(gpu, t, layout, d) -> None:
    _, k, v = _inputs(3, 1, 2, t, d, torch.float16, 10, layout)
    k[0, 0, 0] = 0.25  # a constant row: scale 0
    k[1, 1, 0, :64] *= 3000  # a wide one
    v[2, 0, 0] *= 1e-4  # one of subnormals
    cache = Int4Cache.empty(3, 2, 50, d)
    start, counts = _lens(0, 7, 17), _lens(t, t, max(0, t - 3))
    cache.append(k, v, start, counts)
    for x, codes, params in zip((k, v), _codes(cache), (cache.k_params, cache.v_params), strict=True):
        n, p = _quantized(x)
        for z in range(3):
            at, c = int(start[z]), int(counts[z])
            assert torch.equal(codes[z, :, at : at + c], n[z, :, :c])
            assert torch.equal(params[z, :, at : at + c], p[z, :, :c])
            rest = torch.ones(50, dtype=torch.bool, device="cuda")
            rest[at : at + c] = False
            assert not bool(codes[z, :, rest].any()) and not bool(params[z, :, rest].any())
    values = cache.read(t, start)
    for y, codes, params in zip(values, _codes(cache), (cache.k_params, cache.v_params), strict=True):
        p = params.double()
        want = (p[..., :1] * codes.double().unflatten(-1, (-1, 64)) + p[..., 1:]).flatten(-2).half()
        for z in range(3):
            at = int(start[z])
            assert torch.equal(y[z], want[z, :, at : at + t])
    whole = cache.read(50)
    assert torch.equal(whole[0][1, :, 7 : 7 + t], values[0][1])


@pytest.mark.gpu
def test_codes_are_the_rounded_quotients(gpu) -> None:
    """Quotients at and next to the midpoints between codes, at many scales: as torch divides and rounds."""
    g = torch.Generator().manual_seed(22)
    rows = 20000
    s = (2.0 ** (torch.rand(rows, 1, generator=g) * 24 - 14)).half().double()
    half = torch.randint(0, 31, (rows, 128), generator=g).double() / 2
    x = (s * half + (torch.rand(rows, 1, generator=g) - 0.5).half().double() * s).half()
    x[:, 0::64], x[:, 1::64] = (x.amin(-1, keepdim=True), (x.amin(-1, keepdim=True).double() + 15 * s).half())
    step = torch.randint(-1, 2, x.shape, generator=g, dtype=torch.int16)
    x = torch.where(torch.isfinite(x) & (x.view(torch.int16).abs() > 2), (x.view(torch.int16) + step).view(torch.float16), x)
    x = x.cuda().reshape(1, 1, rows, 128)
    cache = Int4Cache.empty(1, 1, rows, 128)
    cache.append(x, x)
    n, p = _quantized(x)
    assert torch.equal(cache.k_params, p) and torch.equal(_codes(cache)[0], n) and torch.equal(_codes(cache)[1], n)


@pytest.mark.gpu
def test_rows_past_the_capacity(gpu) -> None:
    _, k, v = _inputs(2, 1, 1, 6, 64, torch.float16, 11)
    cache, whole = Int4Cache.empty(2, 1, 10, 64), Int4Cache.empty(2, 1, 20, 64)
    start = _lens(3, 8)
    cache.append(k, v, start)
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    whole.append(k, v, start)
    assert torch.equal(cache.k_codes, whole.k_codes[:, :, :10]) and torch.equal(cache.v_params, whole.v_params[:, :, :10])
    got, want = cache.read(6, start)[0], whole.read(6, start)[0]
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :, :2], want[1, :, :2]) and not bool(got[1, :, 2:].any())
    cache.append(k, v, _lens(-3, 2**31 - 2))
    assert _lib.device_status() == _lib.DEV_INDEX_RANGE
    assert torch.equal(cache.k_codes[0, :, :3], whole_codes(k)[0, :, 3:6])


def whole_codes(k):
    n = _quantized(k)[0]
    return n[..., 0::2] | (n[..., 1::2] << 4)


INT4_CASES = [c for c in CASES]


def _filled(b, hk, cap, d, seed, size=1.0):
    _, k, v = _inputs(b, 1, hk, cap, d, torch.float16, seed)
    cache = Int4Cache.empty(b, hk, cap, d)
    cache.append(k * size, v * size)
    return cache


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend_against_the_definition(gpu, case, d) -> None:
    h, hk, cap, lengths, window, sinks = case
    cache = _filled(len(lengths), hk, cap, d, 12)
    q, _, _ = _inputs(len(lengths), h, 1, 1, d, torch.float16, 13)
    o = cache.attend(q, _lens(*lengths), window, sinks)
    k, v = cache.read(cap)
    # The values are rounded to fp16 on reading and not in the kernel: 2^-11 more of each key and value; a
    # score's error is 2^-11 sum |q k| scale, itself some times the score's size.
    assert_within(o, *_decode64(q, k, v, lengths, window, sinks, 1 / math.sqrt(d), 4e-3, 2.0**-11), "o")
    exact = _exact_values(cache)
    assert_within(o, *_decode64(q, *exact, lengths, window, sinks, 1 / math.sqrt(d), 1e-3, 2.0**-11), "o")


def _exact_values(cache):
    """Scale * code + minimum without the rounding to fp16."""
    out = []
    for codes, params in zip(_codes(cache), (cache.k_params, cache.v_params), strict=True):
        p = params.double()
        out.append((p[..., :1] * codes.double().unflatten(-1, (-1, 64)) + p[..., 1:]).flatten(-2))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2e-4, 1000.0])
def test_attend_small_and_large_values(gpu, size) -> None:
    """Scales near fp16's subnormals, and scores of thousands (2^-23 of them in the exponent: 1e-3 in c)."""
    cache = _filled(2, 2, 200, 128, 14, size)
    q, _, _ = _inputs(2, 4, 1, 1, 128, torch.float16, 15)
    o = cache.attend(q, _lens(200, 150))
    assert_within(o, *_decode64(q, *_exact_values(cache), (200, 150), None, 0, 128**-0.5, 3e-3, 2.0**-11), "o")


@pytest.mark.gpu
def test_attend_with_very_unequal_tokens(gpu) -> None:
    """Values of neighbouring tokens a thousand times apart, either kind first, the small ones with nearly all
    of the weight: weights are scaled by the largest value scale so far, and 2^-24 of that is what a small
    token's weight may lose."""
    for first in (1.0, 1e-3):
        _, k, v = _inputs(1, 1, 1, 300, 64, torch.float16, 16)
        sizes = torch.where(torch.arange(300, device="cuda") % 150 < 75, first, 1e-3 / first).half()
        v = v * sizes[None, None, :, None]
        q, _, _ = _inputs(1, 2, 1, 1, 64, torch.float16, 17)
        k[0, 0, :, 0] = torch.where(sizes < 0.5, 2.0, -2.0).half()
        q[..., 0] = 20
        cache = Int4Cache.empty(1, 1, 300, 64)
        cache.append(k, v)
        o = cache.attend(q, _lens(300))
        kx, vx = _exact_values(cache)
        want, bound = _decode64(q, kx, vx, (300,), None, 0, 0.125, 1e-3, 2.0**-11)
        assert_within(o, want, bound + 300 * 15 * 2.0**-24 * float(cache.v_params[..., 0].max()), "o")


@pytest.mark.gpu
def test_attend_ignores_rows_past_a_length(gpu) -> None:
    cache = _filled(2, 1, 100, 64, 18)
    q, _, _ = _inputs(2, 2, 1, 1, 64, torch.float16, 19)
    want = cache.attend(q, _lens(0, 41))
    for p in (cache.k_params, cache.v_params):
        p[0], p[1, :, 41:] = math.nan, math.nan
    got = cache.attend(q, _lens(0, 41))
    assert torch.equal(got, want) and not bool(got[0].any())


@pytest.mark.gpu
def test_a_captured_step(gpu) -> None:
    """Append and attend in a CUDA graph, replayed as the lengths grow on the device."""
    b, h, hk, d = 2, 4, 2, 64
    _, ks, vs = _inputs(b, 1, hk, 20, d, torch.float16, 20)
    q, _, _ = _inputs(b, h, 1, 1, d, torch.float16, 21)
    cache, other = Int4Cache.empty(b, hk, 32, d), Int4Cache.empty(b, hk, 32, d)
    k, v, held = ks[:, :, :1].clone(), vs[:, :, :1].clone(), _lens(0, 0)

    def step():
        cache.append(k, v, held)
        held.add_(1)
        return cache.attend(q, held, 8, 2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # warm-up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    held.zero_()
    other.append(ks, vs)
    for i in range(20):
        k.copy_(ks[:, :, i : i + 1])
        v.copy_(vs[:, :, i : i + 1])
        graph.replay()
        assert torch.equal(out, other.attend(q, _lens(i + 1, i + 1), 8, 2)), i


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_append_shows_what_is_not_a_number(gpu, d) -> None:
    """A group of 64 dims with a NaN or an infinity among them reads as NaN, wherever it lies and whatever else the
    group holds; every other group is as it would be alone. Attention shows it too."""
    _, k, v = _inputs(2, 1, 2, 80, d, torch.float16, 24)
    clean = Int4Cache.empty(2, 2, 80, d)
    clean.append(k, v)
    hit = [torch.zeros(2, 2, 80, d // 64, dtype=torch.bool, device="cuda") for _ in range(2)]
    kinds = (math.nan, math.inf, -math.inf)
    for i in range(64):  # every place of a group, in different rows
        for x, h, n in ((k, hit[0], i), (v, hit[1], 3 * i)):
            x[i % 2, 0, n % 80, 64 * (i % (d // 64)) + i] = kinds[i % 3]
            h[i % 2, 0, n % 80, i % (d // 64)] = True
    k[0, 0, 79, :2], k[1, 0, 79, :2] = torch.tensor([math.nan, math.inf]), torch.tensor([math.inf, -math.inf])
    hit[0][:, 0, 79, 0] = True
    cache = Int4Cache.empty(2, 2, 80, d)
    cache.append(k, v)
    for got, want, h in zip(cache.read(80), clean.read(80), hit, strict=True):
        h = h.repeat_interleave(64, -1)
        assert bool(got[h].isnan().all()) and torch.equal(got[~h], want[~h])
    q, _, _ = _inputs(2, 2, 1, 1, d, torch.float16, 25)
    o, want = cache.attend(q, _lens(80, 80)), clean.attend(q, _lens(80, 80))
    assert bool(o[:, 0].isnan().all()) and torch.equal(o[:, 1], want[:, 1])
    only_v = Int4Cache(clean.k_codes, clean.k_params, cache.v_codes, cache.v_params)
    o, h = only_v.attend(q, _lens(80, 80)), hit[1].any(2).repeat_interleave(64, -1)[:, :, None]
    assert bool(o[h].isnan().all()) and torch.equal(o[~h], want[~h])


@pytest.mark.gpu
def test_the_whole_range_of_fp16_reads_back_finite(gpu) -> None:
    """Groups that reach 65504, with minima from there down to -65504: each value is within half a step of its own, or
    at the top within what 15 steps of a scale rounded down fall short (15 units in its last place: 120 at most),
    and rounded to fp16 (16 there)."""
    g = torch.Generator().manual_seed(26)
    top = 65504.0
    low = torch.cat((torch.tensor([-top, 0.0, -1.0, 1.0, 600.0, 65000.0, top]), (torch.rand(993, generator=g) * 2 - 1) * top))
    x = (low[:, None] + torch.rand(1000, 64, generator=g) * (top - low[:, None])).half().clamp(-top, top)
    x[:, 0], x[:, 1] = low.half(), top
    x = torch.cat((x, -x), 1).cuda().reshape(1, 1, 1000, 128)  # and the same below zero
    cache = Int4Cache.empty(1, 1, 1000, 128)
    cache.append(x, x)
    for y, p in zip(cache.read(1000), (cache.k_params, cache.v_params), strict=True):
        s = p[..., 0].double().repeat_interleave(64, -1)
        assert_within(y, x.double(), (s / 2).clamp(min=120) + 16, "values")
    q = torch.full((1, 1, 1, 128), 1e-4, device="cuda", dtype=torch.float16)
    assert bool(torch.isfinite(cache.attend(q, _lens(1000))).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("sm_scale", [0.125, -0.125])
def test_scores_of_minus_infinity(gpu, sm_scale, dtype) -> None:
    """Keys with an infinity that makes their scores -infinity weigh nothing, also where they fill whole tiles, ahead
    of all others or behind them; where all that is seen is such keys there is no result."""
    q, k, v = _inputs(3, 4, 2, 700, 64, dtype, 27)
    q[..., 3] = 1.0
    lengths = (700, 300, 90)
    for first, last in ((0, 60), (0, 690), (300, 700), (100, 130)):
        bad = k.clone()
        bad[:, :, first:last, 3] = math.copysign(math.inf, -sm_scale)
        o = decode_attention(q, bad, v, _lens(*lengths), sm_scale=sm_scale)
        for z, n in enumerate(lengths):
            at = [j for j in range(n) if not first <= j < last]
            if not at:
                assert bool(o[z].isnan().all())
                continue
            want, bound = _decode64(
                q[z : z + 1], k[z : z + 1, :, at], v[z : z + 1, :, at], (len(at),), None, 0, sm_scale, *_c(dtype, n)
            )
            assert_within(o[z : z + 1], want, bound, f"{first} to {last}, length {n}")
    cut = decode_attention(q, bad, v, _lens(700, 110, 101), 10, 0, sm_scale)  # the window hides or shows them
    assert bool(torch.isfinite(cut[0]).all()) and bool(cut[1].isnan().all()) and bool(torch.isfinite(cut[2]).all())
    assert not bool(decode_attention(q, bad, v, _lens(0, 0, 0), sm_scale=sm_scale).any())


@pytest.mark.gpu
@pytest.mark.parametrize("sm_scale", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_no_number_shows(gpu, sm_scale) -> None:
    for dtype in (torch.float16, torch.float32):
        q, k, v = _inputs(2, 4, 2, 90, 64, dtype, 28)
        assert bool(decode_attention(q, k, v, _lens(90, 50), sm_scale=sm_scale).isnan().all())
        assert bool(window_attention(q, k, v, 40, sm_scale=sm_scale).isnan().all())
        assert not bool(decode_attention(q, k, v, _lens(0, 0), sm_scale=sm_scale).any())
    assert bool(_filled(2, 2, 90, 64, 29).attend(q.half(), _lens(90, 50), sm_scale=sm_scale).isnan().all())


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(which) -> None:
    """Without a GPU: before the device check."""
    with torch.autograd.forward_ad.dual_level():
        args = [_cpu(2, 4, 1, 64), _cpu(2, 2, 8, 64), _cpu(2, 2, 8, 64)]
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for take in (torch.enable_grad, torch.no_grad):
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                decode_attention(*args, _len(2))
            with take(), pytest.raises(NotImplementedError, match="forward-mode"):
                _cache().append(*args[1:]) if which else _cache().attend(args[0], _len(2))


@pytest.mark.parametrize("which", [1, 2])
def test_keys_and_values_that_need_gradients_are_refused(which) -> None:
    """Of each tensor alone; without gradients being recorded they are taken (as far as the device check)."""
    args = [_cpu(2, 4, 1, 64), _cpu(2, 2, 8, 64), _cpu(2, 2, 8, 64)]
    args[which].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        decode_attention(*args, _len(2))
    with pytest.raises(RuntimeError, match="no gradients"):
        _cache().append(*args[1:])
    with torch.no_grad():
        for call in (lambda: decode_attention(*args, _len(2)), lambda: _cache().append(*args[1:])):
            with pytest.raises(RuntimeError, match="no CPU path"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend_against_the_values_that_codes_stand_for(gpu, case, d) -> None:
    """The format's values are fp16(s n + m), which read gives (checked bit for bit above); over them a 4-bit cache is
    held to what an fp16 cache is."""
    h, hk, cap, lengths, window, sinks = case
    cache = _filled(len(lengths), hk, cap, d, 30)
    q, _, _ = _inputs(len(lengths), h, 1, 1, d, torch.float16, 31)
    o = cache.attend(q, _lens(*lengths), window, sinks)
    k, v = cache.read(cap)
    assert_within(o, *_decode64(q, k, v, lengths, window, sinks, 1 / math.sqrt(d), *_c(torch.float16, cap)), "o")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attend_takes_the_rounded_values(gpu, d) -> None:
    """Keys around 8 in a range of a quarter: fp16(s n + m) is up to 2^-8 from s n + m, which under queries of 16 moves a
    score by some 0.04 and the weights of five tokens by as much. c: 1e-3 as above, and twice what fp32 sums of d
    products (d 2^-24 of the sum of their sizes) leave in the exponent."""
    _, k, v = _inputs(8, 1, 2, 5, d, torch.float16, 32)
    q, _, _ = _inputs(8, 8, 1, 1, d, torch.float16, 33)
    q, k = 16 * q, (8 + 0.05 * k.float()).half()
    cache = Int4Cache.empty(8, 2, 5, d)
    cache.append(k, v)
    o = cache.attend(q, _lens(*[5] * 8))
    k, v = cache.read(5)
    scale = d**-0.5
    size = float((q.double().abs().sum(-1) * 8.2).max()) * scale
    c = 1e-3 + 2 * d * 2.0**-24 * size
    want, bound = _decode64(q, k, v, [5] * 8, None, 0, scale, c, 2.0**-11)
    assert_within(o, want, bound, "o")
    unrounded = []
    for codes, params in zip(_codes(cache), (cache.k_params, cache.v_params), strict=True):
        p = params.double()
        unrounded.append((p[..., :1] * codes.double().unflatten(-1, (-1, 64)) + p[..., 1:]).flatten(-2))
    other, _ = _decode64(q, *unrounded, [5] * 8, None, 0, scale, c, 2.0**-11)
    assert int(((other - want).abs() > bound).sum()) > 100  # the test tells the two apart


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2e-4, 1000.0])
def test_attend_small_and_large_values_as_read(gpu, size) -> None:
    """Scales near fp16's subnormals, and scores of some thousands: fp32 sums of 128 products (128 2^-24 of the sum of
    their sizes) are twice in c."""
    cache = _filled(2, 2, 200, 128, 34, size)
    q, _, _ = _inputs(2, 4, 1, 1, 128, torch.float16, 35)
    k, v = cache.read(200)
    terms = float((q[:, :, 0].double().abs().unflatten(1, (2, 2)) @ k.double().abs().transpose(-1, -2)).max()) * 128**-0.5
    c = 1e-3 + 2 * 128 * 2.0**-24 * terms
    o = cache.attend(q, _lens(200, 150))
    assert_within(o, *_decode64(q, k, v, (200, 150), None, 0, 128**-0.5, c, 2.0**-11), "o")


@pytest.mark.gpu
def test_attend_with_very_unequal_tokens_as_read(gpu) -> None:
    """Values of neighbouring tokens a thousand times apart, either kind first, the small ones with nearly all of the
    weight: nothing is lost beyond each product's own rounding. A weight below 2^-14 of the largest one is rounded to
    2^-25 of that, in fp16's subnormals."""
    for first in (1.0, 1e-3):
        _, k, v = _inputs(1, 1, 1, 300, 64, torch.float16, 36)
        sizes = torch.where(torch.arange(300, device="cuda") % 150 < 75, first, 1e-3 / first).half()
        q, _, _ = _inputs(1, 2, 1, 1, 64, torch.float16, 37)
        k[0, 0, :, 0] = torch.where(sizes < 0.5, 2.0, -2.0).half()
        q[..., 0] = 20
        cache = Int4Cache.empty(1, 1, 300, 64)
        cache.append(k, v * sizes[None, None, :, None])
        o = cache.attend(q, _lens(300))
        kx, vx = cache.read(300)
        want, bound = _decode64(q, kx, vx, (300,), None, 0, 0.125, 1e-3, 2.0**-11)
        most = torch.softmax(kx[0, 0].double() @ q[0, :, 0].double().T * 0.125, 0).max()
        assert_within(o, want, bound + 2.0**-25 * most * vx.double().abs().sum(2, keepdim=True), "o")


@pytest.mark.gpu
def test_caches_on_side_streams(gpu) -> None:
    """Two streams append to caches of their own and attend over them at the same time (parts joined by a second kernel,
    through a workspace): each gets what it gets alone."""
    cap, lengths = 40000, _lens(40000)

    def work(i):
        q, k, v = rows[i]
        cache = Int4Cache.empty(1, 1, cap, 64)
        cache.append(k, v)
        return cache.attend(q, lengths), decode_attention(q, k, v, lengths)

    rows = [_inputs(1, 2, 1, cap, 64, torch.float16, 38 + i) for i in range(2)]
    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(work(i))
    for side in sides:
        side.synchronize()
    for results, first in zip(got, want, strict=True):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, first, strict=True))
