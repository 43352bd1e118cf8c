"""Rotary positions of many tokens and their scaled tables (through libiam.so)
against float64."""
import math

import numpy as np
import pytest

import plain64 as P

pytestmark = pytest.mark.gpu


def frequencies(theta, rot, scaling):
    d = dict(kind="none", factor=1.0, original_ctx=0.0, low=0.0, high=0.0, magnitude=0.0)
    d.update(scaling or {})
    if d["kind"] == "base":
        theta = theta * d["factor"] ** (rot / (rot - 2))
    f, out, size = [theta ** (-2.0 * i / rot) for i in range(rot // 2)], [], 1.0
    for i, x in enumerate(f):
        keep = 1.0
        if d["kind"] == "linear":
            keep = 0.0
        elif d["kind"] == "bands":
            turns = d["original_ctx"] * x / (2 * math.pi)
            keep = min(max((turns - d["low"]) / (d["high"] - d["low"]), 0.0), 1.0)
        elif d["kind"] == "ramp":
            place = [rot * math.log(d["original_ctx"] / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (d["high"], d["low"])]
            lo, hi = max(math.floor(place[0]), 0), min(math.ceil(place[1]), rot - 1)
            keep = 1.0 - min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
        out.append(x * keep + x / d["factor"] * (1.0 - keep))
    if d["kind"] == "ramp":
        size = 0.1 * math.log(d["factor"]) + 1.0
    return np.array(out), d["magnitude"] or size


SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "base", "factor": 8.0},
            {"kind": "bands", "factor": 8.0, "original_ctx": 8192, "low": 1.0, "high": 4.0},
            {"kind": "ramp", "factor": 16.0, "original_ctx": 4096, "low": 1.0, "high": 32.0},
            {"kind": "ramp", "factor": 4.0, "original_ctx": 4096, "low": 1.0, "high": 32.0, "magnitude": 1.25},
            {"kind": "linear", "factor": 2.0, "magnitude": 0.5}]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("theta,rot,max_pos", [(10000.0, 128, 300), (1e6, 64, 70001), (10000.0, 2, 5), (500000.0, 10, 1)])
def test_table(ctx, scaling, theta, rot, max_pos):
    if scaling and scaling["kind"] == "base" and rot == 2:
        pytest.skip("the base's exponent has no value for one pair")
    t = ctx.empty(max_pos * rot, np.float32)
    ctx.rope_scaled_table(theta, rot, max_pos, t, scaling=scaling)
    got = t.read().reshape(max_pos, rot // 2, 2).astype(np.float64)
    t.free()
    f, size = frequencies(theta, rot, scaling)
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * f
    # one rounding to fp32; the angles' own error: their frequencies to a few
    # fp64 steps, times the position, and the same of the fp64 functions
    room = size * (2.0 ** -24 + max_pos * 16 * 2.0 ** -53 * f + 2.0 ** -50)
    assert (np.abs(got[..., 0] - np.cos(angle) * size) <= room).all()
    assert (np.abs(got[..., 1] - np.sin(angle) * size) <= room).all()


def rotate(x, cs, layout, rot):
    """float64 rotation of [n][heads][dim] by rows cs [n][rot/2][2], and its
    size: the sum of the magnitudes of the products."""
    y, size = x.copy(), np.abs(x)
    a = slice(0, rot // 2) if layout == "half" else slice(0, rot, 2)
    b = slice(rot // 2, rot) if layout == "half" else slice(1, rot, 2)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
    size[..., b] = np.abs(x[..., b] * c) + np.abs(x[..., a] * s)
    return y, size


# (tokens, heads, dim, rot, extra values between x rows and out rows, first value)
SHAPES = [(1, 40, 128, 128, 0, 0, 0), (1, 1, 2, 2, 0, 0, 0), (5, 3, 80, 32, 0, 0, 0), (7, 2, 96, 96, 8, 16, 0),
          (33, 40, 128, 64, 64, 0, 0), (300, 9, 64, 64, 3, 1, 1), (17, 5, 66, 40, 0, 0, 3), (129, 8, 256, 128, 0, 0, 8)]


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation(ctx, type, layout, shape):
    n, heads, dim, rot, xe, oe, first = shape
    rng = np.random.default_rng(n * 1000 + dim + len(type))
    xs, os_ = heads * dim + xe, heads * dim + oe
    words, vals = P.to_type(rng.normal(0, 2, first + n * xs + 5), type)
    max_pos = 50
    cs = rng.uniform(-1, 1, (max_pos, rot // 2, 2)).astype(np.float32)
    pos = rng.integers(0, max_pos, n).astype(np.int32)
    pos[::5] = [-1, max_pos, 2 ** 31 - 1, -2 ** 31][n % 4]       # these rows are left alone
    B = words.itemsize
    dx, dt, dp = ctx.upload(words), ctx.upload(cs), ctx.upload(pos)
    was = P.to_type(rng.normal(0, 1, first + n * os_ + 5), type)[0]
    do = ctx.upload(was)
    ctx.rope_tokens(dx.ptr + first * B, type, n, heads, dim, rot, layout, dt, max_pos, dp, do.ptr + first * B,
                    x_stride=xs, out_stride=os_)
    got_w = do.read(words.dtype)
    x = vals[first:first + n * xs].reshape(n, xs)[:, :heads * dim].reshape(n, heads, dim)
    keep = (pos < 0) | (pos >= max_pos)
    want, size = rotate(x, cs.astype(np.float64)[np.where(keep, 0, pos)], layout, rot)
    rows = got_w[first:first + n * os_].reshape(n, os_)
    old = was[first:first + n * os_].reshape(n, os_)
    got = P.from_bits(rows[:, :heads * dim], type).reshape(n, heads, dim)
    # two rounded products and a rounded sum in fp32
    P.close(got[~keep], want[~keep], 3 * 2.0 ** -24 * size[~keep], type)
    assert np.array_equal(got[~keep][..., rot:], x[~keep][..., rot:])        # passed through as they are
    assert np.array_equal(rows[keep].view(np.uint8), old[keep].view(np.uint8))
    assert np.array_equal(rows[:, heads * dim:].view(np.uint8), old[:, heads * dim:].view(np.uint8))
    assert np.array_equal(got_w[:first].view(np.uint8), was[:first].view(np.uint8))
    assert np.array_equal(got_w[first + n * os_:].view(np.uint8), was[first + n * os_:].view(np.uint8))
    # in place
    ctx.rope_tokens(dx.ptr + first * B, type, n, heads, dim, rot, layout, dt, max_pos, dp, dx.ptr + first * B,
                    x_stride=xs, out_stride=xs)
    again = dx.read(words.dtype)[first:first + n * xs].reshape(n, xs)[:, :heads * dim]
    assert np.array_equal(again[~keep].view(np.uint8), rows[~keep][:, :heads * dim].copy().view(np.uint8))
    for d in (dx, dt, dp, do):
        d.free()


def test_equals_the_single_token_rotation(iam, ctx):
    """Half layout over the whole head, fp32, an unscaled table: iam_rope's bits."""
    table = iam.rope_table(10000.0, 128, 64)
    x = np.random.default_rng(3).normal(0, 1, (6, 40 * 128)).astype(np.float32)
    pos = np.array([0, 1, 17, 63, 5, 40], np.int32)
    dx, dt, dp, do, d1 = ctx.upload(x), ctx.upload(table), ctx.upload(pos), ctx.empty(x.size, np.float32), ctx.empty(40 * 128, np.float32)
    ctx.rope_tokens(dx, "f32", 6, 40, 128, 128, "half", dt, 64, dp, do)
    got = do.read().reshape(6, -1)
    for i in range(6):
        ctx.rope(dx.ptr + i * 40 * 128 * 4, dt, dp.ptr + 4 * i, 40, 128, d1)
        assert np.array_equal(got[i].view(np.uint32), d1.read().view(np.uint32))
    for d in (dx, dt, dp, do, d1):
        d.free()


def test_refusals(iam, ctx):
    x, t, p, o = ctx.empty(4 * 256, np.float32), ctx.empty(64 * 64, np.float32), ctx.upload(np.zeros(4, np.int32)), ctx.empty(4 * 256, np.float32)
    good = dict(x=x, type="f32", n_tokens=4, n_heads=2, head_dim=128, rot_dim=64, layout="half", table=t, max_pos=64, pos=p, out=o)

    def call(**kw):
        ctx.rope_tokens(**dict(good, **kw))

    call()
    call(n_tokens=0)
    for bad in (dict(rot_dim=63), dict(rot_dim=0), dict(rot_dim=130), dict(head_dim=127, rot_dim=2), dict(n_heads=0),
                dict(n_tokens=-1), dict(n_tokens=5), dict(max_pos=65), dict(max_pos=0), dict(x_stride=255), dict(out_stride=1),
                dict(x=None), dict(out=None), dict(pos=None), dict(table=None), dict(out=x.ptr + 4), dict(x=x.ptr + 2),
                dict(out=x.ptr, n_tokens=2, out_stride=260), dict(out=t.ptr, n_tokens=1), dict(table=t.ptr + 4, max_pos=8),
                dict(x=12345 * 8)):
        with pytest.raises(iam.IamError) as e:
            call(**bad)
        assert e.value.code == iam.IAM_E_INVALID, bad
    for rot, n, theta, s in ((3, 4, 1e4, None), (0, 4, 1e4, None), (1026, 1, 1e4, None), (64, 0, 1e4, None), (64, 65, 1e4, None), (64, 4, 1.0, None),
                             (64, 4, float("nan"), None), (64, 4, 1e4, {"kind": "linear", "factor": 0.5}),
                             (64, 4, 1e4, {"kind": "bands", "factor": 2.0, "original_ctx": 100, "low": 4.0, "high": 4.0}),
                             (64, 4, 1e4, {"kind": "ramp", "factor": 2.0, "low": 1.0, "high": 4.0}),
                             (64, 4, 1e4, {"kind": "linear", "factor": 2.0, "magnitude": float("inf")})):
        with pytest.raises(iam.IamError) as e:
            ctx.rope_scaled_table(theta, rot, n, t, scaling=s)
        assert e.value.code == iam.IAM_E_INVALID, (rot, n, theta, s)
    for d in (x, t, p, o):
        d.free()


def test_rows_past_64_bits_are_refused(iam, ctx):
    """(n_tokens - 1) * stride is a multiple of 2^64: the range would seem to be one row."""
    x, t, p = ctx.empty(256, np.float32), ctx.empty(64 * 64, np.float32), ctx.upload(np.full(8, -1, np.int32))
    with pytest.raises(iam.IamError) as e:
        ctx.rope_tokens(x, "f32", (1 << 27) + 1, 2, 128, 64, "half", t, 64, p, x, x_stride=1 << 39, out_stride=1 << 39)
    assert e.value.code == iam.IAM_E_INVALID and "rope_tokens x" in str(e.value)
    for d in (x, t, p):
        d.free()
