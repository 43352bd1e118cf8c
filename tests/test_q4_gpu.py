"""Matrices of 4-bit weights and their products (through libiam.so) against
float64."""
import numpy as np
import pytest

import plain64 as P
import plain_rows as R

pytestmark = pytest.mark.gpu

GUARD = 24


def packed(iam, ctx, w):
    m = iam.Q4Matrix(ctx, w.out, w.inp, w.group, zeros=w.zero is not None)
    src = [ctx.upload(w.plain_bytes()), ctx.upload(w.scale)] + ([ctx.upload(w.zero)] if w.zero is not None else [])
    m.pack(*src)
    ctx.sync()
    for b in src:
        b.free()
    return m


def rows_of(rng, rows, inp, type, x_group=0):
    """(stored words, scales or None, float64 values) of random rows."""
    x = rng.normal(0, 1, (rows, inp)) * np.where(rng.random(inp) < 0.02, 20, 1)
    if type in P.TYPES:
        w, v = P.to_type(x, type)
        return w, None, v
    q = rng.integers(-127, 128, (rows, inp)) if type == "int8" else R.e4m3(rng.integers(0, 127, (rows, inp)) | rng.integers(0, 2, (rows, inp)) << 7)
    s = rng.uniform(0.5, 2, (rows, -(-inp // x_group) if x_group else 1)).astype(np.float32)
    return R.bytes_of(q, type), s, q * R.spread(s, x_group, inp)


def product(ctx, m, words, scale, type, y_type, x_group=0, x_stride=0, y_stride=0, first=0):
    """Rows laid out `x_stride` apart from element `first` on; y between guards.
    What lies between the rows is NaN (or the largest number)."""
    rows, inp = words.shape
    xs, ys = x_stride or inp, y_stride or m.desc.out_dim
    out = m.desc.out_dim
    flat = np.full(first + rows * xs + GUARD, 0x7f if words.dtype == np.uint8 else 0x7fff if words.dtype == np.uint16 else np.nan, words.dtype)
    flat[first:first + rows * xs].reshape(rows, xs)[:, :inp] = words
    dt = P.storage(y_type)
    guard = np.full(rows * ys + 2 * GUARD, 77, dt)
    dx, dy = ctx.upload(flat), ctx.upload(guard)
    ds = ctx.upload(scale) if scale is not None else None
    m.mul(dx.ptr + first * words.itemsize, type, rows, dy.ptr + GUARD * dt().itemsize, y_type, x_scale=ds, x_group=x_group,
          x_stride=x_stride, y_stride=y_stride)
    got = dy.read()
    for b in (dx, dy, ds):
        if b is not None:
            b.free()
    body = got[GUARD:-GUARD].reshape(rows, ys)
    assert (got[:GUARD] == 77).all() and (got[-GUARD:] == 77).all() and (body[:, out:] == 77).all()
    return P.from_bits(body[:, :out], y_type)


def check(iam, ctx, rng, rows, inp, out, group, zeros, type, y_type, x_group=0, **kw):
    w = R.random_weights(rng, out, inp, group, zeros)
    m = packed(iam, ctx, w)
    words, scale, x = rows_of(rng, rows, inp, type, x_group)
    got = product(ctx, m, words, scale, type, y_type, x_group, **kw)
    m.free()
    v = w.values()
    P.close(got, x @ v.T, R.product_bound(x, v), y_type)


# one token and few, odd widths, a row or a tile too many or too few of each kind
SHAPES = [(1, 1, 1), (1, 4096, 1024), (1, 14336, 40), (1, 1000, 2001), (2, 31, 17), (3, 129, 16), (4, 700, 100), (5, 100, 33), (5, 2048, 4100),
          (6, 512, 15), (8, 1024, 65), (11, 640, 48), (16, 1100, 70), (17, 1000, 250), (32, 2048, 130), (33, 384, 129), (48, 4096, 64),
          (64, 2048, 96), (65, 257, 130), (100, 5000, 31), (129, 1024, 272), (300, 700, 520), (513, 130, 1030)]


@pytest.mark.parametrize("type", R.ROW_TYPES)
@pytest.mark.parametrize("rows,inp,out", SHAPES)
def test_products(iam, ctx, rows, inp, out, type):
    rng = np.random.default_rng(rows * 7 + inp + out)
    k = rows + inp + R.ROW_TYPES.index(type)
    check(iam, ctx, rng, rows, inp, out, (32, 64, 128)[k % 3], k % 2 == 0, type, P.TYPES[k // 2 % 3], 128 * (k // 3 % 2) if type not in P.TYPES else 0)


@pytest.mark.parametrize("type", R.ROW_TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 7, 40, 200])
def test_whole_numbers_are_exact(iam, ctx, rows, group, zeros, type):
    """Small whole numbers: every product and sum is one that fp32 holds, so the
    result is equal whatever the order (sums below 900 * 15 * 15)."""
    rng = np.random.default_rng(group + rows)
    inp, out = 900, 200
    groups = -(-inp // group)
    w = R.Weights(rng.integers(0, 16, (out, inp)), np.exp2(rng.integers(-1, 2, (out, groups))), rng.integers(0, 16, (out, groups)).astype(np.uint8) if zeros else None, group)
    x = rng.integers(-15, 16, (rows, inp)).astype(np.float64)
    words = P.to_type(x, type)[0] if type in P.TYPES else R.bytes_of(x, type)
    scale = None if type in P.TYPES else np.full((rows, 1), 0.5, np.float32)
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, scale, type, "f32")
    m.free()
    assert np.array_equal(got, (x * (1 if scale is None else 0.5)) @ w.values().T)


@pytest.mark.parametrize("type,first,x_stride", [("f32", 1, 4097), ("f32", 3, 4100), ("f16", 1, 4097), ("bf16", 5, 4104), ("f16", 8, 4104), ("int8", 3, 4099), ("int8", 16, 4112), ("e4m3", 1, 0)])
@pytest.mark.parametrize("rows", [1, 5, 30, 150])
def test_strides_and_alignment(iam, ctx, rows, type, first, x_stride):
    rng = np.random.default_rng(first)
    check(iam, ctx, rng, rows, 4096, 100, 128, False, type, "f16" if type == "f16" else "f32", first=first, x_stride=x_stride, y_stride=103)


@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("type", P.TYPES)
def test_values_far_apart(iam, ctx, rows, type):
    """Tiles of unlike size, tiny and huge ones, all zeros."""
    rng = np.random.default_rng(3)
    w = R.random_weights(rng, 48, 1280, 64, True)
    x = rng.normal(0, 1, (rows, 1280)) * np.repeat(10.0 ** np.array([0, 4, -7, 3, -3, 0, -9, 4, -2, 1]), 128)
    x[:, 640:768] = 0
    if rows > 1:
        x[1] = 0
    words, v = P.to_type(x, type)
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, None, type, "f32")
    m.free()
    P.close(got, v @ w.values().T, R.product_bound(v, w.values()), "f32")


@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_values_near_the_largest(iam, ctx, rows, type):
    """Sums that only the scales bring back into fp32's range: of 640 weights up
    to 15 * 2^-10 and x up to 2^126 they stay below 2^126 * 640 * 15 / 1024, and
    random signs keep them below 2^127."""
    rng = np.random.default_rng(8)
    w = R.random_weights(rng, 40, 640, 128, False)
    w.scale[:] = 2.0 ** -10
    x = rng.uniform(-1, 1, (rows, 640)) * 2.0 ** 126
    words, v = P.to_type(x, type)
    want = v @ w.values().T
    assert np.abs(want).max() < 2.0 ** 127
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, None, type, "f32")
    m.free()
    P.close(got, want, R.product_bound(v, w.values()), "f32")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("type,x_group", [("f32", 0), ("bf16", 0), ("int8", 0), ("int8", 128)])
def test_workgroups_for_every_unit(iam, ctx, type, x_group, group, zeros):
    """As many products as the widest workgroups take."""
    check(iam, ctx, np.random.default_rng(group), 2040, 300, 4090, group, zeros, type, "f32" if zeros else "bf16", x_group, y_stride=4095)


@pytest.mark.parametrize("type", ["f32", "f16", "int8", "e4m3"])
@pytest.mark.parametrize("rows,inp,out", [(1, 14336, 200), (5, 9000, 130), (3, 20000, 1500), (2, 8193, 17), (4, 70001, 16)])
def test_few_rows_of_long_inputs(iam, ctx, rows, inp, out, type):
    rng = np.random.default_rng(rows + inp)
    for k in range(2):     # the counters are left as they were
        check(iam, ctx, rng, rows, inp, out, (32, 64, 128)[(rows + k) % 3], k == 1, type, "f32", 128 * k if type not in P.TYPES else 0)


def test_many_rows_and_outputs(iam, ctx):
    """More rows than a pass takes, more strips than a launch packs."""
    rng = np.random.default_rng(9)
    check(iam, ctx, rng, (1 << 14) + 37, 40, 20, 32, True, "bf16", "f32")
    check(iam, ctx, rng, 1, 1, (1 << 19) + 17, 32, False, "f32", "f32")


@pytest.mark.parametrize("rows", [1, 9, 130])
@pytest.mark.parametrize("type", P.TYPES)
def test_not_finite_rows(iam, ctx, rows, type):
    """An infinity or a NaN makes nothing of its own row's finite, and the others stay."""
    rng = np.random.default_rng(4)
    w = R.random_weights(rng, 70, 600, 128, False)
    w.n[:, 5] = 9    # no zero weight meets it
    x = rng.normal(0, 1, (rows, 600))
    x[0, 5] = np.inf if type != "bf16" else np.nan
    if rows > 3:
        x[3, 599] = -np.inf
        w.n[:, 599] = 3
    words, v = P.to_type(x, type)
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, None, type, "f32")
    m.free()
    assert not np.isfinite(got[0]).any()
    if rows > 3:
        assert not np.isfinite(got[3]).any()
        keep = [r for r in range(rows) if r not in (0, 3)]
        P.close(got[keep], v[keep] @ w.values().T, R.product_bound(v[keep], w.values()), "f32")


def test_not_finite_scales(iam, ctx):
    rng = np.random.default_rng(5)
    w = R.random_weights(rng, 40, 300, 64, False)
    m = packed(iam, ctx, w)
    words, scale, x = rows_of(rng, 3, 300, "int8")
    scale[1] = np.nan
    got = product(ctx, m, words, scale, "int8", "f32")
    m.free()
    assert np.isnan(got[1]).all()
    P.close(got[[0, 2]], x[[0, 2]] @ w.values().T, R.product_bound(x[[0, 2]], w.values()), "f32")


@pytest.mark.parametrize("rows", [1, 6, 150])
def test_calls_repeat(iam, ctx, rows):
    rng = np.random.default_rng(6)
    w = R.random_weights(rng, 500, 3000, 128, True)
    m = packed(iam, ctx, w)
    words = rows_of(rng, rows, 3000, "f32")[0]
    first = product(ctx, m, words, None, "f32", "f32")
    for _ in range(3):
        assert np.array_equal(first, product(ctx, m, words, None, "f32", "f32"))
    m.free()


@pytest.mark.parametrize("out,inp,group,zeros", [(1, 1, 32, False), (17, 33, 32, True), (40, 513, 64, True), (33, 1100, 128, False), (16, 512, 128, True)])
def test_layout_and_read(iam, ctx, out, inp, group, zeros):
    rng = np.random.default_rng(out)
    w = R.random_weights(rng, out, inp, group, zeros)
    m = packed(iam, ctx, w)
    for part, want in zip(m.parts, R.layout(w)):
        assert np.array_equal(part.read(), want.reshape(-1).view(np.uint8))
    d = ctx.empty(out * inp, np.float32)
    m.read(0, out, d)
    assert np.array_equal(d.read().reshape(out, inp), w.values())
    if out > 20:
        m.read(18, 2, d)
        assert np.array_equal(d.read()[:2 * inp].reshape(2, inp), w.values()[18:20])
    m.free()
    d.free()


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("out,inp,group,stride", [(20, 300, 32, 0), (33, 1029, 128, 1031), (1, 5, 64, 0)])
def test_quantize(iam, ctx, out, inp, group, stride, zeros, type):
    rng = np.random.default_rng(inp)
    x = rng.normal(0, 1, (out, inp))
    x[0, :group] = 0
    if out > 2:
        x[2] = np.abs(x[2])
        x[1] = -np.abs(x[1])
        x[-1, 7] = 3e4
    words, v = P.to_type(x, type)
    flat = np.zeros((out, stride or inp), words.dtype)
    flat[:, :inp] = words
    d = ctx.upload(flat)
    m = iam.Q4Matrix(ctx, out, inp, group, zeros=zeros)
    m.quantize(d, type, stride)
    want = R.quantize(v, group, zeros)
    for part, p in zip(m.parts, R.layout(want)):
        assert np.array_equal(part.read(), p.reshape(-1).view(np.uint8))
    m.free()
    d.free()


def test_quantize_not_finite(iam, ctx):
    x = np.ones((3, 128), np.float32)
    x[0, 3], x[1, 40], x[2, 100] = np.inf, np.nan, 3e38
    d, out = ctx.upload(x), ctx.empty(3 * 128, np.float32)
    m = iam.Q4Matrix(ctx, 3, 128, 32, zeros=True)
    m.quantize(d, "f32")
    m.read(0, 3, out)
    got = out.read().reshape(3, 4, 32)
    bad = np.isnan(got).all(2)
    assert bad.tolist() == [[True, False, False, False], [False, True, False, False], [False, False, False, True]]
    # 15 times the scale, which is 1/15 rounded to fp16: off by half a step
    assert (got[~bad] == np.float32(15) * np.float32(np.float16(1 / 15))).all() and abs(15 * np.float64(np.float16(1 / 15)) - 1) <= 2.0 ** -11
    for b in (d, out, m):
        b.free()


@pytest.mark.parametrize("rows", [1, 5, 20, 140])
@pytest.mark.parametrize("type", ["f32", "bf16", "int8", "e4m3"])
def test_large_values_and_large_scales(iam, ctx, rows, type):
    """Values near the largest under zero weights, beside others whose products
    with scales of 2^15 stay small: a tile's power of two (or its scale) and
    the weights' scale together pass fp32's range."""
    rng = np.random.default_rng(9)
    w = R.random_weights(rng, 40, 640, 64, False)
    w.scale[:] = 2.0 ** 15
    w.n[:] = 8
    w.n[:, 3::64] = rng.integers(0, 16, (40, 10))
    m = packed(iam, ctx, w)
    own = np.arange(640) % 64 == 3
    if type in P.TYPES:
        words, v = P.to_type(rng.choice([-1, 1], (rows, 640)) * np.where(own, 2.0 ** 106, 2.0 ** 127), type)
        scale = None
    else:
        q = np.where(own, rng.choice([-1, 1], (rows, 640)), 100 if type == "int8" else 96.0)
        scale = np.full((rows, 5), 2.0 ** 106, np.float32)
        scale[:, 1], q[:, 128 + 3:256:64] = 2.0 ** 127, 0
        words, v = R.bytes_of(q, type), q * R.spread(scale, 128, 640)
    got = product(ctx, m, words, scale, type, "f32", 0 if scale is None else 128)
    m.free()
    # whole multiples of 2^121, at most 80 of them in any sum of an output's
    assert np.array_equal(got, v @ w.values().T)


@pytest.mark.parametrize("size", [3e-37, 1e34])
@pytest.mark.parametrize("x_group", [0, 128])
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 4, 20, 140])
def test_scales_of_rows_near_the_limits(iam, ctx, rows, type, x_group, size):
    rng = np.random.default_rng(rows)
    w = R.random_weights(rng, 70, 1000, 64, True)
    w.scale[:] = w.scale.astype(np.float64) / 10000 if size < 1 else w.scale
    words, scale, v = rows_of(rng, rows, 1000, type, x_group)
    scale = (scale * np.float64(size)).astype(np.float32)
    v = R.values8(words, type) * R.spread(scale, x_group, 1000)
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, scale, type, "f32", x_group)
    m.free()
    P.close(got, v @ w.values().T, R.product_bound(v, w.values()), "f32")


EXACT = [(1, 4096, 1024), (1, 14336, 40), (1, 14336, 200), (2, 8193, 17), (3, 20000, 1500), (4, 9000, 130), (4, 70001, 16), (4, 1100, 8209), (5, 2048, 100), (5, 9000, 130),
         (6, 14336, 64), (11, 900, 12817), (33, 14336, 40), (48, 4096, 64), (64, 900, 12817), (100, 5000, 31), (150, 4096, 100), (300, 14336, 300)]


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("rows,inp,out", EXACT)
def test_every_bit_of_x(iam, ctx, rows, inp, out, type):
    """Each output takes one input alone, times a power of two, so the result is
    equal if all bits of it enter: 24 of fp32 (20 where two fp16 parts take it),
    of values within 2^-6 of their tile's largest."""
    rng = np.random.default_rng(rows + inp + out)
    group, zeros = (32, 64, 128)[(rows + out) % 3], rows % 2 == 0
    bits = 24 if rows <= 4 else 20
    x = rng.integers(2 ** (bits - 6), 2 ** bits, (rows, inp)) | 1
    x = x * rng.choice([-1.0, 1.0], x.shape) * np.repeat(np.exp2(rng.integers(-5, 6, -(-inp // 128)) * (1 if type == "f16" else 6) - bits), 128)[:inp]
    words, v = P.to_type(x, type)
    w = R.random_weights(rng, out, inp, group, zeros)
    w.scale[:] = np.exp2(rng.integers(-3, 4, w.scale.shape))
    w.n[:] = 8 if not zeros else np.repeat(np.clip(w.zero, 1, 14), group, 1)[:, :inp]
    if zeros:
        w.zero[:] = np.clip(w.zero, 1, 14)
    at, sign = rng.integers(0, inp, out), rng.choice([-1, 1], out)
    w.n[np.arange(out), at] += sign
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, None, type, "f32")
    m.free()
    assert np.array_equal(got, v[:, at] * sign * w.scale.astype(np.float64)[np.arange(out), at // group])


@pytest.mark.parametrize("size", [1e-28, 2e-30])
@pytest.mark.parametrize("rows", [1, 4, 5, 20, 140])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_tiny_values(iam, ctx, rows, type, size):
    """Around the size from which on values have a power of their own."""
    rng = np.random.default_rng(10)
    w = R.random_weights(rng, 40, 640, 64, rows % 2 == 0)
    words, v = P.to_type(rng.normal(0, 1, (rows, 640)) * size * np.repeat([1, 0.3, 2, 0.1, 5], 128), type)
    m = packed(iam, ctx, w)
    got = product(ctx, m, words, None, type, "f32")
    m.free()
    # below 2^-102 to 22 bits of that: 2^-124 a value
    room = R.product_bound(v, w.values()) + 2.0 ** -124 * np.abs(w.values()).sum(1)
    P.close(got, v @ w.values().T, room, "f32")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,inp,out,type", [(1, 1100, 8209, "f32"), (4, 700, 8209, "f32"), (5, 1100, 8209, "f32"), (5, 700, 8225, "bf16"), (3, 1540, 8240, "e4m3"), (16, 1100, 8209, "int8"),
                                               (7, 700, 12817, "f16"), (20, 900, 12833, "f32"), (33, 700, 12817, "f32"), (64, 700, 12801, "bf16"), (40, 1100, 12817, "e4m3")])
def test_strips_that_share_a_workgroup(iam, ctx, rows, inp, out, type, group, zeros):
    """Matrices of so many rows that a workgroup takes several strips: inputs that
    end inside a chunk, the last workgroup short of strips."""
    check(iam, ctx, np.random.default_rng(group + rows), rows, inp, out, group, zeros, type, "f32")


@pytest.mark.parametrize("unit", [2.0 ** -149, 2.0 ** -126])
@pytest.mark.parametrize("x_group", [0, 128])
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 4, 20, 140])
@pytest.mark.parametrize("zeros", [False, True])
def test_smallest_scales_of_rows(iam, ctx, rows, type, x_group, unit, zeros):
    """Scales of a few of the smallest numbers: whole multiples of 2^10 units, below
    640 * 15 * 15 * 7 < 2^21 of them, which fp32 holds."""
    rng = np.random.default_rng(rows)
    w = R.random_weights(rng, 70, 640, 64, zeros)
    w.scale[:] = 2.0 ** 10
    q = rng.integers(-15, 16, (rows, 640)).astype(np.float64)
    scale = (rng.integers(1, 8, (rows, 5 if x_group else 1)) * unit).astype(np.float32)
    m = packed(iam, ctx, w)
    got = product(ctx, m, R.bytes_of(q, type), scale, type, "f32", x_group)
    m.free()
    assert np.array_equal(got, (q * R.spread(scale, x_group, 640)) @ w.values().T)


def test_refusals(iam, ctx):
    m = iam.Q4Matrix(ctx, 40, 300, 64)
    z = iam.Q4Matrix(ctx, 40, 300, 64, zeros=True)
    n, s, zero = ctx.empty(40 * 150, np.uint8), ctx.empty(40 * 5, np.uint16), ctx.empty(40 * 5, np.uint8)
    x, y, xs = ctx.empty(4 * 300, np.float32), ctx.empty(4 * 40, np.float32), ctx.empty(4 * 3, np.float32)
    m.pack(n, s)
    z.pack(n, s, zero)
    ok = dict(x=x, type="f32", n_rows=4, y=y, y_type="f32")
    m.mul(**ok)
    m.mul(**dict(ok, n_rows=0))
    m.mul(**dict(ok, type="int8", x_scale=xs, x_group=128))
    refused = [lambda: m.pack(n, s, zero), lambda: z.pack(n, s), lambda: m.pack(None, s), lambda: m.pack(n, s.ptr + 2), lambda: m.pack(n.ptr + 1, s),
               lambda: m.pack(m.parts[0], s), lambda: m.quantize(x, "f32"), lambda: m.quantize(None), lambda: m.read(0, 41, x), lambda: m.read(-1, 2, x),
               lambda: m.read(41, 0, x), lambda: m.read(0, 5, x), lambda: m.read(0, 1, m.parts[0])]
    for bad in (dict(x=None), dict(y=None), dict(n_rows=-1), dict(n_rows=5), dict(x_scale=xs), dict(type="int8"), dict(x_group=128),
                dict(type="int8", x_scale=xs, x_group=64), dict(type="int8", x_scale=xs.ptr + 4, x_group=128), dict(x_stride=299), dict(y_stride=39),
                dict(x_stride=301), dict(y_stride=41), dict(x=x.ptr + 2, n_rows=1), dict(y=x), dict(y=m.parts[0]), dict(n_rows=(1 << 22) + 1),
                dict(x_stride=1 << 40)):
        refused.append(lambda bad=bad: m.mul(**dict(ok, **bad)))
    for call in refused:
        with pytest.raises(iam.IamError) as e:
            call()
        assert e.value.code == iam.IAM_E_INVALID
    for field, v in (("numbers", 0), ("numbers", m.desc.numbers + 8), ("scales", m.desc.scales + 2), ("zeros", m.desc.scales), ("out_dim", 60), ("in_dim", 0), ("group", 48)):
        was = getattr(m.desc, field)
        setattr(m.desc, field, v)
        with pytest.raises(iam.IamError) as e:
            m.mul(**ok)
        assert e.value.code == iam.IAM_E_INVALID, field
        setattr(m.desc, field, was)
    m.mul(**ok)
    for b in (m, z, n, s, zero, x, y, xs):
        b.free()
