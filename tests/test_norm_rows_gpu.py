"""The rows' norm with the residual's addition, in float types and in 8 bits
(through libiam.so), against float64."""
import numpy as np
import pytest

import plain64 as P
import plain_rows as R

pytestmark = pytest.mark.gpu

EPS = 1e-5
GUARD = 16


class Rows:
    """Rows `stride` values apart between guards, on the device."""

    def __init__(self, ctx, words, stride=0, fill=77):
        self.rows, self.dim = words.shape
        self.stride, self.dt, self.fill = stride or self.dim, words.dtype, fill
        flat = np.full(self.rows * self.stride + 2 * GUARD, fill, words.dtype)
        flat[GUARD:-GUARD].reshape(self.rows, self.stride)[:, :self.dim] = words
        self.buf = ctx.upload(flat)
        self.ptr = self.buf.ptr + GUARD * words.dtype.itemsize

    def read(self):
        got = self.buf.read()
        body = got[GUARD:-GUARD].reshape(self.rows, self.stride)
        assert (got[:GUARD] == self.fill).all() and (got[-GUARD:] == self.fill).all() and (body[:, self.dim:] == self.fill).all()
        return body[:, :self.dim]

    def free(self):
        self.buf.free()


def blank(ctx, rows, dim, type, stride=0):
    dt = np.uint8 if type in R.LARGEST else P.storage(type)
    return Rows(ctx, np.full((rows, dim), 77, dt), stride)


def run(ctx, x, type, r=None, r_type="f32", gain=None, out_type="f32", group=0, strides=(0, 0, 0), keep=True, in_place=False, eps=EPS):
    """(float64 x, h kept, y or (scales, bytes)) of the float64 rows x, r."""
    rows, dim = x.shape
    xw, xv = P.to_type(x, type)
    dx = Rows(ctx, xw, strides[0])
    dr = rv = dsum = None
    if r is not None:
        rw, rv = P.to_type(r, r_type)
        dr = Rows(ctx, rw, strides[1])
    if keep:
        dsum = dr if in_place and dr is not None else blank(ctx, rows, dim, r_type if r is not None else type, strides[1])
    out = dx if in_place and out_type == type else blank(ctx, rows, dim, out_type, strides[2])
    eight = out_type in R.LARGEST
    groups = -(-dim // group) if group else 1
    ds = ctx.upload(np.full(rows * groups + 2, 7.25, np.float32)) if eight else None
    dg = ctx.upload(gain.astype(np.float16)) if gain is not None else None
    ctx.rmsnorm_rows(dx.ptr, type, rows, dim, dg, eps, out.ptr, out_type, residual=dr and dr.ptr, residual_type=r_type, sum=dsum and dsum.ptr,
                     scale=ds.ptr + 4 if eight else None, group=group, x_stride=strides[0], residual_stride=strides[1],
                     out_stride=strides[0] if out is dx else strides[2])
    h = P.from_bits(dsum.read(), r_type if r is not None else type) if keep else None
    if eight:
        s = ds.read()
        assert s[0] == 7.25 and s[-1] == 7.25
        scale = s[1:-1].reshape(rows, groups)
        y = (scale, out.read().copy())
        back = ctx.empty(rows * dim, np.float32)
        ctx.rows8_read(out.ptr, out_type, rows, dim, ds.ptr + 4, back, group=group, stride=strides[2])
        with np.errstate(invalid="ignore"):
            want = R.values8(y[1], out_type).astype(np.float32) * R.spread(scale, group, dim).astype(np.float32)
        assert np.array_equal(back.read().reshape(rows, dim), want, equal_nan=True)
        back.free()
    else:
        y = P.from_bits(out.read(), out_type)
    for b in {id(b): b for b in (dx, dr, dsum, out, ds, dg) if b is not None}.values():
        b.free()
    return xv, rv, h, y


def check(ctx, x, type, r=None, r_type="f32", gain=None, out_type="f32", group=0, keep=True, **kw):
    xv, rv, h, y = run(ctx, x, type, r, r_type, gain, out_type, group, keep=keep, **kw)
    g = None if gain is None else gain.astype(np.float16)
    want_h, want = R.norm(xv, rv, r_type, g, kw.get("eps", EPS))
    if keep:
        assert np.array_equal(h, want_h)
    if out_type in P.TYPES:
        # fp64 throughout: one rounding, and fp64's own (2^-44 and less)
        P.close(y, want, np.abs(want) * 2.0 ** -44, out_type)
    else:
        scale, q = R.to_eight(want, out_type, group)
        # scales are fp64 quotients rounded once: equal but where one lies
        # within 2^-44 of a border of fp32's (2^-24 apart)
        assert np.array_equal(y[0], scale)
        assert np.array_equal(y[1], R.bytes_of(q, out_type) * (q != 0) | (y[1] & (q == 0) * 0x80))
        assert (R.values8(y[1], out_type) == q).all()


def rows_of(rng, rows, dim):
    return rng.normal(0, 1, (rows, dim)) * np.where(rng.random(dim) < 0.02, 12, 1)


@pytest.mark.parametrize("out_type", R.ROW_TYPES)
@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 4096), (3, 1), (2, 127), (5, 129), (40, 5001), (9, 8192), (300, 64), (2, 20000), (1, 70001), (600, 256), (17, 2047)])
def test_rows(ctx, rows, dim, type, out_type):
    rng = np.random.default_rng(rows + dim)
    k = rows + dim + P.TYPES.index(type) + R.ROW_TYPES.index(out_type)
    r = rows_of(rng, rows, dim) if k % 3 else None
    r_type = "f32" if k % 3 == 1 else type
    gain = 1 + rng.normal(0, 0.2, dim) if k % 4 else None
    check(ctx, rows_of(rng, rows, dim), type, r, r_type, gain, out_type, 128 * (k // 2 % 2) if out_type in R.LARGEST else 0, keep=k % 5 != 0)


@pytest.mark.parametrize("out_type,group", [("f32", 0), ("int8", 0)])
def test_more_rows_than_a_launch(ctx, out_type, group):
    rng = np.random.default_rng(8)
    rows, dim = (1 << 20) + 5, 2
    check(ctx, rows_of(rng, rows, dim), "f32", rows_of(rng, rows, dim), "f32", np.array([0.5, 2.0]), out_type, group, strides=(3, 2, 4))


@pytest.mark.parametrize("type,r_type,out_type,strides", [("f32", "f32", "int8", (5001, 4999, 5003)), ("f16", "f16", "f16", (4998, 4997, 5005)), ("bf16", "f32", "e4m3", (5008, 5008, 5008)),
                                                          ("bf16", "bf16", "bf16", (4996, 5000, 5001)), ("f16", "f32", "int8", (5000, 5000, 5000))])
def test_strides(ctx, type, r_type, out_type, strides):
    rng = np.random.default_rng(1)
    check(ctx, rows_of(rng, 6, 4996), type, rows_of(rng, 6, 4996), r_type, 1 + rng.normal(0, 0.2, 4996), out_type, 128 if out_type == "e4m3" else 0, strides=strides)


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("dim", [77, 4096, 9000, 40000])
def test_in_place(ctx, type, dim):
    rng = np.random.default_rng(dim)
    check(ctx, rows_of(rng, 4, dim), type, rows_of(rng, 4, dim), type, None, type, in_place=True)
    check(ctx, rows_of(rng, 4, dim), type, rows_of(rng, 4, dim), "f32", None, "int8", in_place=True)


@pytest.mark.parametrize("out_type", ["f32", "int8", "e4m3"])
def test_sizes_of_values(ctx, out_type):
    """Zeros, tiny, huge; eps on its own, and no eps."""
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (6, 300))
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3, 1:] = 0
    x[4, 128:256] = 0
    group = 128 if out_type != "f32" else 0
    check(ctx, x, "f32", None, out_type=out_type, group=group)
    check(ctx, x[1:], "f32", None, out_type=out_type, group=group, eps=0.0)


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("out_type", ["f32", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [300, 4096, 30000])
def test_not_finite(ctx, out_type, group, dim):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (5, dim))
    x[1, 200], x[2, 7] = np.nan, np.inf
    x[3] = 0
    if out_type in P.TYPES:
        y = run(ctx, x, "f32", out_type=out_type)[3]
        assert np.isnan(y[1]).all() and np.isnan(y[2, 7]) and (np.delete(y[2], 7) == 0).all() and np.isfinite(y[[0, 3, 4]]).all()
        return
    scale, b = run(ctx, x, "f32", out_type=out_type, group=group)[3]
    assert np.isnan(scale[1]).all() and (b[1] == 0).all()
    where = np.isnan(scale[2])
    assert where[0] and where.sum() == 1 and (b[2] & 0x7f == 0).all() and (scale[3] == 0).all() and (b[3] == 0).all()
    assert np.isfinite(scale[[0, 4]]).all()


def test_ties_of_the_numbers(ctx):
    """A gain that makes y whole and half steps of its scale: to even."""
    for out_type, steps in (("int8", np.array([127, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -126.5])), ("e4m3", np.array([448, 2.0 ** -10, 3 * 2.0 ** -10, 17, 19, 1.0625, -1.1875, 432]))):
        x = np.ones((1, 8))
        scale, b = run(ctx, x, "f32", gain=steps, out_type=out_type, eps=0.0)[3]
        assert scale[0, 0] == 1
        assert np.array_equal(R.values8(b, out_type)[0], P.numbers(steps, out_type))


@pytest.mark.parametrize("out_type", ["int8", "e4m3"])
@pytest.mark.parametrize("group", [0, 128])
def test_subnormal_scales(ctx, out_type, group):
    """Groups whose scale is a few of the smallest fp32 numbers: quotients up to
    1.5 times the largest number."""
    rng = np.random.default_rng(4)
    x = np.zeros((12, 260))
    for r, top in enumerate((60, 64, 100, 190, 200, 300, 600, 671, 672, 1000, 1500, 5000)):
        x[r] = rng.integers(-top, top + 1, 260)
        x[r, 5], x[r, 130] = top, -top
    # eps 1 is all of the root: y = x
    check(ctx, x * 2.0 ** -149, "f32", out_type=out_type, group=group, eps=1.0)


@pytest.mark.parametrize("out_type", P.TYPES)
@pytest.mark.parametrize("dim", [60, 70001])
def test_infinite_gains(ctx, out_type, dim):
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (3, dim))
    gain = np.ones(dim)
    gain[3:40:2], gain[4:40:4] = np.inf, -np.inf
    y = run(ctx, x, "f32", gain=gain, out_type=out_type)[3]
    at = np.isinf(gain)
    assert np.array_equal(y[:, at], np.sign(x[:, at]) * gain[at]) and np.isfinite(y[:, ~at]).all()


def test_refused_overlaps_of_inputs(iam, ctx):
    """x and the residual may be one array, but then neither is written over."""
    x, s, out = (ctx.empty(4 * 100, np.float32) for _ in range(3))
    g = ctx.empty(100, np.uint16)
    ok = dict(x=x, type="f32", n_rows=2, dim=100, gain=g, eps=EPS, out=out, out_type="f32", residual=x, residual_type="f32", sum=s)
    ctx.rmsnorm_rows(**ok)
    for bad in (dict(sum=x), dict(sum=x, x_stride=200), dict(out=x), dict(out=x, residual_stride=200), dict(sum=x, type="f16", x_stride=200), dict(out=x, out_type="f16", type="f16")):
        with pytest.raises(iam.IamError) as e:
            ctx.rmsnorm_rows(**dict(ok, **bad))
        assert e.value.code == iam.IAM_E_INVALID, bad
    for b in (x, s, out, g):
        b.free()


def test_refusals(iam, ctx):
    x, r, s, out = (ctx.empty(4 * 100, np.float32) for _ in range(4))
    g, sc = ctx.empty(100, np.uint16), ctx.empty(4, np.float32)
    ok = dict(x=x, type="f32", n_rows=4, dim=100, gain=g, eps=EPS, out=out, out_type="f32", residual=r, residual_type="f32", sum=s)
    eight = dict(ok, out_type="int8", scale=sc)
    ctx.rmsnorm_rows(**ok)
    ctx.rmsnorm_rows(**eight)
    ctx.rmsnorm_rows(**dict(ok, n_rows=0))
    ctx.rmsnorm_rows(**dict(ok, sum=r, out=x))
    for base, bad in ((ok, dict(x=None)), (ok, dict(out=None)), (ok, dict(n_rows=5)), (ok, dict(n_rows=-1)), (ok, dict(dim=0)), (ok, dict(dim=101)), (ok, dict(eps=-1.0)),
                      (ok, dict(eps=float("nan"))), (ok, dict(scale=sc)), (ok, dict(group=128)), (eight, dict(scale=None)), (eight, dict(group=64)), (eight, dict(out=x)),
                      (eight, dict(scale=out)), (ok, dict(out=r)), (ok, dict(sum=x)), (ok, dict(sum=out)), (ok, dict(residual_type="f16")), (ok, dict(x_stride=99)),
                      (ok, dict(out_stride=101)), (ok, dict(out=x, out_stride=100, x_stride=0, type="f32", out_type="f16")), (ok, dict(x=x.ptr + 2, n_rows=1)),
                      (ok, dict(gain=g.ptr + 2)), (ok, dict(residual_stride=101)), (eight, dict(dim=100, n_rows=4, scale=sc.ptr + 4))):
        with pytest.raises(iam.IamError) as e:
            ctx.rmsnorm_rows(**dict(base, **bad))
        assert e.value.code == iam.IAM_E_INVALID, bad
    ok = dict(x=out, type="int8", n_rows=4, dim=100, scale=sc, out=x)
    ctx.rows8_read(**ok)
    for bad in (dict(x=None), dict(scale=None), dict(out=None), dict(type="f32"), dict(n_rows=5), dict(dim=101), dict(group=64), dict(stride=99), dict(out=out), dict(out=sc)):
        with pytest.raises(iam.IamError):
            ctx.rows8_read(**dict(ok, **bad))
    for b in (x, r, s, out, g, sc):
        b.free()
