"""Token log probabilities, entropy and alternatives (through libiam.so)
against float64."""
import numpy as np
import pytest

import plain64 as P

pytestmark = pytest.mark.gpu


def run(ctx, x, type, targets, k, stride=0, first=0, entropy=True):
    """x [rows][vocab]: (values, logprob, entropy, ids, tops)."""
    rows, vocab = x.shape
    w, val = P.to_type(x, type)
    s = stride or vocab
    flat = np.full(first + rows * s, 99, w.dtype)         # what lies between is larger than the logits
    flat[first:].reshape(rows, s)[:, :vocab] = w
    dx, dt = ctx.upload(flat), ctx.upload(np.asarray(targets, np.int32))
    guard = np.full(rows + 2, 7.25, np.float32)
    dl, de = ctx.upload(guard), ctx.upload(guard)
    di, dp = ctx.upload(np.full(rows * k + 2, 77, np.int32)), ctx.upload(np.full(rows * k + 2, 7.25, np.float32))
    ctx.token_logprobs(dx.ptr + first * w.itemsize, type, rows, vocab, dt, dl.ptr + 4, de.ptr + 4 if entropy else None, k,
                       di.ptr + 4 if k else None, dp.ptr + 4 if k else None, stride=stride)
    l, e, i, p = dl.read(), de.read(), di.read(), dp.read()
    for g, v in ((l, 7.25), (e, 7.25), (i, 77), (p, 7.25)):
        assert g[0] == v and g[-1] == v
    for b in (dx, dt, dl, de, di, dp):
        b.free()
    return val, l[1:-1], e[1:-1], i[1:-1].reshape(rows, k), p[1:-1].reshape(rows, k)


def check(ctx, x, type, targets, k, **kw):
    val, l, e, ids, top = run(ctx, x, type, targets, k, **kw)
    rows, vocab = x.shape
    targets = np.asarray(targets)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = val.max(1, keepdims=True)
        d = val - m
        p = np.exp(d)
        z = p.sum(1)
        lz = np.log(z)
        w = p / z[:, None]
        h = lz - np.where(p > 0, w * np.where(p > 0, d, 0), 0).sum(1)
        # (x - m) - log z: m + log z first would lose log z to a huge m in
        # float64 too (-3.4e38 + 8.3 is -3.4e38)
        log_p = d - lz[:, None]
        # an exponential's argument is two roundings off (2^-23 |d|), the
        # instruction 2^-22; a thread's terms of s are up to 32 fp32 additions
        term = 2.0 ** -22 * (1 + np.where(p > 0, np.abs(d), 0))
        dz = (w * np.where(p > 0, term, 0)).sum(1) + 2.0 ** -40
        dh = dz + (w * np.where(p > 0, np.abs(d) * (2 * term + 34 * 2.0 ** -24), 0)).sum(1) + np.abs(h - lz) * dz
    there = (targets >= 0) & (targets < vocab)
    want = np.where(there, log_p[np.arange(rows), np.where(there, targets, 0)], 0.0)
    def near(got, want, b):
        with np.errstate(over="ignore", invalid="ignore"):
            past = np.isinf(want.astype(np.float32))     # -6e38 is -inf in fp32
            return np.where(past, got == want.astype(np.float32), np.abs(got - want) <= b + 2.0 ** -24 * (np.abs(want) + b) + 2.0 ** -149)

    assert near(l, want, dz).all(), (l, want)
    if kw.get("entropy", True):
        assert near(e, h, dh).all(), (e, h)
        assert (e >= 0).all()
    if k:
        order = np.argsort(-val, axis=1, kind="stable")[:, :k]
        assert np.array_equal(ids, order)
        assert near(top, np.take_along_axis(log_p, order, 1), dz[:, None]).all()


def logits(rng, rows, vocab):
    x = rng.normal(0, 2, (rows, vocab))
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 8
    return x


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("k", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (3, 64), (2, 131072), (40, 8193), (5, 2047), (700, 999), (9, 8192)])
def test_rows(ctx, type, k, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    check(ctx, logits(rng, rows, vocab), type, rng.integers(0, vocab, rows), k)


@pytest.mark.parametrize("type", P.TYPES)
def test_many_rows(ctx, type):
    rng = np.random.default_rng(1)
    check(ctx, logits(rng, 2500, 8300), type, rng.integers(0, 8300, 2500), 3)


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("k", [0, 1, 33, 64])
@pytest.mark.parametrize("rows,vocab", [(300, 16000), (1100, 8192), (90, 32001)])
def test_many_values(ctx, type, k, rows, vocab):
    """Large chunks: one, two and several of them, segments of one and more."""
    rng = np.random.default_rng(rows)
    check(ctx, logits(rng, rows, vocab), type, rng.integers(0, vocab, rows), k)


@pytest.mark.parametrize("vocab", [1, 2, 7])
def test_tiny_vocabularies(ctx, vocab):
    rng = np.random.default_rng(vocab)
    check(ctx, rng.normal(0, 1, (4, vocab)), "f32", [0, vocab - 1, vocab, -1], vocab)


@pytest.mark.parametrize("type", P.TYPES)
def test_strides_and_alignment(ctx, type):
    rng = np.random.default_rng(2)
    x = logits(rng, 6, 5001)
    for stride, first in ((5001, 1), (5003, 0), (6000, 3), (5008, 8)):
        check(ctx, x, type, rng.integers(0, 5001, 6), 7, stride=stride, first=first)


def test_padding_targets_and_no_entropy(ctx):
    rng = np.random.default_rng(3)
    check(ctx, logits(rng, 5, 3001), "f32", [-1, 3001, 2 ** 31 - 1, -2 ** 31, 4], 2, entropy=False)


@pytest.mark.parametrize("k", [1, 5, 64])
@pytest.mark.parametrize("vocab", [3000, 33000])
def test_ties_and_orders(ctx, k, vocab):
    """All equal, rising, falling, few distinct values, zeros of both signs."""
    rng = np.random.default_rng(4)
    x = np.zeros((6, vocab))
    x[1] = np.arange(vocab) / 64.0
    x[2] = -np.arange(vocab) / 64.0
    x[3] = rng.integers(0, 3, vocab)
    x[4] = np.where(rng.integers(0, 2, vocab), 0.0, -0.0)
    x[5, :] = -50
    x[5, vocab - k:] = 1.0
    check(ctx, x, "f32", [0, vocab - 1, 0, 5, 6, vocab - 1], k)


def test_nearly_certain_and_far_values(ctx):
    """log p near 0 keeps its digits; huge, tiny and lowest values."""
    x = np.full((5, 4000), -20.0)
    x[0, 7] = 5.0
    x[1, 3999] = 60.0
    x[2] = np.linspace(-3e38, 3e38, 4000)
    x[3] = np.finfo(np.float32).min
    x[3, 11] = 0
    x[4] = np.finfo(np.float32).min
    check(ctx, x, "f32", [7, 3999, 0, 12, 2], 4)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("k", [0, 4])
@pytest.mark.parametrize("rows,vocab", [(1, 4096), (1, 70000), (400, 16384), (300, 40003)])
def test_maxima_farther_apart_than_the_largest_number(ctx, type, k, rows, vocab):
    """-3e38 and 3e38 in one row: their difference is past fp32's range, and
    the maxima that a wave, the waves, or a row's segments join lie so far
    apart.  By halves of a wave's loads, of a chunk, of a row, the low ones first
    or last, one high value alone, in turn."""
    x = np.full((rows, vocab), -3e38)
    i = np.arange(vocab)
    for r in range(rows):
        high = (i >= vocab // 2, i < vocab // 2, i // 2048 % 2 == 1, i // 1024 % 2 == 0, i // 256 % 2 == 1, i // 4096 % 2 == 1,
                i // 8192 % 2 == 1, i % 2 == 1, i == vocab - 1, i == 0)[r % 10 if rows > 1 else 0]
        x[r, high] = 3e38
    check(ctx, x, type, i[:rows] if rows > 1 else [vocab - 1], k)


@pytest.mark.parametrize("vocab", [50, 20000])
def test_masked_and_not_finite(ctx, vocab):
    rng = np.random.default_rng(5)
    x = logits(rng, 7, vocab)
    x[0, 5:] = -np.inf
    x[1] = -np.inf
    x[2, 9] = np.nan
    x[3, 9] = np.inf
    x[4] = np.nan
    x[5, :] = -np.inf
    x[5, vocab - 1] = 3.0
    val, l, e, ids, top = run(ctx, x, "f32", [1, 0, 3, 3, 0, vocab - 1, 2], 6)
    f = np.isfinite(x[0])
    lse = np.log(np.exp(val[0, :5] - val[0, :5].max()).sum()) + val[0, :5].max()
    assert abs(l[0] - (val[0, 1] - lse)) <= 2.0 ** -21 * (1 + abs(lse)) + 2.0 ** -24 * abs(l[0])
    assert np.array_equal(ids[0], np.argsort(-val[0], kind="stable")[:6]) and top[0, 5] == -np.inf
    assert np.isneginf(l[1]) and e[1] == 0 and ids[1].tolist() == list(range(6)) and np.isneginf(top[1]).all()
    for r in (2, 3, 4):
        assert np.isnan(l[r]) and np.isnan(e[r]) and np.isnan(top[r]).all()
    assert ids[3, 0] == 9 and 9 not in ids[2] and ids[4].tolist() == list(range(6))
    assert l[5] == 0 and e[5] == 0 and ids[5].tolist() == [vocab - 1] + list(range(5))
    assert top[5, 0] == 0 and np.isneginf(top[5, 1:]).all() and f.sum() == 5
    check(ctx, x[6:], "f32", [2], 6)


@pytest.mark.parametrize("k,low,vocab", [(5, 4, 2 ** 21), (64, 63, 2 ** 17), (64, 63, 12000), (20, 3, 300000), (2, 1, 2 ** 21)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_largest_values_in_few_places(ctx, type, k, low, vocab):
    """The largest values lie at every 64th run of 16 bytes, so that few
    threads see them all; with ties in 16 bits."""
    rng = np.random.default_rng(k)
    x = rng.normal(0, 1, (2, vocab))
    x += np.where(np.arange(vocab) // (4 if type == "f32" else 8) % 64 < low, 20.0, 0.0)
    check(ctx, x, type, [1, vocab - 1], k)


@pytest.mark.parametrize("k,vocab,numbers", [(64, 100000, 3), (5, 2 ** 20, 4), (8, 70, 0), (64, 2000, 63), (1, 9000, 0)])
def test_fewer_numbers_than_alternatives(ctx, k, vocab, numbers):
    """NaN but for a few values: those in order, then the first NaN."""
    rng = np.random.default_rng(vocab)
    x = np.full((3, vocab), np.nan)
    for r in range(3):
        at = np.sort(rng.choice(vocab, numbers, replace=False))
        x[r, at] = rng.integers(0, 2, numbers)
        if r == 2:
            x[r, at] = -np.inf
    val, l, e, ids, top = run(ctx, x, "f32", [0, 1, 2], k)
    for r in range(3):
        want = np.lexsort((np.arange(vocab), np.where(np.isnan(x[r]), 0, -np.nan_to_num(x[r], neginf=-9)), np.isnan(x[r])))
        assert np.array_equal(ids[r], want[:k])
    assert np.isnan(l).all() and np.isnan(top).all()


def test_very_many_rows(ctx):
    """More rows than one launch takes, without and with alternatives."""
    rng = np.random.default_rng(11)
    x = rng.normal(0, 2, (2 ** 22 + 77, 3)).astype(np.float32)
    check(ctx, x, "f32", rng.integers(0, 3, len(x)), 0)
    check(ctx, x, "f16", rng.integers(0, 3, len(x)), 2)


def test_calls_repeat(ctx):
    rng = np.random.default_rng(6)
    a, b = logits(rng, 2, 100000), logits(rng, 300, 9000)
    first = run(ctx, a, "bf16", [1, 2], 20)[1:], run(ctx, b, "f32", np.arange(300), 3)[1:]
    for _ in range(4):
        again = run(ctx, a, "bf16", [1, 2], 20)[1:], run(ctx, b, "f32", np.arange(300), 3)[1:]
        for x, y in zip(first, again):
            assert all(np.array_equal(u.view(np.uint32), w.view(np.uint32)) for u, w in zip(x, y))


def test_logits_of_the_model(iam, ctx):
    """The greedy token of a decode step is its likeliest alternative."""
    cfg = iam.ModelConfig(1, 4096, 4096, 32, 8, 128, 1008, 8, 10000.0, 1e-5)
    m = iam.Model(ctx, cfg)
    m.synthesize(0)
    dl = ctx.empty(1008, np.float32)
    m.forward(3, 0, 0.25, dl)
    x = dl.read()
    di, dt, dp = ctx.empty(1, np.int32), ctx.empty(4, np.int32), ctx.empty(4, np.float32)
    one = ctx.empty(1, np.float32)
    ctx.argmax(dl, 1008, di)
    ctx.token_logprobs(dl, "f32", 1, 1008, di, one, None, 4, dt, dp)
    assert dt.read()[0] == di.read()[0] == int(np.argmax(x))
    assert one.read()[0] == dp.read()[0]
    m.close()
    for b in (dl, di, dt, dp, one):
        b.free()


def test_refusals(iam, ctx):
    x, t = ctx.empty(4 * 100, np.float32), ctx.upload(np.zeros(4, np.int32))
    l, e, i, p = (ctx.empty(4 * 64, np.float32) for _ in range(4))
    good = dict(logits=x, type="f32", n_rows=4, vocab=100, targets=t, logprob=l, entropy=e, top_k=2, top_ids=i, top_logprobs=p)
    ctx.token_logprobs(**good)
    ctx.token_logprobs(**dict(good, n_rows=0))
    ctx.token_logprobs(**dict(good, top_ids=None))
    for bad in (dict(logits=None), dict(targets=None), dict(logprob=None), dict(vocab=0), dict(vocab=101), dict(n_rows=5), dict(n_rows=-1),
                dict(top_k=65), dict(top_k=-1), dict(vocab=3, top_k=4), dict(stride=99), dict(stride=101), dict(logits=x.ptr + 2, n_rows=1),
                dict(entropy=l), dict(top_ids=p), dict(logprob=x), dict(targets=l), dict(vocab=(1 << 30) + 1)):
        with pytest.raises(iam.IamError) as err:
            ctx.token_logprobs(**dict(good, **bad))
        assert err.value.code == iam.IAM_E_INVALID, bad
    for b in (x, t, l, e, i, p):
        b.free()


def test_rows_past_64_bits_are_refused(iam, ctx):
    """2^27 rows 2^39 values apart end at 2^64 bytes, as if they were one."""
    n = (1 << 27) + 1
    x, t, l = ctx.empty(16, np.float32), ctx.empty(n, np.int32), ctx.empty(n, np.float32)
    with pytest.raises(iam.IamError) as e:
        ctx.token_logprobs(x, "f32", n, 16, t, l, stride=1 << 39)
    assert e.value.code == iam.IAM_E_INVALID and "token_logprobs logits" in str(e.value)
    for b in (x, t, l):
        b.free()
