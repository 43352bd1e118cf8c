"""Verification of drafted tokens (through libiam.so) against float64."""
import numpy as np
import pytest

import plain64 as P
import plain_rows as R

pytestmark = pytest.mark.gpu


def stored(ctx, x, type, stride, first):
    """Logits [S][n][V] as rows `stride` apart, the space between larger than any."""
    S, n, V = x.shape
    w, v = P.to_type(x, type)
    st = stride or V
    flat = np.full(first + S * n * st, 0x7f7f if type == "bf16" else 60000, w.dtype)
    flat[first:].reshape(S, n, st)[:, :, :V] = w
    d = ctx.upload(flat)
    return d, d.ptr + first * w.itemsize, v


def run(ctx, target, draft, tokens, count, uniform, temperature, type="f32", draft_type="f32", draft_temperature=None, stride=0, first=0, draft_stride=0):
    S, n1, V = target.shape
    n = n1 - 1
    dt, pt, tv = stored(ctx, target, type, stride, first)
    dd = pd = dv = None
    if draft is not None:
        dd, pd, dv = stored(ctx, draft, draft_type, draft_stride, first)
    bufs = [dt, dd]
    up = lambda a, t: bufs.append(ctx.upload(np.asarray(a, t))) or bufs[-1]   # noqa: E731
    dk = up(tokens, np.int32) if n else None
    dc = up(count, np.int32) if count is not None else None
    du = up(uniform, np.float32) if uniform is not None else None
    do, da = up(np.full(S * n1 + 2, 99), np.int32), up(np.full(S + 2, 99), np.int32)
    ctx.verify_drafts(pt, type, S, n, V, dk, du, do.ptr + 4, da.ptr + 4, temperature=temperature, draft=pd, draft_type=draft_type,
                      draft_temperature=draft_temperature, count=dc, target_stride=stride, draft_stride=draft_stride)
    out, acc = do.read(), da.read()
    assert out[0] == out[-1] == acc[0] == acc[-1] == 99
    for b in bufs:
        if b is not None:
            b.free()
    return tv, dv, out[1:-1].reshape(S, n1), acc[1:-1]


def check(ctx, target, draft, tokens, count, uniform, temperature, **kw):
    tv, dv, out, acc = run(ctx, target, draft, tokens, count, uniform, temperature, **kw)
    want, want_acc = R.verify(tv, dv, tokens, count, uniform, temperature, kw.get("draft_temperature"))
    assert np.array_equal(acc, want_acc), (acc, want_acc)
    assert np.array_equal(out, want), (out, want)
    return out, acc


def made(rng, S, n, V, certain=False, noise=0.7):
    """(target, draft, tokens, uniform): the draft's logits are like the target's."""
    x = rng.normal(0, 1.5, (S, n + 1, V))
    for _ in range(4):
        x[np.arange(S)[:, None], np.arange(n + 1)[None], rng.integers(0, V, (S, n + 1))] += 6
    y = x[:, :n] + rng.normal(0, noise, (S, n, V))
    t = y.argmax(2) if certain else (y + rng.gumbel(0, 1, y.shape)).argmax(2)
    return x, None if certain else y, t, rng.random((S, n + 1)).astype(np.float32)


@pytest.mark.parametrize("type,draft_type", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.0, 2.5])
@pytest.mark.parametrize("S,n,V", [(1, 4, 32000), (16, 5, 8193), (40, 1, 257), (5, 8, 20000), (2, 3, 131072), (3, 2, 1), (4, 3, 7), (9, 0, 3000)])
def test_sequences(ctx, S, n, V, temperature, certain, type, draft_type):
    rng = np.random.default_rng(S * 10 + n + V)
    x, y, t, u = made(rng, S, n, V, certain)
    check(ctx, x, y, t, None, u, temperature, type=type, draft_type=draft_type)


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_ragged_counts(ctx, temperature):
    rng = np.random.default_rng(1)
    x, y, t, u = made(rng, 12, 6, 5000)
    check(ctx, x, y, t, [0, 1, 2, 3, 4, 5, 6, 7, -1, 6, 100, -2 ** 31], u, temperature)
    check(ctx, x, None, t, [0, 1, 2, 3, 4, 5, 6, 7, -1, 6, 100, -2 ** 31], u, temperature)


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("stride,first", [(5001, 1), (5003, 0), (5008, 8), (6000, 3)])
def test_strides(ctx, type, stride, first):
    rng = np.random.default_rng(stride)
    x, y, t, u = made(rng, 4, 3, 5001)
    for temperature in (0.7, 0.0):
        check(ctx, x, y, t, None, u, temperature, type=type, draft_type=type, stride=stride, first=first, draft_stride=stride + 2)


def test_draft_temperature(ctx):
    rng = np.random.default_rng(2)
    x, y, t, u = made(rng, 20, 4, 3001)
    check(ctx, x, y, t, None, u, 0.8, draft_temperature=1.7)
    check(ctx, x, y, t, None, u, 1e-3, draft_temperature=50.0)


def test_most_drafted_tokens(ctx):
    rng = np.random.default_rng(3)
    x, y, t, u = made(rng, 2, 64, 500, noise=0.02)
    u[0] *= 0.5
    _, acc = check(ctx, x, y, t, None, u, 1.0)
    assert acc[0] > 20
    check(ctx, x, x[:, :64].copy(), x[:, :64].argmax(2), None, u, 1.0)      # p is q: all are kept
    check(ctx, x, None, x[:, :64].argmax(2), None, u, 0.0)


@pytest.mark.parametrize("V", [9, 4000, 40000])
def test_masked_and_not_finite(ctx, V):
    rng = np.random.default_rng(4)
    x, y, t, u = made(rng, 10, 2, V)
    x[0, :, V // 2:] = -np.inf            # masked tails
    x[1, 0, :] = -np.inf                  # no distribution
    x[2, 1, 3] = np.nan
    x[3, 0, 3] = np.inf
    y[4, 0, :] = -np.inf
    y[5, 1, 1] = np.nan
    x[6, :, :] = -np.inf
    x[6, :, V - 1] = 2.0                  # one token alone
    t[6] = V - 1
    y[7] = x[7, :2]
    t[7] = x[7, :2].argmax(1)             # p is q
    t[8] = [-1, V]                        # outside the vocabulary
    t[9] = [V, 2 ** 31 - 1]
    u[:, 0] = 0.3
    for temperature in (1.0, 0.0):
        for draft in (y, None):
            check(ctx, x, draft, t, None, u, temperature)


def test_drafts_that_cannot_be(ctx):
    """q is 0 at the token (kept if p is not), p is 0 there, p - q nowhere positive."""
    x = np.full((4, 2, 50), -np.inf)
    y = np.full((4, 1, 50), -np.inf)
    x[:, :, :4], y[:, :, :4] = 0, 0
    t = np.array([[10], [2], [3], [0]])
    x[0, 0, 10] = 0
    y[1, 0, 2], x[1, 0, 2] = 0, -np.inf
    u = np.array([[0.5, 0.1], [0.0, 0.9], [0.99, 0.5], [0.99999994, 0.99999994]], np.float32)
    out, acc = check(ctx, x, y, t, None, u, 1.0)
    assert acc.tolist() == [1, 0, 1, 1]
    # the certain draft is the only token of any weight: rejected by u = 1 - 2^-24 never, so p stays
    x[:, 0, :] = -np.inf
    x[:, 0, 7] = 1
    check(ctx, x, None, np.full((4, 1), 7), None, u, 1.0)
    check(ctx, x, None, np.full((4, 1), 8), None, u, 1.0)


@pytest.mark.parametrize("V", [5, 1000, 33333])
def test_borders_of_the_random_numbers(ctx, V):
    """Weights that are powers of two: u = 0, u on the border of two tokens (the
    next one's), the largest u."""
    x = np.full((6, 1, V), -np.inf)
    at = [1, V // 2, V - 2]
    x[:, 0, at[0]], x[:, 0, at[1]], x[:, 0, at[2]] = 0, 0, np.log(2)      # 1/4, 1/4, 1/2 to 2^-54
    x[:, 0, V - 1] = -np.inf
    u = np.array([[0], [0.2499], [0.2501], [0.4999], [0.5001], [0.99999994]], np.float32)
    _, _, out, _ = run(ctx, x, None, np.zeros((6, 0)), None, u, 1.0)
    assert out[:, 0].tolist() == [at[0], at[0], at[1], at[1], at[2], at[2]]
    x[:, 0, at[2]] = 0
    x[:, 0, 0] = 0                                                          # four of 1/4: borders are exact
    u = np.array([[0], [0.25], [0.5], [0.75], [0.24999999], [0.99999994]], np.float32)
    _, _, out, _ = run(ctx, x, None, np.zeros((6, 0)), None, u, 1.0)
    assert out[:, 0].tolist() == [0, at[0], at[1], at[2], 0, at[2]]


def test_greedy_ties(ctx):
    """The first of equal logits, in 16 bits too."""
    x = np.zeros((2, 3, 9000))
    x[:, :, 5000] = x[:, :, 4000] = x[:, :, 8999] = 3
    x[1, 0, 7] = 3.001
    _, _, out, acc = run(ctx, x, None, np.array([[4000, 5000], [7, 4000]]), None, None, 0.0, type="bf16")
    assert acc.tolist() == [1, 2] and out.tolist() == [[4000, 4000, -1], [7, 4000, 4000]]
    check(ctx, x, None, np.array([[4000, 5000], [7, 4000]]), None, None, 0.0, type="f32")


def test_distribution(ctx):
    """What comes out first is distributed as p, whatever the draft: 40000
    sequences of a vocabulary of 8.  A count of a probability w is off by at most
    6 sqrt(S w (1 - w)) in all but one of 10^8 cases."""
    rng = np.random.default_rng(5)
    S, V = 40000, 8
    x, y = np.tile(rng.normal(0, 1, (1, 2, V)), (S, 1, 1)), np.tile(rng.normal(0, 1, (1, 1, V)), (S, 1, 1))
    t = (y + rng.gumbel(0, 1, y.shape)).argmax(2)
    u = rng.random((S, 2)).astype(np.float32)
    tv, _, out, acc = run(ctx, x, y, t, None, u, 1.0)
    p = R.softmax(tv[0, 0], 1.0)
    count = np.bincount(out[:, 0], minlength=V)
    assert 0.2 * S < acc.sum() < S
    assert (np.abs(count - S * p) <= 6 * np.sqrt(S * p * (1 - p))).all()


def test_calls_repeat(ctx):
    rng = np.random.default_rng(6)
    made_ = made(rng, 7, 4, 30011)
    x, y, t, u = made_
    first = run(ctx, x, y, t, None, u, 0.9)[2:]
    for _ in range(4):
        run(ctx, x[:, :, :100], None, t % 100, None, u, 0.0)
        again = run(ctx, x, y, t, None, u, 0.9)[2:]
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("stride,draft_stride", [(0, 0), (1, 3)])
@pytest.mark.parametrize("vocab", [9, 1000, 4000, 40000])
def test_rejected_where_the_distributions_are_equal(ctx, vocab, stride, draft_stride, type):
    """A token that both rows give no probability: p - q is 0 everywhere, however
    the two rows lie in memory, and the next token is drawn from p."""
    rng = np.random.default_rng(vocab)
    S, n = 24, 2
    x = rng.normal(0, 1.5, (S, n + 1, vocab))
    x[::2, :, rng.integers(0, vocab, 8)] += 6
    x[S // 2:] = np.round(x[S // 2:])                          # many equal ones
    t = np.stack([rng.permutation(vocab)[:n] for _ in range(S)])
    x[np.arange(S)[:, None], np.arange(n)[None], t] = -np.inf
    u = rng.random((S, n + 1)).astype(np.float32)
    _, acc = check(ctx, x, x[:, :n].copy(), t, None, u, 1.0, type=type, draft_type=type, stride=vocab + stride if stride else 0,
                   draft_stride=vocab + draft_stride if draft_stride else 0)
    assert (acc == 0).all()
    if type == "f32":
        # the same distributions at other temperatures
        check(ctx, x, 4 * P.to_type(x[:, :n], "f32")[1], t, None, u, 0.7, draft_temperature=2.8, stride=vocab + stride if stride else 0)


@pytest.mark.parametrize("vocab,span", [(600, 512), (2041, 300), (9000, 9000)])
def test_borders_behind_masked_tokens(ctx, vocab, span):
    """Equal logits among masked ones and random numbers on their borders: by
    rounding the token on one side of the border or the other, and no third."""
    rng = np.random.default_rng(1)
    x, u, sides = [], [], []
    for count in (3, 6, 12, 20, 24, 28, 40, 48, 56, 80, 88, 96, 100, 200):
        for _ in range(8):
            at = np.sort(rng.choice(span, count, replace=False))
            row = np.full(vocab, -np.inf)
            row[at] = 1.5
            for j in range(1, count):
                if float(np.float32(j / count)) * count == j:
                    x.append(row)
                    u.append(j / count)
                    sides.append((at[j - 1], at[j]))
    x, S = np.array(x)[:, None], len(x)
    out = run(ctx, x, None, np.zeros((S, 0)), None, np.array(u, np.float32)[:, None], 1.0)[2][:, 0]
    assert ((out[:, None] == np.array(sides)).any(1)).all()


def test_refusals(iam, ctx):
    x, y = ctx.empty(2 * 4 * 100, np.float32), ctx.empty(2 * 3 * 100, np.float32)
    t, u, c, o, a = ctx.upload(np.zeros(6, np.int32)), ctx.upload(np.zeros(8, np.float32)), ctx.upload(np.zeros(2, np.int32)), ctx.empty(8, np.int32), ctx.empty(2, np.int32)
    x.zero()
    y.zero()
    ok = dict(target=x, type="f32", n_seq=2, n_draft=3, vocab=100, tokens=t, uniform=u, out=o, accepted=a, temperature=1.0, draft=y, count=c)
    ctx.verify_drafts(**ok)
    ctx.verify_drafts(**dict(ok, n_seq=0))
    ctx.verify_drafts(**dict(ok, n_draft=0, tokens=None))
    ctx.verify_drafts(**dict(ok, temperature=0.0, uniform=None, draft=None))
    for bad in (dict(target=None), dict(out=None), dict(accepted=None), dict(tokens=None), dict(uniform=None), dict(n_seq=-1), dict(n_seq=3), dict(n_draft=-1), dict(n_draft=65),
                dict(n_draft=4), dict(vocab=0), dict(vocab=101), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e-30), dict(temperature=float("inf")),
                dict(draft_temperature=0.0), dict(target_stride=99), dict(target_stride=101), dict(draft_stride=101), dict(out=t), dict(accepted=o), dict(out=x),
                dict(target=x.ptr + 2, n_seq=1), dict(n_seq=(1 << 16) + 1)):
        with pytest.raises(iam.IamError) as e:
            ctx.verify_drafts(**dict(ok, **bad))
        assert e.value.code == iam.IAM_E_INVALID, bad
    for b in (x, y, t, u, c, o, a):
        b.free()
