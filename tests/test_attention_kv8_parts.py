"""That the attention over the 8-bit cache keeps the low parts of an fp32 q and
of the probabilities: inputs whose scores are exact in fp32, so that the room
for the rest is far below what either low part is worth.

Every query value is 1 + r 2^-14 with a whole r of 0 to 7, and the keys' numbers
come in pairs c, -c.  The high fp16 parts of q are all alike and their products
cancel: the scores are the low parts' alone.  All products and sums of a score are
whole multiples of 2^-5 below 2^18 (in units of the keys' scale and of q's), 23
bits, so that fp32 adds them without rounding in any order.  V has one value in
a block and dimension, none of them negative, so that probabilities that are
cut short all move the result one way and few of them make each result."""
import numpy as np
import pytest

import plain64 as P

UNIT = 0.125     # close to the scale of every block


def keys_values(rng, S, T, kv, dim, format):
    """Rows [S][T][kv][dim]; each block's largest numbers (127 or 448) cancel too."""
    top = 127 if format == "int8" else 448
    c = rng.integers(1, 5, (S, T, kv, dim // 2)) * rng.choice([-1, 1], (S, T, kv, dim // 2))
    k = np.stack([c, -c], -1).reshape(S, T, kv, dim).astype(np.float64)
    k[:, ::P.BLOCK, :, 0], k[:, ::P.BLOCK, :, 1] = top, -top
    v = rng.integers(60, 128, (S, T, kv, dim)) if format == "int8" else rng.integers(8, 15, (S, T, kv, dim)) * 32
    v[:, ::P.BLOCK, :, 0] = top
    t, d = np.arange(T)[:, None, None], np.arange(dim)
    v = np.where(t % P.BLOCK == d % P.BLOCK, v, 0).astype(np.float64)
    return k * UNIT, v * UNIT


def queries(rng, *shape):
    r = rng.integers(0, 8, shape)
    r[..., 0] = 0
    r[..., 1] = 0
    return 1 + r * 2.0 ** -14


def scale_for(dim):
    """Scores of deviation 1: dim / 2 differences of two r, 5.25 variance each,
    times c, 7.5 mean square."""
    return float(np.float32(1 / (UNIT * 2.0 ** -14 * np.sqrt(dim / 2 * 2 * 5.25 * 7.5))))


def room(s, w, v):
    """How far an fp32 evaluation of one row (scores s, probabilities w, values
    v [m][dim]) may be off:

    - in units of log 2, a score S = s / ln 2 has two factors' roundings (2 |S|), the
      maximum's shift by 12 (12 + |S|), the sum of both (12 + 2 |S|), and the
      difference of two maxima (2 |S|): (24 + 7 |S|) 2^-24, times ln 2;
    - p = 2^x by an instruction good to 2^-22;
    - p's high part leaves less than 2^-10 of it, of which the low one keeps all but
      2^-11: 2^-21;
    - sums: 64 additions in a block, one and a rescaling (2^-22 and a rounding) a
      block, 16 where parts join, each up to 2^-23.
    All enter sum p v and sum p."""
    m = len(s)
    ds = (17 + 7 * np.abs(s).max()) * 2.0 ** -24
    rel = 2 * (ds + 2.0 ** -22 + 2.0 ** -21) + 2 * (64 + 4 * (m / 64) + 16) * 2.0 ** -23
    return rel * (w @ v)


def plain(q, k, v, pos, scale):
    """q [n][heads][dim] from position pos on, k, v [T][kv][dim]: (out, room)."""
    out, r = np.zeros_like(q), np.zeros_like(q)
    rep = q.shape[1] // k.shape[1]
    for i in range(q.shape[0]):
        for h in range(q.shape[1]):
            kk, vv = k[:pos + i + 1, h // rep], v[:pos + i + 1, h // rep]
            s = kk @ q[i, h] * scale
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[i, h], r[i, h] = w @ vv, room(s, w, vv)
    return out, r


def within(got, want, r):
    return np.abs(got - want) <= r + (np.abs(want) + r) * P.HALF_STEP["f32"]


def model(q, k, v, pos, scale, q_low, p_low):
    """The scheme in numpy: q and p in two fp16 parts, the low ones as said
    ("kept", "dropped", "another's": of the next row)."""
    rep = q.shape[1] // k.shape[1]
    x = q * 512
    high = x.astype(np.float16).astype(np.float64)
    low = (x - high).astype(np.float16).astype(np.float64)
    low = {"kept": low, "dropped": 0 * low, "another's": np.roll(low, 1, 1)}[q_low]
    out = np.zeros_like(q)
    for i in range(q.shape[0]):
        for h in range(q.shape[1]):
            kk, vv = k[:pos + i + 1, h // rep], v[:pos + i + 1, h // rep]
            s = kk @ (high[i, h] + low[i, h]) / 512 * scale
            p = np.exp(s - s.max()) * 2.0 ** 12
            ph = p.astype(np.float16).astype(np.float64)
            ph = np.where(ph > p, np.nextafter(ph.astype(np.float16), np.float16(0)).astype(np.float64), ph)
            pl = (p - ph).astype(np.float16).astype(np.float64)
            pl = {"kept": pl, "dropped": 0 * pl, "another's": np.roll(pl, 1)}[p_low]
            out[i, h] = (ph + pl) @ vv / p.sum()
    return out


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,kv,dim,T", [(1, 8, 2, 128, 200), (1, 4, 1, 64, 1000), (3, 4, 2, 256, 70), (20, 4, 1, 128, 500)])
def test_the_room_tells_the_parts_apart(format, n, heads, kv, dim, T):
    rng = np.random.default_rng(T + dim)
    k, v = keys_values(rng, 1, T, kv, dim, format)
    k, v = (P.stands_for(x[0].astype(np.float16), format)[0].astype(np.float64) for x in (k, v))
    q, scale = queries(rng, n, heads, dim), scale_for(dim)
    want, r = plain(q, k, v, T - n, scale)
    assert within(model(q, k, v, T - n, scale, "kept", "kept"), want, r).all()
    for parts in (("dropped", "kept"), ("kept", "dropped"), ("dropped", "dropped"), ("another's", "kept"), ("kept", "another's")):
        ok = within(model(q, k, v, T - n, scale, *parts), want, r)
        # of every row, hardly any value by chance
        assert ok.mean(-1).max() < 0.5 and ok.mean() < 0.25, (parts, ok.mean())


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("n,heads,kv,dim,T", [(1, 32, 8, 128, 200), (1, 4, 4, 64, 700), (2, 8, 1, 256, 333), (1, 32, 8, 128, 1000), (8, 8, 2, 128, 640),
                                              (70, 8, 2, 128, 300), (40, 16, 2, 64, 200), (30, 8, 1, 256, 260), (150, 4, 1, 128, 700), (33, 4, 1, 64, 1000)])
def test_low_parts(iam, ctx, format, n, heads, kv, dim, T):
    """Few and many rows, single workgroups and joined ones, full and open blocks."""
    from test_attention_kv8_gpu import attend, values
    from test_kv8_gpu import Cache

    rng = np.random.default_rng(T + dim)
    c = Cache(iam, ctx, 1, T, kv, dim, format)
    k, v = keys_values(rng, 1, T, kv, dim, format)
    c.append(k, v, pos=[0])
    assert (c.k[0] == k[0]).all() and (c.v[0] == v[0]).all()      # exact in fp16
    q, scale = queries(rng, 1, n, heads, dim), scale_for(dim)
    got, _, val = attend(ctx, c, q, "f32", [T - n], scale=scale)
    assert (val == q).all()
    k, v = values(c, 0)
    want, r = plain(q[0], k, v, T - n, scale)
    ok = within(got[0], want, r)
    assert ok.all(), (float((np.abs(got[0] - want) / r).max()), np.argwhere(~ok)[:3].tolist())
    c.free()
