"""Attention over the 8-bit cache (through libiam.so) against float64 of what
the cache stands for, within the bounds that plain64.attention derives."""
import numpy as np
import pytest

import plain64 as P
from test_kv8_gpu import Cache

pytestmark = pytest.mark.gpu


def fill(iam, ctx, rng, S, T, kv, dim, format, lengths, chunk=None):
    c = Cache(iam, ctx, S, T, kv, dim, format)
    n = max(max(lengths), 1)
    k, v = (rng.normal(0, 1, (S, n, kv, dim)) * np.exp(rng.normal(0, 0.5, (kv, dim))) for _ in range(2))
    c.append(k, v, pos=[0] * S, type="f16", count=lengths)
    return c


def values(c, s):
    n = int(c.len[s])
    return [P.stands_for(x[s, :n], c.format)[0].astype(np.float64) for x in (c.k, c.v)]


def attend(ctx, c, q, type, pos, window=0, scale=0.0, count=None, qpad=0, opad=0, in_place=False):
    """The library's rows as float64, and the stored words before and after."""
    S, n, heads, dim = q.shape
    w, val = P.to_type(q, type)
    rows = np.zeros((S, n, heads * dim + qpad), w.dtype)
    rows[..., :heads * dim] = w.reshape(S, n, -1)
    dq = ctx.upload(rows)
    old = P.to_type(np.full((S, n, heads * dim + opad), 7.25), type)[0]
    do = dq if in_place else ctx.upload(old)
    dp = ctx.upload(np.asarray(pos, np.int32))
    dc = None if count is None else ctx.upload(np.asarray(count, np.int32))
    c.c.attention(dq, type, heads, n, dp, do, count=dc, window=window, scale=scale, q_stride=heads * dim + qpad if qpad else 0,
                  out_stride=heads * dim + opad if opad else 0)
    got = do.read(w.dtype).reshape(S, n, -1)
    for b in {dq, do, dp} | ({dc} if dc else set()):
        b.free()
    return P.from_bits(got[..., :heads * dim], type).reshape(S, n, heads, dim), got, val


def check(ctx, c, q, type, pos, window=0, scale=0.0, count=None, **kw):
    got, words, val = attend(ctx, c, q, type, pos, window, scale, count, **kw)
    S, n = q.shape[:2]
    for s in range(S):
        m = n if count is None else min(n, count[s])
        if m > 0:
            if pos[s] < 0:
                assert (got[s, :m] == 0).all()
            else:
                k, v = values(c, s)
                want, bound = P.attention(val[s, :m], k, v, pos[s], window, scale)
                P.close(got[s, :m], want, bound, type)
        if not kw.get("in_place"):
            assert (got[s, max(m, 0):] == 7.25).all()
    return words


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (4, 4, 64), (8, 1, 256), (10, 2, 128), (32, 1, 64), (6, 2, 256)])
def test_one_token(iam, ctx, type, format, heads, kv, dim):
    """Contexts of one token, the ends of blocks, and enough to be shared out."""
    rng = np.random.default_rng(heads * dim)
    lengths = [1, 63, 64, 65, 200, 1000]
    c = fill(iam, ctx, rng, len(lengths), 1024, kv, dim, format, lengths)
    check(ctx, c, rng.normal(0, 1, (len(lengths), 1, heads, dim)), type, [n - 1 for n in lengths])
    c.free()


@pytest.mark.parametrize("length", [1, 5, 64, 257, 4091, 9000])
def test_one_sequence(iam, ctx, length):
    rng = np.random.default_rng(length)
    c = fill(iam, ctx, rng, 1, 9001, 8, 128, "int8", [length])
    a = check(ctx, c, rng.normal(0, 1, (1, 1, 32, 128)), "f32", [length - 1])
    rng = np.random.default_rng(length)
    rng.normal(0, 1, 1)
    c.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,kv,dim,length", [(2, 8, 2, 64, 66), (5, 32, 8, 128, 70), (37, 12, 4, 128, 300), (130, 4, 4, 64, 130),
                                                   (64, 8, 1, 256, 200), (3, 32, 1, 128, 1000)])
def test_chunks_of_a_prompt(iam, ctx, type, n, heads, kv, dim, length):
    rng = np.random.default_rng(n)
    lengths = [length, max(n, length // 2)]
    c = fill(iam, ctx, rng, 2, length + 10, kv, dim, "e4m3", lengths)
    check(ctx, c, rng.normal(0, 1, (2, n, heads, dim)), type, [x - n for x in lengths])
    c.free()


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
@pytest.mark.parametrize("n", [1, 9, 90])
def test_windows(iam, ctx, window, n):
    rng = np.random.default_rng(window)
    lengths = [400, 129, 90]
    c = fill(iam, ctx, rng, 3, 400, 2, 64, "int8", lengths)
    check(ctx, c, rng.normal(0, 1, (3, n, 8, 64)), "f32", [x - n for x in lengths], window=window)
    c.free()


def test_padded_batch_strides_scale_and_in_place(iam, ctx):
    rng = np.random.default_rng(2)
    lengths = [100, 70, 200, 64, 1, 0]
    c = fill(iam, ctx, rng, 6, 256, 2, 128, "int8", lengths)
    q = rng.normal(0, 1, (6, 7, 6, 128))
    pos, count = [93, 66, -1, 60, 0, -3], [7, 4, 3, 0, 1, 7]
    for type in P.TYPES:
        check(ctx, c, q, type, pos, count=count)
        words = check(ctx, c, q, type, pos, count=count, qpad=3, opad=9, scale=0.031, window=80)
        assert (P.from_bits(words[..., 6 * 128:], type) == 7.25).all()     # between the rows
        check(ctx, c, q[:, :1], type, [99, 69, 199, 63, 0, -1], in_place=True)
    c.free()


def test_sharp_and_flat_rows(iam, ctx):
    """Logits far above 1 (one position takes all), a rising maximum over the
    blocks, all equal, a query of zeros, of tiny and of huge values."""
    rng = np.random.default_rng(4)
    T, kv, dim = 700, 1, 64
    c = Cache(iam, ctx, 1, T, kv, dim, "int8")
    k, v = rng.normal(0, 1, (1, T, kv, dim)), rng.normal(0, 3, (1, T, kv, dim))
    k *= np.linspace(0.2, 3, T)[None, :, None, None]      # later blocks reach higher
    c.append(k, v, pos=[0])
    q = rng.normal(0, 1, (1, 1, 8, dim))
    q[0, 0, 1] = 0
    q[0, 0, 2] *= 1e-30
    q[0, 0, 3] *= 8
    q[0, 0, 4] = np.exp2(np.linspace(-40, 4, dim))
    q[0, 0, 5] = 1e-41                                    # subnormal in fp32
    q[0, 0, 6, 1:] = 0
    check(ctx, c, q, "f32", [T - 1])
    q[0, 0, 2] *= 1e29
    check(ctx, c, q, "bf16", [T - 1])
    c.free()


@pytest.mark.parametrize("type", ["f32", "f16"])
def test_not_finite(iam, ctx, type):
    """NaN and infinities reach exactly the rows that see them."""
    rng = np.random.default_rng(6)
    S, T, kv, dim, heads = 4, 200, 2, 64, 8
    c = Cache(iam, ctx, S, T, kv, dim, "e4m3")
    k, v = rng.normal(0, 1, (S, 150, kv, dim)), rng.normal(0, 1, (S, 150, kv, dim))
    v[0, 140, 1, 3] = np.nan          # in the open block (128 ..): by token
    v[1, 140, 0, 3] = np.inf
    k[2, 70, 1, 0] = np.nan           # in a full block (64 .. 127): by block
    c.append(k, v, pos=[0] * S)
    n = 30
    q = rng.normal(0, 1, (S, n, heads, dim))
    q[3, 4, 2, 7] = np.nan
    q[3, 5, 3, 0] = np.inf
    got, _, val = attend(ctx, c, q, type, [120] * S)
    h = np.arange(heads) // (heads // kv)
    row, head = np.meshgrid(np.arange(n), np.arange(heads), indexing="ij")
    bad = np.zeros((S, n, heads), bool)
    bad[0] = (row + 120 >= 140) & (h[head] == 1)
    bad[1] = (row + 120 >= 140) & (h[head] == 0)
    bad[2] = h[head] == 1
    bad[3] = ((row == 4) & (head == 2)) | ((row == 5) & (head == 3))
    fine = np.isfinite(got).all(-1)
    assert np.array_equal(fine, ~bad)
    for s in range(S):
        kk, vv = values(c, s)
        want, bound = P.attention(np.where(np.isfinite(val[s]), val[s], 0), np.nan_to_num(kk, posinf=0, neginf=0),
                                  np.nan_to_num(vv, posinf=0, neginf=0), 120)
        P.close(got[s][fine[s]], want[fine[s]], bound[fine[s]], type)
    # a window past the poisoned block, and rows before the bad token
    got, _, val = attend(ctx, c, q[:, :1], type, [139] * S, window=12)
    assert np.isfinite(got[:3]).all()
    c.free()


@pytest.mark.parametrize("n,heads,kv,dim", [(1, 8, 2, 64), (4, 8, 2, 128), (2, 3, 1, 256), (16, 64, 32, 64)])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_not_finite_few_rows(iam, ctx, format, n, heads, kv, dim):
    """The same for few rows: a poisoned block of K, of V, and tokens of the
    open block, seen or behind or before what is seen."""
    rng = np.random.default_rng(8)
    S, T = 2, 64 * 5 + 30
    c = Cache(iam, ctx, S, T, kv, dim, format)
    k, v = rng.normal(0, 1, (S, T, kv, dim)), rng.normal(0, 1, (S, T, kv, dim))
    k[0, 70, kv - 1, 0] = np.inf       # block 1 of K
    v[1, 140, 0, 3] = np.nan           # block 2 of V
    v[:, T - 10, kv - 1, 5] = -np.inf  # open
    k[1, T - 3, 0, 5] = np.nan
    c.append(k, v, pos=[0, 0])
    h = np.arange(heads) // (heads // kv)
    q = rng.normal(0, 1, (S, n, heads, dim))
    for pos in (10, 63, 64 * 2 + 7, 64 * 4, T - 30, T - 10, T - 4, T - n):
        for window in (0, 40, 100):
            got, _, val = attend(ctx, c, q, "f16", [pos] * S, window=window)
            for s in range(S):
                kk, vv = values(c, s)
                poison = ~np.isfinite(kk).all(-1) | ~np.isfinite(vv).all(-1)        # [T][kv]
                if n == 1 or pos + n <= T:
                    for i in range(n):
                        p = min(pos + i, T - 1)
                        lo = max(0, p - window + 1) if window else 0
                        bad = poison[lo:p + 1].any(0)[h]
                        assert np.array_equal(np.isfinite(got[s, i]).all(-1), ~bad), (pos, window, s, i)
                want, bound = P.attention(val[s], np.nan_to_num(kk, posinf=0, neginf=0), np.nan_to_num(vv, posinf=0, neginf=0), pos, window)
                fine = np.isfinite(got[s]).all(-1)
                P.close(got[s][fine], want[fine], bound[fine], "f16")
    c.free()


@pytest.mark.parametrize("n,heads,kv,dim", [(1, 8, 2, 64), (1, 4, 2, 128), (2, 6, 2, 256), (20, 12, 2, 128), (40, 16, 2, 64), (30, 4, 2, 256)])
@pytest.mark.parametrize("type", P.TYPES)
def test_infinite_keys_of_the_open_block(iam, ctx, type, n, heads, kv, dim):
    """Keys past fp16's range (infinities) of both signs: every row that sees one
    is NaN or infinite, whatever the sign of its query there, as it is
    once the block is full; the others are as without them."""
    rng = np.random.default_rng(21)
    S, T = 2, 64 * 3
    c = Cache(iam, ctx, S, T, kv, dim, "int8")
    k, v = rng.normal(0, 1, (S, 120, kv, dim)), rng.normal(0, 1, (S, 120, kv, dim))
    k[0, 70, 1, 5], k[0, 90, 0, dim - 1] = 1e6, -1e6
    k[1, 85, 0, 3], k[1, 100, 1, 0] = -1e6, 1e6
    c.append(k, v, pos=[0] * S)
    q = rng.normal(0, 1, (S, n, heads, dim))
    h = np.arange(heads) // (heads // kv)

    def see(pos, window):
        got, _, val = attend(ctx, c, q, type, [pos] * S, window=window)
        for s in range(S):
            kk, vv = values(c, s)
            poison = ~np.isfinite(kk).all(-1)
            for i in range(n):
                lo = max(0, pos + i - window + 1) if window else 0
                bad = poison[lo:pos + i + 1].any(0)[h]
                assert np.array_equal(np.isfinite(got[s, i]).all(-1), ~bad), (pos, window, s, i)
            want, bound = P.attention(val[s], np.nan_to_num(kk, posinf=0, neginf=0), vv, pos, window)
            fine = np.isfinite(got[s]).all(-1)
            P.close(got[s][fine], want[fine], bound[fine], type)

    for pos in (66, 75, 120 - n):
        for window in (0, 12):
            see(pos, window)
    more = rng.normal(0, 1, (S, 8, kv, dim))
    c.append(more, more, pos=[120] * S)          # the block is full
    see(128 - n, 0)
    c.free()


@pytest.mark.parametrize("n,heads,kv,dim,T", [(1, 8, 2, 64, 50), (1, 4, 2, 128, 700), (2, 6, 2, 256, 128), (20, 12, 2, 128, 300),
                                              (40, 16, 2, 64, 64), (30, 4, 2, 256, 90)])
@pytest.mark.parametrize("type", P.TYPES)
def test_infinite_queries(iam, ctx, type, n, heads, kv, dim, T):
    """A query with an infinity is a row of NaN, also where all its scores are
    -inf; the others are as without it."""
    rng = np.random.default_rng(22)
    c = Cache(iam, ctx, 1, T, kv, dim, "e4m3")
    k, v = rng.normal(0, 1, (1, T, kv, dim)), rng.normal(0, 1, (1, T, kv, dim))
    k[..., 3] = np.abs(k[..., 3]) + 1
    c.append(k, v, pos=[0])
    q = rng.normal(0, 1, (1, n, heads, dim))
    bad = np.zeros((n, heads), bool)
    for x in (-np.inf, np.inf):
        i, j = int(rng.integers(n)), int(rng.integers(heads))
        q[0, i, j, 3] = x
        bad[i, j] = True
    got, _, val = attend(ctx, c, q, type, [T - n])
    assert np.array_equal(np.isnan(got[0]).all(-1), bad)
    kk, vv = values(c, 0)
    want, bound = P.attention(np.where(np.isfinite(val[0]), val[0], 0), kk, vv, T - n)
    P.close(got[0][~bad], want[~bad], bound[~bad], type)
    c.free()


def test_what_the_open_block_held_before(iam, ctx):
    """A slot used again: NaN of the sequence before behind the new one's end."""
    rng = np.random.default_rng(9)
    c = Cache(iam, ctx, 1, 256, 1, 64, "int8")
    c.append(np.full((1, 190, 1, 64), np.nan), np.full((1, 190, 1, 64), np.nan), pos=[0])
    for n in (1, 40, 64, 70):
        k, v = rng.normal(0, 1, (1, n, 1, 64)), rng.normal(0, 1, (1, n, 1, 64))
        c.append(k, v, pos=[0])
        check(ctx, c, rng.normal(0, 1, (1, min(n, 3), 4, 64)), "f32", [n - min(n, 3)])
    c.free()


def test_past_the_end_and_far_offsets(iam, ctx):
    """Positions past max_ctx see all of it; a cache of more than 2^32 bytes."""
    rng = np.random.default_rng(10)
    c = fill(iam, ctx, rng, 1, 130, 1, 64, "int8", [130])
    q = rng.normal(0, 1, (1, 3, 2, 64))
    got, _, val = attend(ctx, c, q, "f32", [129])
    k, v = values(c, 0)
    want, bound = P.attention(val[0], k, v, 129)
    P.close(got[0], want, bound, "f32")
    got, _, _ = attend(ctx, c, q, "f32", [2 ** 31 - 2])
    P.close(got[0], np.stack([P.attention(val[0, i:i + 1], k, v, 129)[0][0] for i in range(3)]), bound, "f32")
    c.free()
    S, T = 5, (1 << 20) - 30
    big = iam.Kv8Cache(ctx, S, T, 8, 128, "int8")
    x = [rng.normal(0, 1, (S, 100, 8, 128)).astype(np.float16) for _ in range(2)]
    first = T - 100 - 62
    first -= first % 64
    pos = ctx.upload(np.full(S, first, np.int32))
    dk, dv = ctx.upload(x[0]), ctx.upload(x[1])
    big.append(dk, dv, "f16", 100, pos)
    q = rng.normal(0, 1, (S, 1, 32, 128)).astype(np.float32)
    dq, do, at = ctx.upload(q), ctx.empty(q.size, np.float32), ctx.upload(np.full(S, first + 99, np.int32))
    big.attention(dq, "f32", 32, 1, at, do, window=100)
    got = do.read().reshape(q.shape).astype(np.float64)
    ko, vo = ctx.empty(x[0].size, np.float32), ctx.empty(x[0].size, np.float32)
    big.read(pos, 100, ko, vo)
    kr, vr = ko.read().reshape(x[0].shape), vo.read().reshape(x[0].shape)
    for s in range(S):
        k, v = (P.stands_for(t[s], "int8")[0] for t in x)
        assert np.array_equal(kr[s], k) and np.array_equal(vr[s], v)
        want, bound = P.attention(q[s].astype(np.float64), k.astype(np.float64), v.astype(np.float64), 99)
        P.close(got[s], want, bound, "f32")
    for b in (pos, dk, dv, dq, do, at, ko, vo):
        b.free()
    big.free()


def test_calls_repeat_and_interleave(iam, ctx):
    """The same call gives the same bits whatever ran between (the workspaces
    are left as they were found), shared out or not, from two contexts too."""
    rng = np.random.default_rng(12)
    a = fill(iam, ctx, rng, 1, 4100, 8, 128, "int8", [4091])
    b = fill(iam, ctx, rng, 9, 700, 2, 64, "e4m3", [700, 1, 64, 65, 300, 128, 699, 2, 512])
    qa, qb = rng.normal(0, 1, (1, 1, 32, 128)), rng.normal(0, 1, (9, 3, 6, 64))
    pb = [int(n) - 1 for n in b.len]
    first = attend(ctx, a, qa, "f32", [4090])[1], attend(ctx, b, qb, "f32", pb)[1]
    for _ in range(5):
        again = attend(ctx, a, qa, "f32", [4090])[1], attend(ctx, b, qb, "f32", pb)[1]
        assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(first, again))
    with iam.Ctx(0) as other:
        c = Cache(iam, other, 1, 4100, 8, 128, "int8")
        c.append(a.k[:, :4091], a.v[:, :4091], pos=[0], type="f16")
        assert np.array_equal(attend(other, c, qa, "f32", [4090])[1].view(np.uint32), first[0].view(np.uint32))
    a.free()
    b.free()


def test_decode_step_as_it_is_used(iam, ctx):
    """Rotation of q and k side by side, append, attention, token by token
    behind a prompt: the chain against float64."""
    rng = np.random.default_rng(14)
    heads, kv, dim, T = 8, 2, 64, 150
    width = (heads + 2 * kv) * dim
    x = rng.normal(0, 1, (T, width)).astype(np.float32)
    table = ctx.empty(T * dim, np.float32)
    ctx.rope_scaled_table(10000.0, dim, T, table, scaling={"kind": "linear", "factor": 2.0})
    c = iam.Kv8Cache(ctx, 1, T, kv, dim, "int8")
    dx, do = ctx.upload(x), ctx.empty(T * heads * dim, np.float32)
    at = ctx.upload(np.arange(T, dtype=np.int32))
    B = 4

    def step(first, n):
        q = dx.ptr + first * width * B
        p = at.ptr + first * 4
        ctx.rope_tokens(q, "f32", n, heads + kv, dim, dim, "half", table, T, p, q, x_stride=width, out_stride=width)
        c.append(q + heads * dim * B, q + (heads + kv) * dim * B, "f32", n, p, stride=width)
        c.attention(q, "f32", heads, n, p, do.ptr + first * heads * dim * B, q_stride=width)

    step(0, 100)
    for t in range(100, T):
        step(t, 1)
    got = do.read().reshape(T, heads, dim).astype(np.float64)
    rot = dx.read().reshape(T, width)
    # the rotated rows themselves
    angle = np.arange(T)[:, None] * (10000.0 ** (-2.0 * np.arange(dim // 2) / dim) / 2.0)
    y = x[:, :(heads + kv) * dim].reshape(T, heads + kv, dim).astype(np.float64)
    a, b = y[..., :dim // 2], y[..., dim // 2:]
    cs, sn = np.cos(angle)[:, None], np.sin(angle)[:, None]
    want = np.concatenate([a * cs - b * sn, b * cs + a * sn], -1)
    # the table's rounding, two products, a sum
    room = 4 * 2.0 ** -24 * (np.concatenate([np.abs(a * cs) + np.abs(b * sn), np.abs(b * cs) + np.abs(a * sn)], -1)) + \
        2.0 ** -24 * np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    assert (np.abs(rot[:, :(heads + kv) * dim].reshape(y.shape) - want) <= room).all()
    q = rot[:, :heads * dim].reshape(T, heads, dim).astype(np.float64)
    k = rot[:, heads * dim:(heads + kv) * dim].reshape(T, kv, dim).astype(np.float16)
    v = rot[:, (heads + kv) * dim:].reshape(T, kv, dim).astype(np.float16)
    held = [(0, 100)] + [(t, 1) for t in range(100, T)]
    for first, n in held:
        kk, vv = (P.stands_for(z[:first + n], "int8")[0].astype(np.float64) for z in (k, v))
        w, bound = P.attention(q[first:first + n], kk, vv, first)
        P.close(got[first:first + n], w, bound, "f32")
    for b in (dx, do, at, table):
        b.free()
    c.free()


# sequences, tokens, heads, KV heads, width, longest: more items than the card
# holds workgroups (taken as one row of blocks), more than are dealt out by
# length, and the same by rows of a chunk
@pytest.mark.parametrize("S,n,heads,kv,dim,longest", [(300, 1, 4, 2, 64, 400), (70, 1, 16, 8, 128, 900), (2100, 1, 2, 1, 64, 70),
                                                      (30, 2, 32, 8, 64, 700), (2100, 20, 1, 1, 64, 70), (3, 150, 4, 1, 256, 500),
                                                      (5, 70, 8, 4, 128, 333), (260, 20, 4, 2, 64, 130)])
def test_many_sequences(iam, ctx, S, n, heads, kv, dim, longest):
    rng = np.random.default_rng(S + n)
    lengths = rng.integers(n, longest + 1, S)
    lengths[:3] = [longest, n, min(max(n, 64), longest)]
    c = fill(iam, ctx, rng, S, longest, kv, dim, "int8", lengths.tolist())
    pos = (lengths - n).tolist()
    pos[S // 2] = -1
    got, _, val = attend(ctx, c, rng.normal(0, 1, (S, n, heads, dim)), "f32", pos)
    assert (got[S // 2] == 0).all()
    for s in set(range(0, S, max(1, S // 60))) | {0, 1, 2, S - 1}:
        if pos[s] < 0:
            continue
        k, v = values(c, s)
        rows = sorted({0, n - 1, n // 2})
        for i in rows:
            want, bound = P.attention(val[s, i:i + 1], k, v, pos[s] + i)
            P.close(got[s, i:i + 1], want, bound, "f32")
    c.free()


@pytest.mark.parametrize("S,n,heads,kv,dim,T,window", [(1, 32, 8, 2, 128, 256, 0), (3, 11, 16, 2, 256, 130, 0), (2, 90, 2, 2, 64, 250, 0),
                                                       (2, 30, 8, 2, 128, 3000, 90), (40, 16, 8, 2, 128, 200, 0), (1, 129, 1, 1, 128, 256, 0)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_many_rows_of_little_context(iam, ctx, type, S, n, heads, kv, dim, T, window):
    """Small caches and windows, up to 128 rows and past them."""
    rng = np.random.default_rng(T + n)
    lengths = rng.integers(n, T + 1, S).tolist()
    lengths[0] = T
    c = fill(iam, ctx, rng, S, T, kv, dim, "int8", lengths)
    check(ctx, c, rng.normal(0, 1, (S, n, heads, dim)), type, [x - n for x in lengths], window=window)
    c.free()


@pytest.mark.parametrize("seed", range(30))
def test_drawn(iam, ctx, seed):
    """Shapes, windows, counts and types drawn over the whole range."""
    rng = np.random.default_rng(1000 + seed)
    kv, rep, dim = int(rng.choice([1, 2, 4, 8])), int(rng.choice([1, 2, 3, 4, 7, 8])), int(rng.choice([64, 128, 256]))
    S = int(rng.integers(1, 6))
    n = int(np.exp(rng.uniform(0, np.log(90))))
    T = n + int(np.exp(rng.uniform(0, np.log(900))))
    format, type = str(rng.choice(["int8", "e4m3"])), str(rng.choice(P.TYPES))
    lengths = rng.integers(n, T + 1, S).tolist()
    c = fill(iam, ctx, rng, S, T + int(rng.integers(0, 70)), kv, dim, format, lengths)
    back = int(rng.integers(0, 40)) if rng.random() < 0.3 else 0       # tokens in the cache behind the queries
    pos = [max(0, x - n - back) for x in lengths]
    count = rng.integers(-1, n + 2, S).tolist() if rng.random() < 0.4 else None
    window = int(rng.integers(1, T + 1)) if rng.random() < 0.4 else 0
    q = rng.normal(0, 1, (S, n, kv * rep, dim)) * np.exp2(rng.integers(-6, 3))
    check(ctx, c, q, type, pos, window=window, count=count, qpad=int(rng.choice([0, 0, 1, 8])), opad=int(rng.choice([0, 0, 3])))
    c.free()


@pytest.mark.parametrize("S,n,heads,kv,dim,length", [(1, 1, 8, 1, 256, 73769), (1, 2, 8, 1, 256, 9001), (2, 1, 16, 1, 128, 30000),
                                                     (3, 4, 4, 1, 64, 20011), (1, 16, 1, 1, 128, 50000)])
def test_many_parts_of_one_sequence(iam, ctx, S, n, heads, kv, dim, length):
    """Few KV heads and a long context: more parts than one workgroup joins at
    once; twice, since the second call finds the first one's counters."""
    rng = np.random.default_rng(length)
    lengths = [length - 1000 * s for s in range(S)]
    c = fill(iam, ctx, rng, S, length, kv, dim, "int8", lengths)
    q = rng.normal(0, 1, (S, n, heads, dim)) * 2
    pos = [x - n for x in lengths]
    first = attend(ctx, c, q, "f32", pos)[1]
    for _ in range(3):
        assert np.array_equal(attend(ctx, c, q, "f32", pos)[1].view(np.uint32), first.view(np.uint32))
    check(ctx, c, q, "f32", pos)
    check(ctx, c, q, "bf16", pos, window=length // 2)
    c.free()


def test_blocks_of_unlike_scales(iam, ctx):
    """V from block to block 2^-20 to 2^12 of another, blocks of zeros among
    them, for single tokens and by rows."""
    rng = np.random.default_rng(20)
    c = Cache(iam, ctx, 1, 64 * 12 + 10, 1, 128, "int8")
    k, v = rng.normal(0, 1, (1, 64 * 12 + 5, 1, 128)), rng.normal(0, 1, (1, 64 * 12 + 5, 1, 128))
    for b, e in enumerate([0, 8, -6, -20, 12, 0, -8, 3, -3, 1, 10, -10]):
        v[:, 64 * b:64 * b + 64] *= 2.0 ** e
    v[:, 64 * 5:64 * 6] = 0
    k[:, 64 * 7:64 * 8] = 0
    c.append(k, v, pos=[0])
    for n in (1, 30, 200):
        check(ctx, c, rng.normal(0, 1, (1, n, 4, 128)), "f32", [64 * 12 + 5 - n])
    # windows that end in each of them alone
    for b in range(12):
        check(ctx, c, rng.normal(0, 1, (1, 20, 4, 128)), "f32", [64 * b + 44], window=21)
    c.free()


def test_refusals(iam, ctx):
    c = iam.Kv8Cache(ctx, 2, 64, 2, 64, "int8")
    n = 2 * 3 * 4 * 64
    q, o, p = ctx.empty(n, np.float32), ctx.empty(n, np.float32), ctx.upload(np.full(2, -1, np.int32))
    good = dict(q=q, type="f32", n_heads=4, n_tokens=3, pos=p, out=o)
    c.attention(**good)
    c.attention(**dict(good, n_tokens=0))
    for bad in (dict(q=None), dict(out=None), dict(pos=None), dict(n_heads=3), dict(n_heads=1), dict(n_heads=0), dict(n_tokens=-1),
                dict(n_tokens=4), dict(q_stride=255), dict(q_stride=300), dict(out_stride=1), dict(window=-1), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(out=q.ptr + 256), dict(out=q, out_stride=257, n_tokens=1),
                dict(q=q.ptr + 2), dict(out=c.parts[0].ptr, n_tokens=1), dict(pos=p.ptr + 4), dict(count=p.ptr + 4),
                dict(n_tokens=1, pos=o.ptr)):
        with pytest.raises(iam.IamError) as e:
            c.attention(**dict(good, **bad))
        assert e.value.code == iam.IAM_E_INVALID, bad
    c.attention(**good)
    for b in (q, o, p):
        b.free()
    c.free()
