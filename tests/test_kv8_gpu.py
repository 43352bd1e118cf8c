"""The 8-bit KV cache (through libiam.so): what it holds and reads back, byte
for byte, against its definition in float64."""
import numpy as np
import pytest

import plain64 as P

pytestmark = pytest.mark.gpu


class Cache:
    """A library cache beside the fp16 rows that it was given."""

    def __init__(self, iam, ctx, n_seq, max_ctx, kv, dim, format):
        self.ctx, self.shape, self.format = ctx, (n_seq, max_ctx, kv, dim), format
        self.c = iam.Kv8Cache(ctx, n_seq, max_ctx, kv, dim, format)
        self.k = np.zeros((n_seq, max_ctx, kv, dim), np.float16)
        self.v = np.zeros_like(self.k)
        self.len = np.zeros(n_seq, np.int64)

    def append(self, k, v, pos, type="f32", count=None, pad=0):
        """k, v [n_seq][n][kv][dim] float; rows `pad` values further apart."""
        S, T, kv, dim = self.shape
        n = k.shape[1]
        bufs = []
        for x, held in ((k, self.k), (v, self.v)):
            w, val = P.to_type(x, type)
            row = np.zeros((S, n, kv * dim + pad), w.dtype)
            row[..., :kv * dim] = w.reshape(S, n, -1)
            bufs.append(self.ctx.upload(row))
            with np.errstate(over="ignore"):
                h = val.astype(np.float16)
            for s in range(S):
                m = min(n if count is None else min(n, count[s]), T - pos[s])
                if pos[s] >= 0 and m > 0:
                    held[s, pos[s]:pos[s] + m] = h[s, :m]
        for s in range(S):
            m = min(n if count is None else min(n, count[s]), T - pos[s])
            if pos[s] >= 0 and m > 0:
                self.len[s] = pos[s] + m
        bufs.append(self.ctx.upload(np.asarray(pos, np.int32)))
        dc = None if count is None else self.ctx.upload(np.asarray(count, np.int32))
        self.c.append(bufs[0], bufs[1], type, n, bufs[2], count=dc, stride=kv * dim + pad if pad else 0)
        self.ctx.sync()
        for b in bufs + ([dc] if dc else []):
            b.free()

    def read(self, first, n):
        S, _, kv, dim = self.shape
        out = [self.ctx.upload(np.full((S, n, kv, dim), 7.25, np.float32)) for _ in range(2)]
        p = self.ctx.upload(np.asarray(first, np.int32))
        self.c.read(p, n, out[0], out[1])
        got = [o.read(np.float32).reshape(S, n, kv, dim) for o in out]
        for b in out + [p]:
            b.free()
        return got

    def check(self):
        """Everything each sequence holds, and its scales."""
        S, T, kv, dim = self.shape
        got = self.read([0] * S, T)
        blocks = (T + 63) // 64
        for which, (g, held) in enumerate(zip(got, (self.k, self.v))):
            scales = self.c.parts[2 + which].read(np.float32).reshape(S, blocks, kv)
            for s in range(S):
                n = int(self.len[s])
                want, sc = P.stands_for(held[s, :n], self.format)
                assert np.array_equal(scales[s, :n // 64].view(np.uint32), sc.view(np.uint32)) or \
                    np.array_equal(scales[s, :n // 64], sc, equal_nan=True)
                assert np.array_equal(g[s, :n], want, equal_nan=True), (which, s, n)
                if n % 64:
                    assert (scales[s, n // 64] == -1).all()

    def raw(self):
        return [b.read() for b in self.c.parts]

    def free(self):
        self.c.free()


def rows(rng, *shape):
    """Values over many binades, with zeros, ties and equal magnitudes."""
    x = rng.normal(0, 1, shape) * np.exp2(rng.integers(-9, 3, shape))
    x[..., ::17] = 0
    x[..., 3::29] = np.rint(x[..., 3::29] * 4) / 4
    return x


def test_numbers_of_the_formats():
    # the oracle's own rounding: ties to even, both formats' ends
    assert P.numbers(np.array([0.5, 1.5, -2.5, 126.5, 127.0]), "int8").tolist() == [0, 2, -2, 126, 127]
    q = np.array([448, 440, 17, 17.0001, 19, 2.0 ** -6, 1.5 * 2 ** -9, 2.5 * 2 ** -9, 0.4 * 2 ** -9, -0.0137])
    want = [448, 448, 16, 18, 20, 2.0 ** -6, 2 ** -8, 2 ** -8, 0, -0.013671875]
    assert P.numbers(q, "e4m3").tolist() == want


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,kv", [(64, 3), (128, 8), (256, 1)])
def test_prompt_and_bytes(iam, ctx, format, dim, kv):
    rng = np.random.default_rng(dim + kv)
    c = Cache(iam, ctx, 2, 320, kv, dim, format)
    x = rows(rng, 2, 200, kv, dim), rows(rng, 2, 200, kv, dim)
    c.append(*x, pos=[0, 64], type="f16")
    c.k[1, :64] = c.v[1, :64] = 0                      # never written: not looked at
    got = c.read([0, 64], 200)
    for g, held in zip(got, (c.k, c.v)):
        assert np.array_equal(g[0], P.stands_for(held[0, :200], format)[0])
        assert np.array_equal(g[1], P.stands_for(held[1, 64:264], format)[0])
    # the documented order of the bytes, one block
    t, d = np.meshgrid(np.arange(64), np.arange(dim), indexing="ij")
    for which, at in ((0, P.k_place(t, d, dim)), (1, P.v_place(t, d, dim))):
        assert sorted(at.ravel().tolist()) == list(range(64 * dim))
        tile = c.raw()[which].reshape(2, 5, kv, 64 * dim)[0, 1, kv - 1]
        held = (c.k, c.v)[which][0, 64:128, kv - 1]
        s = P.block_scale(held, format)
        n = P.numbers(held.astype(np.float64) / np.float64(s), format)
        if format == "int8":
            assert np.array_equal(tile[at].astype(np.int64) - 128, n.astype(np.int64))
        opened = c.raw()[4 + which].view(np.float16).reshape(2, kv, 64 * dim)[0, 0]
        assert np.array_equal(opened[at][:200 % 64], (c.k, c.v)[which][0, 192:200, 0])
    c.free()


@pytest.mark.parametrize("type", P.TYPES)
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_tokens_come_as_they_like(iam, ctx, type, format):
    """Any split of the tokens into calls leaves the same bytes, a batch of
    ragged sequences with padding among them."""
    rng = np.random.default_rng(5)
    T, kv, dim, S = 210, 2, 64, 3
    x = rows(rng, S, T, kv, dim), rows(rng, S, T, kv, dim)
    end = [210, 64, 131]
    whole = Cache(iam, ctx, S, T, kv, dim, format)
    whole.append(*x, pos=[0] * S, type=type, count=end)
    whole.check()
    parts = Cache(iam, ctx, S, T, kv, dim, format)
    at = [0] * S
    for n in (1, 1, 61, 1, 1, 30, 70, 1, 33, 500):
        n = min(n, T)
        take = [min(n, e - a) for a, e in zip(at, end)]
        chunk = [np.zeros((S, n, kv, dim)) for _ in range(2)]
        for s in range(S):
            for cc, xx in zip(chunk, x):
                cc[s, :take[s]] = xx[s, at[s]:at[s] + take[s]]
                cc[s, take[s]:] = np.nan                 # padding is not read
        parts.append(*chunk, pos=[a if t else -1 for a, t in zip(at, take)], type=type, count=take, pad=8 if n % 2 else 0)
        at = [a + t for a, t in zip(at, take)]
        parts.check()
    assert at == end
    blocks = 4
    for which in range(4):
        a, b = whole.raw()[which], parts.raw()[which]
        a, b = a.reshape(S, blocks, -1), b.reshape(S, blocks, -1)
        for s in range(S):
            assert np.array_equal(a[s, :end[s] // 64], b[s, :end[s] // 64])
    whole.free()
    parts.free()


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_scales_and_borders(iam, ctx, format):
    """Zeros, one value, subnormals, the largest numbers, ties on the border of
    two numbers and values that are not finite."""
    rng = np.random.default_rng(8)
    kv, dim = 1, 64
    blocks = []
    blocks.append(np.zeros((64, kv, dim)))
    one = np.zeros((64, kv, dim))
    one[63, 0, 63] = -3.0
    blocks.append(one)
    blocks.append(np.full((64, kv, dim), 2.0 ** -24))
    big = np.full((64, kv, dim), 65504.0)
    big[::2] *= -1
    blocks.append(big)
    top = 127.0 if format == "int8" else 448.0           # quotients are the values, up to the scale's rounding
    tie = rng.integers(-253, 254, (64, kv, dim)) / 2.0 if format == "int8" else \
        np.ldexp(rng.integers(-31, 32, (64, kv, dim)) / 1.0, rng.integers(-10, 4, (64, kv, dim)))
    tie[0, 0, 0] = top
    blocks.append(tie)
    for bad in (np.nan, np.inf, -np.inf, 70000.0):       # 70000 is infinite in fp16
        x = rows(rng, 64, kv, dim)
        x[17, 0, 5] = bad
        blocks.append(x)
    blocks.append(rows(rng, 64, kv, dim))
    x = np.concatenate(blocks)[None]
    c = Cache(iam, ctx, 1, x.shape[1], kv, dim, format)
    c.append(x, x[:, ::-1].copy(), pos=[0])
    c.check()
    c.free()


def test_random_quotients_round_correctly(iam, ctx):
    """Many scales and values: every number equals the exact quotient's rounding."""
    rng = np.random.default_rng(11)
    for format in ("int8", "e4m3"):
        c = Cache(iam, ctx, 4, 64 * 40, 2, 128, format)
        k = rng.normal(0, 1, (4, 64 * 40, 2, 128)) * np.exp2(rng.integers(-12, 12, (4, 1, 2, 1)))
        c.append(k, k[:, ::-1].copy(), pos=[0] * 4, type="f16")
        c.check()
        c.free()


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_going_back(iam, ctx, format):
    """Appending inside a full block: its earlier tokens are what they stood for."""
    rng = np.random.default_rng(13)
    c = Cache(iam, ctx, 2, 256, 2, 128, format)
    c.append(rows(rng, 2, 150, 2, 128), rows(rng, 2, 150, 2, 128), pos=[0, 0])
    back = [100, 64]
    for held in (c.k, c.v):
        want = P.stands_for(held[0, :128], format)[0]
        held[0, 64:100] = want[64:100].astype(np.float16)
    c.append(rows(rng, 2, 20, 2, 128), rows(rng, 2, 20, 2, 128), pos=back)
    c.check()
    # on to the end of the block, one at a time
    for i in range(10):
        c.append(rows(rng, 2, 1, 2, 128), rows(rng, 2, 1, 2, 128), pos=[120 + i, 84 + i])
    c.check()
    # over the whole again from the start
    c.append(rows(rng, 2, 128, 2, 128), rows(rng, 2, 128, 2, 128), pos=[0, 0])
    c.check()
    c.free()


def test_ends_of_the_cache(iam, ctx):
    """Tokens past max_ctx are dropped, negative positions skipped, rows of
    positions outside are left alone."""
    rng = np.random.default_rng(17)
    c = Cache(iam, ctx, 3, 100, 1, 64, "int8")
    before = [b.copy() for b in c.raw()]
    c.append(rows(rng, 3, 4, 1, 64), rows(rng, 3, 4, 1, 64), pos=[-1, 100, 2 ** 31 - 1])
    assert all(np.array_equal(a, b) for a, b in zip(before, c.raw()))
    c.append(rows(rng, 3, 120, 1, 64), rows(rng, 3, 120, 1, 64), pos=[0, 0, -5])
    c.len[2] = 0
    c.check()
    c.append(rows(rng, 3, 3, 1, 64), rows(rng, 3, 3, 1, 64), pos=[98, 99, 0], count=[3, 0, -7])
    c.check()
    k, v = c.read([98, -2, 2 ** 31 - 2], 4)
    for g, held in ((k, c.k), (v, c.v)):
        assert np.array_equal(g[0, :2, 0], held[0, 98:, 0].astype(np.float32)) and (g[0, 2:] == 7.25).all()
        assert (g[1, :2] == 7.25).all() and np.array_equal(g[1, 2:], P.stands_for(held[1], "int8")[0][:2])
        assert (g[2] == 7.25).all()
    c.free()


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_reads_at_any_place(iam, ctx, format, dim):
    rng = np.random.default_rng(dim)
    T, held = 230, 211
    c = Cache(iam, ctx, 2, T, 3, dim, format)
    c.append(rows(rng, 2, held, 3, dim), rows(rng, 2, held, 3, dim), pos=[0, 0])
    stand = [[P.stands_for(x[s, :held], format)[0] for s in range(2)] for x in (c.k, c.v)]
    for n in (1, 3, 4, 5, 63, 64, 65, 130, 300):
        for first in ((0, 1), (13, 63), (64, 70), (-3, 200), (127, -64)):
            for got, want in zip(c.read(first, n), stand):
                for s in range(2):
                    for i in range(n):
                        p = first[s] + i
                        if p < 0 or p >= T:
                            assert (got[s, i] == 7.25).all()
                        elif p < held:
                            assert np.array_equal(got[s, i], want[s][p]), (n, p)
    c.free()


def test_refusals(iam, ctx):
    import ctypes as C
    for bad in ((0, 64, 1, 64), (65536, 64, 1, 64), (1, 0, 1, 64), (1, (1 << 24) + 1, 1, 64), (1, 64, 0, 64), (1, 64, 513, 64), (1, 64, 1, 96)):
        with pytest.raises(iam.IamError):
            iam.check(iam.lib().iam_kv8_size(*bad, None, None, None))
    c = iam.Kv8Cache(ctx, 2, 64, 2, 64, "int8")
    x, p = ctx.empty(2 * 4 * 128, np.float32), ctx.upload(np.zeros(2, np.int32))
    o1, o2 = ctx.empty(2 * 4 * 128, np.float32), ctx.empty(2 * 4 * 128, np.float32)

    def refused(f, *a, **k):
        with pytest.raises(iam.IamError) as e:
            f(*a, **k)
        assert e.value.code == iam.IAM_E_INVALID

    c.append(x, x, "f32", 4, p)
    c.append(x, x, "f32", 0, p)
    c.read(p, 4, o1, o2)
    c.read(p, 0, o1, o2)
    for a in ((None, x, "f32", 4, p), (x, None, "f32", 4, p), (x, x, "f32", 4, None), (x, x, "f32", 5, p), (x, x, "f32", -1, p),
              (x.ptr + 2, x, "f32", 1, p), (x, c.parts[4], "f32", 1, p), (x, x, "f32", 1, p.ptr + 4)):
        refused(c.append, *a)
    refused(c.append, x, x, "f32", 4, p, stride=127)
    refused(c.append, x, x, "f32", 4, p, stride=200)
    refused(c.append, x, x, "f32", 4, p, count=p.ptr + 4)
    for a in ((None, 4, o1, o2), (p, 4, o1, o1), (p, 5, o1, o2), (p, -1, o1, o2), (p, 4, o1.ptr + 4, o2), (p, 1, c.parts[0], o2), (p, 1, o1, None)):
        refused(c.read, *a)
    for field, value in (("format", 2), ("head_dim", 96), ("n_seq", 3), ("max_ctx", 65), ("k", None), ("v_scale", c.parts[3].ptr + 4),
                         ("v", c.parts[0].ptr)):
        was = getattr(c.desc, field)
        setattr(c.desc, field, value)
        refused(c.append, x, x, "f32", 4, p)
        refused(c.read, p, 4, o1, o2)
        refused(c.reset)
        setattr(c.desc, field, was)
    c.append(x, x, "f32", 4, p)
    for b in (x, p, o1, o2):
        b.free()
    c.free()


def test_rows_past_64_bits_are_refused(iam, ctx):
    """641 * 6700417 - 1 is 2^32: rows 2^30 values apart end at 2^64 bytes, as
    if they were one."""
    c = iam.Kv8Cache(ctx, 641, 64, 1, 64, "int8")
    x, pos = ctx.empty(64, np.float32), ctx.upload(np.full(641, -1, np.int32))
    with pytest.raises(iam.IamError) as e:
        c.append(x, x, "f32", 6700417, pos, stride=1 << 30)
    assert e.value.code == iam.IAM_E_INVALID and "kv8_append k" in str(e.value)
    with pytest.raises(iam.IamError) as e:
        c.attention(x, "f32", 1, 6700417, pos, x, q_stride=1 << 30, out_stride=1 << 30)
    assert e.value.code == iam.IAM_E_INVALID and "attention_kv8 q" in str(e.value)
    for d in (x, pos):
        d.free()
    c.free()
