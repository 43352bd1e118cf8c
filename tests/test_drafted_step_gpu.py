"""A step of a small model with 4-bit weights over drafted tokens, as a serving
loop runs it: norm to 8 bits, 4-bit products, rotary positions, the 8-bit cache
and its attention, the FFN, the head, the verification.  Each call's result is
read back and checked against the float64 form of what the call was given."""
import numpy as np
import pytest

import plain64 as P
import plain_rows as R

pytestmark = pytest.mark.gpu

DIM, FFN, HEADS, KV, HD, VOCAB, CTX, LAYERS, EPS = 256, 640, 4, 2, 64, 1000, 256, 2, 1e-5


class Layer:
    def __init__(self, iam, ctx, rng, zeros):
        self.m, self.v = {}, {}
        shapes = {"qkv": ((HEADS + 2 * KV) * HD, DIM), "o": (DIM, HEADS * HD), "up": (2 * FFN, DIM), "down": (DIM, FFN)}
        for name, (out, inp) in shapes.items():
            d = ctx.upload(rng.normal(0, 1 / np.sqrt(inp), (out, inp)).astype(np.float16))
            self.m[name] = iam.Q4Matrix(ctx, out, inp, 64, zeros=zeros)
            self.m[name].quantize(d, "f16")
            back = ctx.empty(out * inp, np.float32)
            self.m[name].read(0, out, back)
            self.v[name] = back.read().reshape(out, inp).astype(np.float64)
            d.free()
            back.free()
        self.gains = [ctx.upload((1 + rng.normal(0, 0.1, DIM)).astype(np.float16)) for _ in range(2)]
        self.cache = iam.Kv8Cache(ctx, 2, CTX, KV, HD, "int8")


class Step:
    """Two sequences' drafted tokens through the model."""

    def __init__(self, iam, ctx):
        rng = np.random.default_rng(0)
        self.iam, self.ctx = iam, ctx
        self.layers = [Layer(iam, ctx, rng, z) for z in (False, True)]
        self.embed = rng.normal(0, 1, (VOCAB, DIM)).astype(np.float16)
        d = ctx.upload(rng.normal(0, 0.3, (VOCAB, DIM)).astype(np.float16))
        self.head = iam.Q4Matrix(ctx, VOCAB, DIM, 128)
        self.head.quantize(d, "f16")
        back = ctx.empty(VOCAB * DIM, np.float32)
        self.head.read(0, VOCAB, back)
        self.head_v = back.read().reshape(VOCAB, DIM).astype(np.float64)
        self.gain = ctx.upload((1 + rng.normal(0, 0.1, DIM)).astype(np.float16))
        self.table = ctx.empty(CTX * HD, np.float32)
        ctx.rope_scaled_table(10000.0, HD, CTX, self.table)

    def norm8(self, x, rows, gain, residual=None):
        """8-bit rows of the norm of x + residual (kept there)."""
        ctx = self.ctx
        xv = x.read().reshape(rows, DIM).astype(np.float64)
        rv = None if residual is None else residual.read().reshape(rows, DIM).astype(np.float64)
        out, scale = ctx.empty(rows * DIM, np.uint8), ctx.empty(rows * 2, np.float32)
        ctx.rmsnorm_rows(x, "f32", rows, DIM, gain, EPS, out, "int8", residual=residual, residual_type="f32", sum=residual, scale=scale, group=128)
        h, y = R.norm(xv, rv, "f32", gain.read(), EPS) if rv is not None else R.norm(xv, None, "f32", gain.read().view(np.float16), EPS)
        s, q = R.to_eight(y, "int8", 128)
        assert np.array_equal(scale.read().reshape(rows, 2), s) and np.array_equal(out.read().view(np.int8).reshape(rows, DIM), q)
        if rv is not None:
            assert np.array_equal(residual.read().reshape(rows, DIM), h)
        return out, scale, q * R.spread(s, 128, DIM)

    def mul(self, matrix, v, x, rows, xv, type="int8", scale=None):
        y = self.ctx.empty(rows * len(v), np.float32)
        matrix.mul(x, type, rows, y, "f32", x_scale=scale, x_group=128 if scale else 0)
        P.close(y.read().reshape(rows, -1).astype(np.float64), xv @ v.T, R.product_bound(xv, v), "f32")
        return y

    def logits(self, tokens, pos):
        """Target logits [2][n][VOCAB] (device) of tokens [2][n] at pos[s] and on."""
        ctx = self.ctx
        S, n = tokens.shape
        rows = S * n
        h = ctx.upload(self.embed[tokens.reshape(-1)].astype(np.float32))
        dpos = ctx.upload(np.asarray(pos, np.int32))
        tpos = ctx.upload((np.asarray(pos)[:, None] + np.arange(n)).astype(np.int32).reshape(-1))
        delta = None
        for layer in self.layers:
            if delta is None:
                x, s, xv = self.norm8(h, rows, layer.gains[0])
            else:
                x, s, xv = self.norm8(delta, rows, layer.gains[0], h)
            qkv = self.mul(layer.m["qkv"], layer.v["qkv"], x, rows, xv, scale=s)
            width = (HEADS + 2 * KV) * HD
            ctx.rope_tokens(qkv, "f32", rows, HEADS + KV, HD, HD, "half", self.table, CTX, tpos, qkv, x_stride=width, out_stride=width)
            k, v = qkv.ptr + HEADS * HD * 4, qkv.ptr + (HEADS + KV) * HD * 4
            layer.cache.append(k, v, "f32", n, dpos, stride=width)
            a = ctx.empty(rows * HEADS * HD, np.float32)
            layer.cache.attention(qkv, "f32", HEADS, n, dpos, a, q_stride=width)
            av = a.read().reshape(rows, -1).astype(np.float64)
            assert np.isfinite(av).all()
            delta = self.mul(layer.m["o"], layer.v["o"], a, rows, av, "f32")
            x, s, xv = self.norm8(delta, rows, layer.gains[1], h)
            up = self.mul(layer.m["up"], layer.v["up"], x, rows, xv, scale=s)
            act = ctx.empty(rows * FFN, np.float32)
            for r in range(rows):
                at = up.ptr + r * 2 * FFN * 4
                ctx.silu_mul(at, at + FFN * 4, FFN, act.ptr + r * FFN * 4)
            actv = act.read().reshape(rows, FFN).astype(np.float64)
            delta = self.mul(layer.m["down"], layer.v["down"], act, rows, actv, "f32")
        x, s, xv = self.norm8(delta, rows, self.gain, h)
        return self.mul(self.head, self.head_v, x, rows, xv, scale=s)

    def verify(self, logits, drafts, uniform, temperature, count=None):
        ctx = self.ctx
        S, n = drafts.shape
        out, acc = ctx.empty(S * (n + 1), np.int32), ctx.empty(S, np.int32)
        ctx.verify_drafts(logits, "f32", S, n, VOCAB, ctx.upload(drafts.astype(np.int32)), ctx.upload(uniform), out, acc, temperature=temperature,
                          count=None if count is None else ctx.upload(np.asarray(count, np.int32)))
        want, want_acc = R.verify(logits.read().reshape(S, n + 1, VOCAB).astype(np.float64), None, drafts, count, uniform, temperature)
        assert np.array_equal(out.read().reshape(S, n + 1), want) and np.array_equal(acc.read(), want_acc)
        return want, want_acc


def test_step(iam):
    """Greedy tokens one by one, then the same tokens drafted: those that are
    right are kept up to the first wrong one, and the step goes on behind them."""
    with iam.Ctx(0) as ctx:
        step = Step(iam, ctx)
        rng = np.random.default_rng(1)
        prompt = rng.integers(0, VOCAB, (2, 70))
        u = rng.random((2, 6)).astype(np.float32)
        none = np.zeros((2, 0), np.int32)

        first = step.logits(prompt, [0, 0]).read().reshape(2, 70, VOCAB)[:, -1]
        token = first.argmax(1)
        alone = [token]
        for i in range(5):
            t, _ = step.verify(step.logits(alone[-1][:, None], [70 + i] * 2), none, u[:, :1].copy(), 0.0)
            alone.append(t[:, 0])
        alone = np.stack(alone, 1)                       # [2][6]

        # back to the position behind the prompt, with drafts; sequence 1's third is wrong
        drafts = alone[:, 1:].copy()
        drafts[1, 2] = (drafts[1, 2] + 1) % VOCAB
        logits = step.logits(np.concatenate((alone[:, :1], drafts), 1), [70, 70])
        got, kept = step.verify(logits, drafts, u, 0.0)
        x = logits.read().reshape(2, 6, VOCAB)
        # the chunk's attention reads the open block's tokens in one order, a
        # single token's in another: tokens may differ only where the two
        # largest logits nearly tie
        for s in range(2):
            top = np.sort(x[s], 1)
            clear = top[:, -1] - top[:, -2] > 0.05
            right = 5 if s == 0 else 2
            if clear[:right].all():
                assert kept[s] >= right and got[s, :right].tolist() == drafts[s, :right].tolist()
            if s == 1 and clear[:3].all():
                assert kept[s] == 2 and got[s, 2] == alone[1, 3]
        # the same logits with given random numbers, some sequences shorter
        step.verify(logits, drafts, u, 0.8)
        step.verify(logits, drafts, u, 1.0, [3, 5])
        # on from behind what was kept
        token = got[[0, 1], kept]
        step.logits(token[:, None], 71 + kept)
