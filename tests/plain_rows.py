"""Plain float64 forms of the 4-bit products, the rows' norm and the verification
of drafted tokens, in numpy.  Written from the definitions in include/iam.h;
nothing here calls the library."""
import numpy as np

import plain64 as P

TILE = 128
LARGEST = {"int8": 127.0, "e4m3": 448.0}
ROW_TYPES = P.TYPES + ("int8", "e4m3")


def bytes_of(q, type):
    """The bytes of numbers of an 8-bit type (exact ones)."""
    if type == "int8":
        return np.asarray(q).astype(np.int8).view(np.uint8)
    m = np.abs(q)
    e = np.where(m > 0, np.maximum(np.frexp(m)[1] - 1, -6), -6)
    n = np.rint(np.ldexp(m, 3 - e)).astype(np.int64)
    b = np.where((e == -6) & (n < 8), n, (e + 7) * 8 + n - 8)
    return (b | np.where(np.signbit(q), 0x80, 0)).astype(np.uint8)


def e4m3(b):
    """The values of e4m3 bytes."""
    b = np.asarray(b, np.int64)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.ldexp(1.0, np.maximum(e, 1) - 10))
    v = np.where((b & 0x7f) == 0x7f, np.nan, v)
    return np.where(b & 0x80, -v, v)


def values8(b, type):
    return np.asarray(b, np.uint8).view(np.int8).astype(np.float64) if type == "int8" else e4m3(b)


def spread(scale, group, dim):
    """[rows][groups] scales as [rows][dim]."""
    return np.repeat(np.asarray(scale, np.float64), group or dim, 1)[:, :dim]


# --------------------------------------------------------- 4-bit weights --

class Weights:
    """A matrix: numbers 0 .. 15, fp16 scales and zero points (or None)."""

    def __init__(self, n, scale, zero, group):
        self.n, self.scale, self.zero, self.group = n, np.asarray(scale, np.float16), zero, group
        self.out, self.inp = n.shape

    def values(self):
        z = 8 if self.zero is None else np.repeat(self.zero.astype(np.float64), self.group, 1)[:, :self.inp]
        s = np.repeat(self.scale.astype(np.float64), self.group, 1)[:, :self.inp]
        return s * (self.n - z)

    def plain_bytes(self):
        n = np.pad(self.n, ((0, 0), (0, self.inp % 2))).astype(np.uint8)
        return np.ascontiguousarray(n[:, 0::2] | n[:, 1::2] << 4)


def random_weights(rng, out, inp, group, zeros):
    groups = (inp + group - 1) // group
    return Weights(rng.integers(0, 16, (out, inp)), rng.uniform(0.5, 2, (out, groups)) * 0.01,
                   rng.integers(0, 16, (out, groups)).astype(np.uint8) if zeros else None, group)


def layout(w):
    """The bytes of the parts numbers, scales, zeros in the order the header states."""
    out, inp, G = w.out, w.inp, w.group
    strips, tiles, chunks, per = -(-out // 16), -(-inp // 128), -(-inp // 512), 512 // G
    words = np.zeros((strips, tiles, 64, 4), np.uint32)
    order = [0, 2, 4, 6, 1, 3, 5, 7]
    for o in range(out):
        for k in range(inp):
            j, g, e = k % 128 // 32, k % 32 // 8, k % 8
            words[o // 16, k // 128, 16 * g + o % 16, j] |= np.uint32((int(w.n[o, k]) ^ 8) << 4 * order.index(e))
    scales = np.zeros((strips, chunks, 4, per, 4), np.float16)
    zeros = np.zeros((strips, chunks, 16, per), np.uint8)
    for o in range(out):
        for g in range(w.scale.shape[1]):
            scales[o // 16, g // per, o % 16 // 4, g % per, o % 4] = w.scale[o, g]
            if w.zero is not None:
                zeros[o // 16, g // per, o % 16, g % per] = w.zero[o, g]
    return words, scales, zeros


def quantize(w, group, zeros):
    """(n, scale, zero) of the header's rounding, quotients in fp32."""
    w = np.asarray(w, np.float32)
    out, inp = w.shape
    groups = -(-inp // group)
    n = np.zeros((out, inp), np.int64)
    scale, zero = np.zeros((out, groups), np.float16), np.zeros((out, groups), np.uint8)
    for o in range(out):
        for g in range(groups):
            x = w[o, g * group:(g + 1) * group]
            low, high = min(x.min(), np.float32(0)), max(x.max(), np.float32(0))
            with np.errstate(over="ignore"):
                s = np.float16((high - low) / np.float32(15) if zeros else max(high, -low) / np.float32(7))
            z = np.float32(8)
            if zeros:
                z = np.float32(np.clip(np.rint(-low / np.float32(s)), 0, 15)) if s > 0 else np.float32(0)
            q = np.rint(x / np.float32(s)) + z if s > 0 else np.full_like(x, z)
            n[o, g * group:(g + 1) * group] = np.clip(q, 0, 15)
            scale[o, g], zero[o, g] = s, z
    return Weights(n, scale, zero if zeros else None, group)


def product_bound(x, w):
    """How far y = x w^T (float64) may be off before its rounding, at most:

    - a float x enters as whole numbers of 22 bits of its tile's largest value
      (half a unit: 2^-22 of that value), or in two fp16 parts (2^-22 of each
      value and 2^-40 of the row's largest): 2^-21 of the tile's largest value
      times |w| covers either, the row's part added;
    - whole-number (or fp16 times 4-bit) products are exact, their sums over a
      tile exact or fp32; over tiles, digits and waves they are fp32 additions
      of terms whose magnitudes add up to at most 3 |x| |w| (a digit's carry
      doubles what it carries over), each after two roundings of its scale:
      (tiles + 128 + 32) 2^-24 of them."""
    rows, inp = x.shape
    tiles = -(-inp // TILE)
    pad = ((0, 0), (0, tiles * TILE - inp))
    top = np.abs(np.pad(x, pad)).reshape(rows, tiles, TILE).max(2)
    wsum = np.abs(np.pad(w, pad)).reshape(len(w), tiles, TILE).sum(2)
    return (2.0 ** -21 * top @ wsum.T + 2.0 ** -40 * top.max(1, keepdims=True) * wsum.sum(1)
            + 3 * (tiles + 160) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T))


# ------------------------------------------------------------------- norm --

def norm(x, r, r_type, gain, eps):
    """(h as it is kept, y in float64) of rows x, r (float64 values of their types)."""
    h = x.copy()
    if r is not None:
        h = P.to_type((x.astype(np.float32) + r.astype(np.float32)), r_type)[1]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        inv = 1 / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(eps)))
        y = h * inv * (1.0 if gain is None else gain.astype(np.float64))
    return h, y


def to_eight(y, type, group):
    """(scales, numbers as float64) of rows y."""
    rows, dim = y.shape
    g = group or dim
    scale, q = np.zeros((rows, -(-dim // g)), np.float32), np.zeros_like(y)
    for i in range(scale.shape[1]):
        b = y[:, i * g:(i + 1) * g]
        fine = np.isfinite(b).all(1)
        top = np.abs(np.where(np.isfinite(b), b, 0)).max(1)
        scale[:, i] = np.where(fine, top / LARGEST[type], np.nan)
        s = np.where(scale[:, i] > 0, scale[:, i], 1).astype(np.float64)[:, None]
        v = P.numbers(np.where(np.isfinite(b), b, 0) / s, type)
        q[:, i * g:(i + 1) * g] = np.where(scale[:, i:i + 1] > 0, np.clip(v, -LARGEST[type], LARGEST[type]), 0)
    return scale, q


# ----------------------------------------------------------------- verify --

def softmax(x, t):
    """The distribution of a row, or None."""
    m = x.max() if not np.isnan(x).any() else np.nan
    if not np.isfinite(m):
        return None
    e = np.exp((x - m) / t)
    return e / e.sum()


def verify(target, draft, tokens, count, uniform, temperature, draft_temperature=None):
    """(out [S][n + 1], accepted [S]) of float64 logits target [S][n + 1][V], draft
    [S][n][V] or None."""
    S, n1, V = target.shape
    n = n1 - 1
    out, accepted = np.full((S, n1), -1, np.int32), np.zeros(S, np.int32)
    td = temperature if draft_temperature is None else draft_temperature
    for s in range(S):
        m = n if count is None else min(max(int(count[s]), 0), n)
        for i in range(m + 1):
            x = target[s, i]
            t = int(tokens[s, i]) if i < m else -1
            there = 0 <= t < V
            if temperature == 0:
                best = -1 if softmax(x, 1.0) is None else int(np.argmax(x))
                if i < m and best == t and there:
                    out[s, i] = t
                    continue
                out[s, i] = best
            else:
                p = softmax(x, temperature)
                q = None
                if i < m and there:
                    q = np.eye(1, V, t)[0] if draft is None else softmax(draft[s, i], td)
                if p is not None and q is not None and float(uniform[s, i]) * q[t] < p[t]:
                    out[s, i] = t
                    continue
                if p is not None:
                    r = p if q is None else np.maximum(p - q, 0)
                    r = r if r.sum() > 0 else p
                    c = np.cumsum(r)
                    at = np.nonzero(c > float(uniform[s, n]) * c[-1])[0]
                    out[s, i] = at[0] if len(at) else np.nonzero(r)[0][-1]
            accepted[s] = i
            break
    return out, accepted
