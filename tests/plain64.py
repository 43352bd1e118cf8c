"""Plain float64 forms of the long-context operators, in numpy, and the number
types their inputs and outputs come in.  Written from the definitions in
include/iam.h; nothing here calls the library."""
import numpy as np

BLOCK = 64
# half a step of each type, relative to the value (torch.finfo(t).eps / 2)
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# the same for values under the normal range
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
TYPES = ("f32", "f16", "bf16")


def to_type(x, type):
    """The stored words of x rounded to the type, and the float64 values they
    stand for."""
    x32 = np.asarray(x, np.float32)
    if type == "f32":
        return x32, x32.astype(np.float64)
    if type == "f16":
        with np.errstate(over="ignore"):
            h = x32.astype(np.float16)
        return h, h.astype(np.float64)
    u = np.ascontiguousarray(x32).view(np.uint32).astype(np.uint64)
    w = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    w = np.where(np.isnan(x32), np.uint16(0x7FC0), w)
    return w, from_bits(w, "bf16")


def storage(type):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[type]


def from_bits(w, type):
    """float64 values of stored words."""
    if type == "bf16":
        return (np.asarray(w, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(w).astype(np.float64)


# ------------------------------------------------------------ 8-bit cache --

def numbers(q, format):
    """Quotients rounded to the format's numbers, nearest even."""
    if format == "int8":
        return np.rint(q)
    m, e = np.frexp(q)
    normal = np.ldexp(np.rint(m * 16) / 16, e)
    return np.where(np.abs(q) < 2.0 ** -6, np.rint(q * 512) / 512, normal)


def block_scale(x16, format):
    """The fp32 scale of one block of one head (x16 fp16)."""
    x = np.asarray(x16, np.float32)
    if not np.isfinite(x).all():
        return np.float32(np.nan)
    return np.abs(x).max() * (np.float32(1) / np.float32(127 if format == "int8" else 448))


def stands_for(x16, format):
    """fp32 values of a cache that holds the fp16 rows x16 [T][kv][dim], and the
    scales [T // 64][kv]."""
    T = x16.shape[0]
    out = x16.astype(np.float32)
    scales = np.zeros((T // BLOCK, x16.shape[1]), np.float32)
    for b in range(T // BLOCK):
        for h in range(x16.shape[1]):
            x = x16[b * BLOCK:(b + 1) * BLOCK, h]
            s = scales[b, h] = block_scale(x, format)
            if np.isnan(s):
                out[b * BLOCK:(b + 1) * BLOCK, h] = np.nan
            elif s == 0:
                out[b * BLOCK:(b + 1) * BLOCK, h] = 0
            else:
                n = numbers(x.astype(np.float64) / np.float64(s), format)
                out[b * BLOCK:(b + 1) * BLOCK, h] = n.astype(np.float32) * s
    return out, scales


def k_place(t, d, dim):
    return ((t // 16 * (dim // 64) + d // 64) * 64 + d % 64 // 16 * 16 + t % 16) * 16 + d % 16


def v_place(t, d, dim):
    return (d // 16 * 64 + t // 4 % 4 * 16 + d % 16) * 16 + t // 32 * 8 + t // 16 % 2 * 4 + t % 4


def attention(q, k, v, pos, window=0, scale=0.0):
    """q [n][heads][dim] at positions pos .. over k, v [T][kv][dim] (float64):
    (out, bound) where bound is how far an fp32 evaluation may be off:

    - a logit is a sum of dim products in fp32, of numbers held to 22 bits
      (q in two parts; the parts' products add one more sum), scaled by two
      factors: its error is at most (2 dim + 8) 2^-24 sum |q k| scale + 2^-22 of
      the same sum;
    - p = 2^x by an instruction good to 2^-22, x's own subtractions to 4 |s|
      2^-24, and p held to 21 bits;
    - the sums over T positions, block by block: (64 + T / 64 + 8) 2^-24, twice
      (over p v and over p), and the rescalings of the running maximum, one
      rounding each (T / 64 + 8 at most)."""
    n, heads, dim = q.shape
    T, kv = k.shape[:2]
    rep = heads // kv
    scale = scale or 1.0 / np.sqrt(dim)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for i in range(n):
        if pos < 0:
            continue
        p = min(pos + i, T - 1)
        lo = max(0, p - window + 1) if window > 0 else 0
        for h in range(heads):
            kk, vv = k[lo:p + 1, h // rep], v[lo:p + 1, h // rep]
            s = kk @ q[i, h] * scale
            size = (np.abs(kk) @ np.abs(q[i, h]) * scale).max() if len(s) else 0.0
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[i, h] = w @ vv
            m = len(s)
            ds = ((2 * dim + 8) * 2.0 ** -24 + 2.0 ** -22) * size + 8 * np.abs(s).max() * 2.0 ** -24
            rel = 2 * (ds + 2.0 ** -21) + 2 * (64 + 2 * (m / 64) + 16) * 2.0 ** -24
            bound[i, h] = rel * (w @ np.abs(vv)) + 2.0 ** -126
    return out, bound


def close(got, want, bound, type):
    """got (float64 values of the type) within bound and one rounding of want."""
    room = np.asarray(bound) + (np.abs(want) + bound) * HALF_STEP[type] + TINY[type]
    bad = ~(np.abs(got - want) <= room)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3], room[bad][:3])
