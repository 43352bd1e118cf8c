"""Argument checks of the long-context operators that need no device, and the
float64 forms' own roundings."""
import ctypes as C

import numpy as np

import plain64 as P


def test_null_contexts_are_refused(iam):
    L = iam.lib()
    p = 64
    assert L.iam_rope_tokens(None, p, 0, 1, 1, 64, 64, 0, 0, p, 1, p, p, 0) == iam.IAM_E_INVALID
    assert L.iam_rope_scaled_table(None, C.c_double(1e4), 64, 1, None, C.c_void_p(p)) == iam.IAM_E_INVALID
    assert L.iam_kv8_append(None, p, p, p, 0, 1, 0, p, None) == iam.IAM_E_INVALID
    assert L.iam_kv8_read(None, p, p, 1, p, p) == iam.IAM_E_INVALID
    assert L.iam_kv8_reset(None, C.c_void_p(p)) == iam.IAM_E_INVALID
    assert L.iam_attention_kv8(None, p, p, 0, 1, 1, 0, p, None, 0, 0.0, p, 0) == iam.IAM_E_INVALID
    assert L.iam_token_logprobs(None, p, 0, 1, 1, 0, p, p, None, 0, None, None) == iam.IAM_E_INVALID
    assert "null" in iam.last_error()


def test_cache_sizes(iam):
    a, b, c = C.c_size_t(), C.c_size_t(), C.c_size_t()
    iam.check(iam.lib().iam_kv8_size(3, 65, 2, 128, C.byref(a), C.byref(b), C.byref(c)))
    assert (a.value, b.value, c.value) == (3 * 2 * 2 * 64 * 128, 3 * 2 * 2 * 4, 3 * 2 * 64 * 128 * 2)
    iam.check(iam.lib().iam_kv8_size(65535, 1 << 24, 512, 256, C.byref(a), None, None))
    assert a.value == 65535 * (1 << 18) * 512 * 64 * 256
    for bad in ((0, 64, 1, 64), (1, 0, 1, 64), (1, 64, 0, 64), (1, 64, 1, 32), (1, 64, 1, 192), (-1, 64, 1, 64)):
        assert iam.lib().iam_kv8_size(*bad, None, None, None) == iam.IAM_E_INVALID


def test_plain_roundings():
    x = np.array([1.0, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, -2.0 ** -133, 3.4e38], np.float32)
    assert P.to_type(x, "bf16")[1].tolist() == [1.0, 1.0, 1.0 + 2.0 ** -6, -2.0 ** -133, np.inf]
    for format, top in (("int8", 127), ("e4m3", 448)):
        v, s = P.stands_for(np.full((64, 1, 4), 2.0, np.float16), format)
        assert s[0, 0] == np.float32(2.0) * (np.float32(1.0) / np.float32(top)) and (v == np.float32(top) * s[0, 0]).all()
    q, k = np.ones((1, 2, 4)), np.zeros((3, 1, 4))
    out, bound = P.attention(q, k, np.arange(12.0).reshape(3, 1, 4), 2)
    assert np.allclose(out[0, 1], [4, 5, 6, 7]) and (bound < 1e-4).all()
