"""Argument checks of the 4-bit products, the rows' norm and the verification of
drafted tokens that need no device, and the float64 forms' own roundings."""
import ctypes as C

import numpy as np

import plain_rows as R


def test_null_contexts_are_refused(iam):
    L, p = iam.lib(), 64
    assert L.iam_q4_pack(None, p, p, p, None) == iam.IAM_E_INVALID
    assert L.iam_q4_quantize(None, p, p, 0, 0) == iam.IAM_E_INVALID
    assert L.iam_q4_read(None, p, 0, 1, p) == iam.IAM_E_INVALID
    assert L.iam_q4_mul(None, p, p, 0, 0, None, 0, 1, p, 0, 0) == iam.IAM_E_INVALID
    assert L.iam_rmsnorm_rows(None, p, 0, 0, None, 0, 0, None, 1, 1, None, 0.0, p, 0, 0, None, 0) == iam.IAM_E_INVALID
    assert L.iam_rows8_read(None, p, 3, 0, p, 0, 1, 1, p) == iam.IAM_E_INVALID
    assert L.iam_verify_drafts(None, p, 0, 0, None, 0, 0, 1, 1, 1, 1.0, 1.0, p, None, p, p, p) == iam.IAM_E_INVALID
    assert "null" in iam.last_error()


def test_matrix_sizes(iam):
    a, b, c = C.c_size_t(), C.c_size_t(), C.c_size_t()
    iam.check(iam.lib().iam_q4_size(33, 513, 64, C.byref(a), C.byref(b), C.byref(c)))
    assert (a.value, b.value, c.value) == (3 * 5 * 1024, 3 * 2 * 8 * 16 * 2, 3 * 2 * 8 * 16)
    iam.check(iam.lib().iam_q4_size(1 << 24, 1 << 20, 32, C.byref(a), None, None))
    assert a.value == 1 << 43
    for bad in ((0, 1, 32), (1, 0, 32), (-1, 1, 32), (1, 1, 16), (1, 1, 0), ((1 << 24) + 1, 1, 32), (1, (1 << 20) + 1, 32)):
        assert iam.lib().iam_q4_size(*bad, None, None, None) == iam.IAM_E_INVALID


def test_plain_forms():
    b = np.arange(256)
    v = R.e4m3(b)
    fine = ~np.isnan(v)
    assert np.isnan(v).sum() == 2 and v[0x7e] == 448 and v[1] == 2.0 ** -9 and v[0x38] == 1
    assert np.array_equal(R.bytes_of(v[fine], "e4m3"), b[fine])
    w = R.quantize(np.array([[7, -7, 3.4, 0], [0, 0, 0, 0]]), 32, False)
    assert w.n.tolist() == [[15, 1, 11, 8], [8, 8, 8, 8]] and w.values()[0].tolist() == [7, -7, 3, 0]
    w = R.quantize(np.array([[-1, 14, 2, 0]]), 32, True)
    assert w.n.tolist() == [[0, 15, 3, 1]] and w.zero[0, 0] == 1 and w.values()[0].tolist() == [-1, 14, 2, 0]
    words, scales, zeros = R.layout(w)
    assert words[0, 0, 0, 0] == (0 ^ 8) | (3 ^ 8) << 4 | (15 ^ 8) << 16 | (1 ^ 8) << 20 and scales[0, 0, 0, 0, 0] == 1 and zeros[0, 0, 0, 0] == 1
    s, q = R.to_eight(np.array([[254.0, -1.0, 3.0, 0]]), "int8", 0)
    assert s[0, 0] == 2 and q[0].tolist() == [127, -0.0, 2, 0]
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.1, 0.2, 0.7]]]))
    for u, want in ((0.4, [0, 2]), (0.6, [2, -1])):
        out, a = R.verify(x, None, np.array([[0]]), None, np.array([[u, 0.6]], np.float32), 1.0)
        assert out[0].tolist() == want and a[0] == (u < 0.5)
