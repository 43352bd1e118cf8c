// The entry point of the products of rows with a matrix of 4-bit weights.
#include "q4_mul.h"

using namespace iam;

extern "C" int iam_q4_mul(iam_ctx* c, const iam_q4_matrix* m, const void* x, int x_type, size_t x_stride, const float* x_scale,
                          int x_group, int rows, void* y, int y_type, size_t y_stride)
{
    if (!c || !m || !x || !y) return fail(IAM_E_INVALID, "q4_mul: null argument");
    IAM_TRY(q4_check(c, m, "q4_mul"));
    IAM_REQUIRE(is_float_type(x_type) || is_8bit_type(x_type), "q4_mul: unknown type of x");
    IAM_REQUIRE(is_float_type(y_type), "q4_mul: y must be of a float type");
    IAM_REQUIRE(is_8bit_type(x_type) == (x_scale != nullptr), "q4_mul: rows in 8 bits come with scales, others without");
    IAM_REQUIRE(x_group == 0 || (x_scale && x_group == kTile), "q4_mul: x_group must be 0, or 128 for rows in 8 bits");
    IAM_REQUIRE(rows >= 0 && rows <= (1 << 22), "q4_mul: n_rows must be 0 to 2^22");
    const size_t xb = row_type_bytes(x_type), yb = type_bytes(y_type), in = (size_t)m->in_dim, out = (size_t)m->out_dim;
    if (!x_stride) x_stride = in;
    if (!y_stride) y_stride = out;
    IAM_REQUIRE(x_stride >= in && y_stride >= out && x_stride < ((size_t)1 << 40) && y_stride < ((size_t)1 << 40),
                "q4_mul: a stride is smaller than a row");
    IAM_REQUIRE(aligned(x, xb) && aligned(y, yb) && aligned(x_scale, 4), "q4_mul: pointers must be aligned to their type");
    if (rows == 0) return IAM_OK;
    const size_t n = (size_t)rows, x_groups = x_group ? (size_t)q4_tiles(m->in_dim) : 1;
    const size_t x_bytes = rows_bytes(n, in, x_stride, xb), y_bytes = rows_bytes(n, out, y_stride, yb);
    IAM_TRY(check_dev_range(c, x, x_bytes, "q4_mul x"));
    IAM_TRY(check_dev_range(c, y, y_bytes, "q4_mul y"));
    if (x_scale) IAM_TRY(check_dev_range(c, x_scale, n * x_groups * 4, "q4_mul x_scale"));
    IAM_REQUIRE(!overlaps(y, y_bytes, x, x_bytes) && !(x_scale && overlaps(y, y_bytes, x_scale, n * x_groups * 4)) &&
                    !q4_overlaps(m, y, y_bytes),
                "q4_mul: y overlaps an input");
    DeviceGuard on(c);
    MulArgs a{};
    a.m = q4_of(m);
    a.x = x;
    a.x_type = x_type;
    a.x_stride = x_stride;
    a.x_scale = x_scale;
    a.x_groups = (int)x_groups;
    a.rows = rows;
    a.y = y;
    a.y_type = y_type;
    a.y_stride = y_stride;
    return q4_takes_few(a) ? q4_mul_few(c, a) : q4_mul_rows(c, a);
}
