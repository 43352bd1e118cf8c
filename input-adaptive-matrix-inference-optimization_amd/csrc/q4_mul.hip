// Products of rows with a matrix of 4-bit weights.
#include "q4_mul.h"

namespace iam {

constexpr int kMulThreads = 256;

// a value of a row: a float type's, or an 8-bit number's
template <typename T>
__device__ __forceinline__ float value_of(T v) { return to_f32(v); }
template <>
__device__ __forceinline__ float value_of<int8_t>(int8_t v) { return (float)v; }
template <>
__device__ __forceinline__ float value_of<uint8_t>(uint8_t v) { return e4m3_value(v); }   // e4m3

// A wave takes a strip of 16 rows for one row of x: lane 16 g + r the words of
// row r that lie in it.
template <typename T>
__global__ __launch_bounds__(kMulThreads) void k_q4_mul(MulArgs a)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int strips = q4_strips(a.m.out);
    const size_t w = (size_t)blockIdx.x * (kMulThreads / 64) + (threadIdx.x >> 6);
    if (w >= (size_t)strips * a.rows) return;
    const int strip = (int)(w % strips), row = (int)(w / strips), o = strip * kStrip + r;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.x_stride;
    const uint4* words = reinterpret_cast<const uint4*>(a.m.numbers) + (size_t)strip * a.m.tiles * 64 + lane;
    float sum = 0.0f;
    for (int t = 0; t < a.m.tiles; t++) {
        const uint4 q = words[(size_t)t * 64];
        const uint32_t wd[4] = {q.x, q.y, q.z, q.w};
        float tile = 0.0f;
        for (int j = 0; j < 4; j++) {
            const int k = t * kTile + 32 * j + 8 * g;
            const float s = (float)__builtin_bit_cast(_Float16, a.m.scales[q4_scale(a.m, o, k)]);
            const int z = a.m.zeros ? a.m.zeros[q4_zero(a.m, o, k)] : 8;
            float part = 0.0f;
            for (int e = 0; e < 8; e++)
                if (k + e < a.m.in) part += value_of<T>(x[k + e]) * (float)((int)((wd[j] >> q4_shift(e) & 15u) ^ 8u) - z);
            tile += part * s;
        }
        sum += a.x_scale ? tile * a.x_scale[(size_t)row * a.x_groups + (a.x_groups > 1 ? t : 0)] : tile;
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g == 0 && o < a.m.out) put_value(a.y, a.y_type, (size_t)row * a.y_stride + o, sum);
}

template <typename T>
static int mul_typed(Ctx* c, MulArgs a)
{
    const size_t waves = (size_t)q4_strips(a.m.out) * a.rows;
    return launch(c, "q4_mul", k_q4_mul<T>, dim3((unsigned)((waves + 3) / 4)), dim3(kMulThreads), 0, a);
}

}  // namespace iam

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
    if (rows <= q4_few_most(x_type)) return q4_mul_few(c, a);
    switch (x_type) {
    case IAM_F32: return mul_typed<float>(c, a);
    case IAM_F16: return mul_typed<_Float16>(c, a);
    case IAM_BF16: return mul_typed<__bf16>(c, a);
    case IAM_I8: return mul_typed<int8_t>(c, a);
    default: return mul_typed<uint8_t>(c, a);
    }
}
