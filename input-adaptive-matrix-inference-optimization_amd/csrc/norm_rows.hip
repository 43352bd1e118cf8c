// The root-mean-square norm of rows, with the residual's addition before it and
// results in float types or in 8 bits with scales.
//
//   h = x + r,   y = h / sqrt(sum h^2 / dim + eps) * gain,   number = round(y / scale)
//
// Everything from h on in fp64, so that a number next to the border between
// two 8-bit ones falls on its own side.
#include "q4.h"
#include "wave.h"

namespace iam {

constexpr int kNormThreads = 256, kNormWaves = 4;

struct NormArgs {
    const void* x;
    const void* r;           // may be null
    void* sum;               // may be null
    const uint16_t* gain;    // may be null
    void* out;
    float* scale;            // 8-bit results
    size_t x_stride, r_stride, out_stride;
    int dim, group, groups;  // group: values of a scale (0: the row)
    int out_type;
    float eps;
};

// the sum / largest value of the workgroup's, in every thread
__device__ __forceinline__ double block_sum(double v, double* red)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kNormWaves; w++) v += red[w];
    return v;
}

template <typename X, typename R>
__device__ __forceinline__ float norm_h(const NormArgs& a, size_t row, int i)
{
    const float x = to_f32(reinterpret_cast<const X*>(a.x)[row * a.x_stride + i]);
    if (!a.r) return x;
    return to_f32(from_f32<R>(x + to_f32(reinterpret_cast<const R*>(a.r)[row * a.r_stride + i])));
}

// the scale of values whose largest magnitude is m: m / 127 or 448, NaN where one is not finite
__device__ __forceinline__ float scale_of(double m, int type)
{
    return m < (double)INFINITY ? (float)(m / (type == IAM_I8 ? 127.0 : 448.0)) : NAN;
}
__device__ __forceinline__ uint8_t number8(double y, float scale, int type)
{
    if (!(scale > 0.0f)) return 0;
    const double q = y / (double)scale;
    if (type == IAM_I8) return (uint8_t)(int8_t)(int)fmin(fmax(rint(q), -127.0), 127.0);
    // e4m3: three bits behind the leading one, steps of 2^-9 at least
    const double m = fabs(q);
    int e = -6;
    if (m > 0.0) (void)frexp(m, &e);
    e = max(e - 1, -6);
    const int n = (int)rint(ldexp(m, 3 - e));   // 0 .. 16 steps of 2^(e - 3)
    int bits = e == -6 && n < 8 ? n : (e + 7) * 8 + (n - 8);   // 16 steps are the next exponent's first
    bits = min(bits, 0x7e);
    return (uint8_t)(bits | (q < 0.0 ? 0x80 : 0));
}

// A workgroup takes a row, in three passes over it.
template <typename X, typename R>
__global__ __launch_bounds__(kNormThreads) void k_rmsnorm_rows(NormArgs a)
{
    __shared__ double red[kNormWaves];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x;
    double ss = 0.0;
    for (int i = tid; i < a.dim; i += kNormThreads) {
        const double h = norm_h<X, R>(a, row, i);
        ss += h * h;
    }
    const double inv = 1.0 / sqrt(block_sum(ss, red) / a.dim + (double)a.eps);
    auto y_of = [&](int i) {
        const double g = a.gain ? (double)(float)__builtin_bit_cast(_Float16, a.gain[i]) : 1.0;
        return (double)norm_h<X, R>(a, row, i) * inv * g;
    };
    const bool eight = is_8bit_type(a.out_type);
    if (eight) {
        for (int g = tid >> 6; g < a.groups; g += kNormWaves) {
            const int k0 = g * a.group, k1 = a.group ? min(a.dim, k0 + a.group) : a.dim;
            double m = 0.0;
            for (int i = k0 + (tid & 63); i < k1; i += 64) {
                const double v = fabs(y_of(i));
                m = v > m || v != v ? v : m;
            }
            for (int d = 1; d < 64; d *= 2) {
                const double v = __shfl_xor(m, d);
                m = v > m || v != v ? v : m;
            }
            if ((tid & 63) == 0) a.scale[row * a.groups + g] = scale_of(m, a.out_type);
        }
        __syncthreads();
    }
    for (int i = tid; i < a.dim; i += kNormThreads) {
        const double y = y_of(i);
        const float h = norm_h<X, R>(a, row, i);
        if (a.sum) reinterpret_cast<R*>(a.sum)[row * a.r_stride + i] = from_f32<R>(h);
        const size_t at = row * a.out_stride + i;
        if (eight)
            reinterpret_cast<uint8_t*>(a.out)[at] = number8(y, a.scale[row * a.groups + (a.group ? i / a.group : 0)], a.out_type);
        else if (a.out_type == IAM_F32) reinterpret_cast<float*>(a.out)[at] = (float)y;
        else if (a.out_type == IAM_F16) reinterpret_cast<_Float16*>(a.out)[at] = (_Float16)y;
        else reinterpret_cast<__bf16*>(a.out)[at] = (__bf16)y;
    }
}

struct Read8Args {
    const uint8_t* x;
    const float* scale;
    float* out;
    size_t stride;
    int rows, dim, group, groups, type;
};

__global__ __launch_bounds__(256) void k_rows8_read(Read8Args a)
{
    const size_t all = (size_t)a.rows * a.dim;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        const size_t row = i / a.dim;
        const int k = (int)(i - row * a.dim);
        const uint8_t b = a.x[row * a.stride + k];
        const float v = a.type == IAM_I8 ? (float)(int8_t)b : e4m3_value(b);
        a.out[i] = v * a.scale[row * a.groups + (a.group ? k / a.group : 0)];
    }
}

template <typename X>
static int norm_typed(Ctx* c, const NormArgs& a, int r_type, int rows)
{
    const dim3 grid((unsigned)rows);
    if (r_type == IAM_F32) return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, float>, grid, dim3(kNormThreads), 0, a);
    return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, X>, grid, dim3(kNormThreads), 0, a);
}

}  // namespace iam

using namespace iam;

extern "C" {

int iam_rmsnorm_rows(iam_ctx* c, const void* x, int type, size_t x_stride, const void* r, int r_type, size_t r_stride, void* sum,
                     int rows, int dim, const uint16_t* gain, float eps, void* out, int out_type, size_t out_stride, float* scale,
                     int group)
{
    if (!c || !x || !out) return fail(IAM_E_INVALID, "rmsnorm_rows: null argument");
    IAM_REQUIRE(is_float_type(type), "rmsnorm_rows: unknown type of x");
    IAM_REQUIRE(is_float_type(out_type) || is_8bit_type(out_type), "rmsnorm_rows: unknown type of out");
    if (!r) r_type = type;
    IAM_REQUIRE(r_type == type || r_type == IAM_F32, "rmsnorm_rows: the residual must be of x's type or fp32");
    IAM_REQUIRE(rows >= 0 && rows <= (1 << 22) && dim >= 1 && dim <= (1 << 20), "rmsnorm_rows: n_rows must be 0 to 2^22, dim 1 to 2^20");
    const bool eight = is_8bit_type(out_type);
    IAM_REQUIRE(eight == (scale != nullptr), "rmsnorm_rows: results in 8 bits have scales, others have none");
    IAM_REQUIRE(group == 0 || (eight && group == 128), "rmsnorm_rows: group must be 0, or 128 for results in 8 bits");
    IAM_REQUIRE(eps >= 0.0f && eps < INFINITY, "rmsnorm_rows: eps must be finite and not negative");
    const size_t n = (size_t)rows, d = (size_t)dim, xb = type_bytes(type), rb = type_bytes(r_type), ob = row_type_bytes(out_type);
    if (!x_stride) x_stride = d;
    if (!r_stride) r_stride = d;
    if (!out_stride) out_stride = d;
    const size_t far = (size_t)1 << 40;
    IAM_REQUIRE(x_stride >= d && r_stride >= d && out_stride >= d && x_stride < far && r_stride < far && out_stride < far,
                "rmsnorm_rows: a stride is smaller than a row");
    IAM_REQUIRE(aligned(x, xb) && aligned(r, rb) && aligned(sum, rb) && aligned(gain, 2) && aligned(out, ob) && aligned(scale, 4),
                "rmsnorm_rows: pointers must be aligned to their type");
    if (rows == 0) return IAM_OK;
    const int groups = group ? (dim + group - 1) / group : 1;
    struct {
        const void* p;
        size_t bytes;
        const char* what;
        bool written;
    } const part[] = {{out, rows_bytes(n, d, out_stride, ob), "rmsnorm_rows out", true},
                      {sum, rows_bytes(n, d, r_stride, rb), "rmsnorm_rows sum", true},
                      {scale, n * groups * 4, "rmsnorm_rows scale", true},
                      {x, rows_bytes(n, d, x_stride, xb), "rmsnorm_rows x", false},
                      {r, rows_bytes(n, d, r_stride, rb), "rmsnorm_rows residual", false},
                      {gain, d * 2, "rmsnorm_rows gain", false}};
    for (int i = 0; i < 6; i++) {
        if (!part[i].p) continue;
        IAM_TRY(check_dev_range(c, part[i].p, part[i].bytes, part[i].what));
        for (int j = 0; j < i; j++) {
            if (!part[j].p || !part[j].written) continue;
            const bool in_place = (part[i].p == r && part[j].p == sum && sum == r) ||
                                  (part[i].p == x && part[j].p == out && out == x && out_type == type && out_stride == x_stride);
            IAM_REQUIRE(in_place || !overlaps(part[i].p, part[i].bytes, part[j].p, part[j].bytes),
                        "rmsnorm_rows: an output overlaps another array");
        }
    }
    DeviceGuard on(c);
    const NormArgs a{x, r, sum, gain, out, scale, x_stride, r_stride, out_stride, dim, group, groups, out_type, eps};
    if (type == IAM_F32) return norm_typed<float>(c, a, r_type, rows);
    if (type == IAM_F16) return norm_typed<_Float16>(c, a, r_type, rows);
    return norm_typed<__bf16>(c, a, r_type, rows);
}

int iam_rows8_read(iam_ctx* c, const void* x, int type, size_t stride, const float* scale, int group, int rows, int dim, float* out)
{
    if (!c || !x || !scale || !out) return fail(IAM_E_INVALID, "rows8_read: null argument");
    IAM_REQUIRE(is_8bit_type(type), "rows8_read: the type must be IAM_I8 or IAM_E4M3");
    IAM_REQUIRE(rows >= 0 && rows <= (1 << 22) && dim >= 1 && dim <= (1 << 20), "rows8_read: n_rows must be 0 to 2^22, dim 1 to 2^20");
    IAM_REQUIRE(group == 0 || group == 128, "rows8_read: group must be 0 or 128");
    const size_t n = (size_t)rows, d = (size_t)dim;
    if (!stride) stride = d;
    IAM_REQUIRE(stride >= d && stride < ((size_t)1 << 40), "rows8_read: the stride is smaller than a row");
    IAM_REQUIRE(aligned(scale, 4) && aligned(out, 4), "rows8_read: pointers must be aligned to their type");
    if (rows == 0) return IAM_OK;
    const int groups = group ? (dim + group - 1) / group : 1;
    const size_t xb = rows_bytes(n, d, stride, 1), sb = n * groups * 4, yb = n * d * 4;
    IAM_TRY(check_dev_range(c, x, xb, "rows8_read x"));
    IAM_TRY(check_dev_range(c, scale, sb, "rows8_read scale"));
    IAM_TRY(check_dev_range(c, out, yb, "rows8_read out"));
    IAM_REQUIRE(!overlaps(out, yb, x, xb) && !overlaps(out, yb, scale, sb), "rows8_read: out overlaps an input");
    DeviceGuard on(c);
    const Read8Args a{reinterpret_cast<const uint8_t*>(x), scale, out, stride, rows, dim, group, groups, type};
    const size_t blocks = std::min<size_t>((n * d + 255) / 256, 16384);
    return launch(c, "rows8_read", k_rows8_read, dim3((unsigned)blocks), dim3(256), 0, a);
}

}  // extern "C"
