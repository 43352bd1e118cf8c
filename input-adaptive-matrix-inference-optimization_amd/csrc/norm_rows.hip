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

constexpr int kNormMaxThreads = 1024, kNormMaxWaves = 16;
constexpr int kNormMaxKept = 8;          // runs of 8 values that a thread keeps, at most

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

template <typename T>
struct Eight {
    T v[8];
};
// values i .. i + 7 of a row of n (zeros past it)
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int i, int n)
{
    if (i + 8 <= n) return __builtin_bit_cast(Eight<T>, *reinterpret_cast<const Pack<T, 8, (int)sizeof(T)>*>(p + i));
    Eight<T> r;
#pragma unroll
    for (int e = 0; e < 8; e++) r.v[e] = i + e < n ? p[i + e] : (T)0.0f;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_eight(T* p, int i, int n, const Eight<T>& x)
{
    if (i + 8 <= n) {
        *reinterpret_cast<Pack<T, 8, (int)sizeof(T)>*>(p + i) = __builtin_bit_cast(Pack<T, 8, (int)sizeof(T)>, x);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (i + e < n) p[i + e] = x.v[e];
}

// the workgroup's sum / largest value, in every thread (red: LDS, a place a wave)
__device__ __forceinline__ double block_sum(double v, double* red)
{
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    const int waves = blockDim.x >> 6;
    for (int w = 0; w < waves; w++) v += red[w];
    return v;
}
__device__ __forceinline__ double block_max(double v, double* red)
{
    v = wave_max_t(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    const int waves = blockDim.x >> 6;
    for (int w = 1; w < waves; w++) v = fmax(v, red[w]);
    return v;
}
// the largest of 16 neighbouring lanes', in each of them
__device__ __forceinline__ double max16(double v)
{
    v = fmax(v, dpp_t<0x128>(v, v));
    v = fmax(v, dpp_t<0x124>(v, v));
    v = fmax(v, dpp_t<0x122>(v, v));
    return fmax(v, dpp_t<0x121>(v, v));
}

// the magnitude of y, infinite where y is NaN
__device__ __forceinline__ double size_of(double y) { return y != y ? (double)INFINITY : fabs(y); }
// the scale of values whose largest magnitude is m: m / 127 or 448, NaN where one is not finite
__device__ __forceinline__ float scale_of(double m, int type)
{
    return m < (double)INFINITY ? (float)(m / (type == IAM_I8 ? 127.0 : 448.0)) : NAN;
}

// y / s for r = 1 / s: the product's error taken out
__device__ __forceinline__ double quotient(double y, double s, double r)
{
    const double q = y * r;
    return __builtin_fma(__builtin_fma(-q, s, y), r, q);
}
// q rounded to fp32 to odd: one more rounding to fewer bits is then right
// (infinities and NaN, whose e is NaN, as they are)
__device__ __forceinline__ float to_odd(double q)
{
    const float f = (float)q;
    const double e = q - (double)f;
    int b = __float_as_int(f);
    if (fabs(e) > 0.0 && !(b & 1)) b += (e > 0.0) == (q > 0.0) ? 1 : -1;
    return __int_as_float(b);
}
// (a scale of a few of the smallest fp32 numbers may be rounded to two thirds of what
// it should be: quotients then lie past the largest number, which the
// conversion would answer with NaN)
__device__ __forceinline__ uint32_t e4m3_of(double q)
{
    const float f = __builtin_amdgcn_fmed3f(to_odd(q), -448.0f, 448.0f);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, 0.0f, 0, false) & 0xffu;
}
__device__ __forceinline__ uint32_t int8_of(double q) { return (uint32_t)(int)rint(fmin(fmax(q, -127.0), 127.0)) & 0xffu; }

// the numbers of eight values, at p + i of a row of n
__device__ __forceinline__ void put_numbers(uint8_t* p, int i, int n, const double* y, float scale, int type)
{
    Eight<uint8_t> o;
    const double s = (double)scale, r = 1.0 / s;
    const bool live = scale > 0.0f;
    if (type == IAM_I8) {
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = live ? (uint8_t)int8_of(quotient(y[e], s, r)) : (uint8_t)0;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = live ? (uint8_t)e4m3_of(quotient(y[e], s, r)) : (uint8_t)0;
    }
    store_eight(p, i, n, o);
}
__device__ __forceinline__ void put_floats(void* p, size_t row, int i, int n, const double* y, int type)
{
    if (type == IAM_F32) {
        Eight<float> o;
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = (float)y[e];
        store_eight(reinterpret_cast<float*>(p) + row, i, n, o);
    } else if (type == IAM_F16) {
        Eight<_Float16> o;
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = (_Float16)to_odd(y[e]);
        store_eight(reinterpret_cast<_Float16*>(p) + row, i, n, o);
    } else {
        Eight<__bf16> o;
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = (__bf16)to_odd(y[e]);
        store_eight(reinterpret_cast<__bf16*>(p) + row, i, n, o);
    }
}

// h of eight values: x + r, rounded to R
template <typename X, typename R>
__device__ __forceinline__ void sum_eight(const NormArgs& a, size_t row, int i, float* h)
{
    const Eight<X> x = load_eight(reinterpret_cast<const X*>(a.x) + row * a.x_stride, i, a.dim);
    if (!a.r) {
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = to_f32(x.v[e]);
        return;
    }
    const Eight<R> r = load_eight(reinterpret_cast<const R*>(a.r) + row * a.r_stride, i, a.dim);
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = to_f32(from_f32<R>(to_f32(x.v[e]) + to_f32(r.v[e])));
}
template <typename R>
__device__ __forceinline__ void keep_eight(const NormArgs& a, size_t row, int i, const float* h)
{
    Eight<R> o;
#pragma unroll
    for (int e = 0; e < 8; e++) o.v[e] = from_f32<R>(h[e]);
    store_eight(reinterpret_cast<R*>(a.sum) + row * a.r_stride, i, a.dim, o);
}
__device__ __forceinline__ void gain_eight(const NormArgs& a, int i, const float* h, double inv, double* y)
{
    Eight<_Float16> g;
    if (a.gain) g = load_eight(reinterpret_cast<const _Float16*>(a.gain), i, a.dim);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        y[e] = (double)h[e] * inv;
        if (a.gain) y[e] *= (double)(float)g.v[e];
    }
}

// A workgroup takes a row, which stays in its registers: J runs of 8 values a
// thread.  Bound by memory where there are many rows (4096 of 4096, bf16 on an fp32
// residual that is kept, to e4m3: 43 us, 4.3 TB/s); one row by the launch and the
// two reductions (4.5 us).
template <typename X, typename R, int J>
__global__ __launch_bounds__(kNormMaxThreads) void k_rmsnorm_rows(NormArgs a)
{
    __shared__ double red[2][kNormMaxWaves];
    const size_t row = blockIdx.x;
    const int step = blockDim.x * 8, i0 = threadIdx.x * 8;
    float h[J][8];
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < J; j++) {
        if (J > 1 && i0 + j * step >= a.dim) {
#pragma unroll
            for (int e = 0; e < 8; e++) h[j][e] = 0.0f;
            continue;
        }
        sum_eight<X, R>(a, row, i0 + j * step, h[j]);
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fma((double)h[j][e], (double)h[j][e], ss);
        if (a.sum) keep_eight<R>(a, row, i0 + j * step, h[j]);
    }
    const double inv = 1.0 / sqrt(block_sum(ss, red[0]) / a.dim + (double)a.eps);
    if (!is_8bit_type(a.out_type)) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (i0 + j * step >= a.dim) continue;
            double y[8];
            gain_eight(a, i0 + j * step, h[j], inv, y);
            put_floats(a.out, row * a.out_stride, i0 + j * step, a.dim, y, a.out_type);
        }
        return;
    }
    uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + row * a.out_stride;
    if (a.group) {
        // 16 threads' runs are a group
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int i = i0 + j * step;
            double y[8], m = 0.0;
            if (i < a.dim) {
                gain_eight(a, i, h[j], inv, y);
#pragma unroll
                for (int e = 0; e < 8; e++) m = i + e < a.dim ? fmax(m, size_of(y[e])) : m;
            }
            const float scale = scale_of(max16(m), a.out_type);
            if (i >= a.dim) continue;
            if ((threadIdx.x & 15) == 0) a.scale[row * a.groups + i / 128] = scale;
            put_numbers(out, i, a.dim, y, scale, a.out_type);
        }
        return;
    }
    double m = 0.0;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int i = i0 + j * step;
        if (i >= a.dim) continue;
        double y[8];
        gain_eight(a, i, h[j], inv, y);
#pragma unroll
        for (int e = 0; e < 8; e++) m = i + e < a.dim ? fmax(m, size_of(y[e])) : m;
    }
    const float scale = scale_of(block_max(m, red[1]), a.out_type);
    if (threadIdx.x == 0) a.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int i = i0 + j * step;
        if (i >= a.dim) continue;
        double y[8];
        gain_eight(a, i, h[j], inv, y);
        put_numbers(out, i, a.dim, y, scale, a.out_type);
    }
}

// The same for rows that a workgroup's registers do not hold (over 65536
// values): two passes over x and the residual, three for 8 bits with one scale
// a row; h is kept in the last one, which reads a place before it writes there.
// 64 rows of 131072 fp32 values with residuals, to e4m3 by 128s: 74 us, 1.5 TB/s.
template <typename X, typename R>
__global__ __launch_bounds__(kNormMaxThreads) void k_rmsnorm_long(NormArgs a)
{
    __shared__ double red[2][kNormMaxWaves];
    const size_t row = blockIdx.x;
    const int step = kNormMaxThreads * 8, i0 = threadIdx.x * 8;
    double ss = 0.0;
    for (int i = i0; i < a.dim; i += step) {
        float h[8];
        sum_eight<X, R>(a, row, i, h);
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fma((double)h[e], (double)h[e], ss);
    }
    const double inv = 1.0 / sqrt(block_sum(ss, red[0]) / a.dim + (double)a.eps);
    const bool eight = is_8bit_type(a.out_type);
    float scale = 0.0f;
    if (eight && !a.group) {
        double m = 0.0;
        for (int i = i0; i < a.dim; i += step) {
            float h[8];
            double y[8];
            sum_eight<X, R>(a, row, i, h);
            gain_eight(a, i, h, inv, y);
#pragma unroll
            for (int e = 0; e < 8; e++) m = i + e < a.dim ? fmax(m, size_of(y[e])) : m;
        }
        scale = scale_of(block_max(m, red[1]), a.out_type);
        if (threadIdx.x == 0) a.scale[row] = scale;
    }
    uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + row * a.out_stride;
    const int rounds = (a.dim + step - 1) / step;
    for (int k = 0; k < rounds; k++) {
        const int i = i0 + k * step;
        float h[8];
        double y[8], m = 0.0;
        if (i < a.dim) {
            sum_eight<X, R>(a, row, i, h);
            gain_eight(a, i, h, inv, y);
            if (a.sum) keep_eight<R>(a, row, i, h);
#pragma unroll
            for (int e = 0; e < 8; e++) m = i + e < a.dim ? fmax(m, size_of(y[e])) : m;
        }
        if (eight && a.group) scale = scale_of(max16(m), a.out_type);
        if (i >= a.dim) continue;
        if (!eight) {
            put_floats(a.out, row * a.out_stride, i, a.dim, y, a.out_type);
            continue;
        }
        if (a.group && (threadIdx.x & 15) == 0) a.scale[row * a.groups + i / 128] = scale;
        put_numbers(out, i, a.dim, y, scale, a.out_type);
    }
}

struct Read8Args {
    const uint8_t* x;
    const float* scale;
    float* out;
    size_t stride;
    int dim, group, groups, type;
    int parts;               // workgroups of a row
};

constexpr int kReadThreads = 256;

__global__ __launch_bounds__(kReadThreads) void k_rows8_read(Read8Args a)
{
    const size_t row = blockIdx.x / a.parts;
    const int i = ((int)(blockIdx.x - row * a.parts) * kReadThreads + (int)threadIdx.x) * 8;
    if (i >= a.dim) return;
    const Eight<uint8_t> b = [&] {
        const uint8_t* p = a.x + row * a.stride;
        if (i + 8 <= a.dim) return __builtin_bit_cast(Eight<uint8_t>, *reinterpret_cast<const Pack<uint8_t, 8, 1>*>(p + i));
        Eight<uint8_t> r;
#pragma unroll
        for (int e = 0; e < 8; e++) r.v[e] = i + e < a.dim ? p[i + e] : (uint8_t)0;
        return r;
    }();
    const float s = a.scale[row * a.groups + (a.group ? i / 128 : 0)];
    Eight<float> o;
#pragma unroll
    for (int e = 0; e < 8; e++) o.v[e] = (a.type == IAM_I8 ? (float)(int8_t)b.v[e] : e4m3_value(b.v[e])) * s;
    store_eight(a.out + row * a.dim, i, a.dim, o);
}

// ------------------------------------------------------------------ host ---
template <typename X, typename R>
static int norm_launch(Ctx* c, const NormArgs& a, int rows)
{
    const dim3 grid((unsigned)rows);
    const int runs = (a.dim + 7) / 8;
    if (runs > kNormMaxThreads * kNormMaxKept) return launch(c, "rmsnorm_rows", k_rmsnorm_long<X, R>, grid, dim3(kNormMaxThreads), 0, a);
    // one run a thread, more where rows are long
    int j = 1;
    while (j < kNormMaxKept && runs > j * kNormMaxThreads) j *= 2;
    const dim3 block((unsigned)(((runs + j - 1) / j + 63) / 64 * 64));
    switch (j) {
    case 1: return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, R, 1>, grid, block, 0, a);
    case 2: return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, R, 2>, grid, block, 0, a);
    case 4: return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, R, 4>, grid, block, 0, a);
    default: return launch(c, "rmsnorm_rows", k_rmsnorm_rows<X, R, 8>, grid, block, 0, a);
    }
}

template <typename X>
static int norm_typed(Ctx* c, const NormArgs& a, int r_type, int rows)
{
    return r_type == IAM_F32 ? norm_launch<X, float>(c, a, rows) : norm_launch<X, X>(c, a, rows);
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
            // the residual's sum where the residual was, y where x was
            const bool in_place = (i == 4 && j == 1 && sum == r) || (i == 3 && j == 0 && out == x && out_type == type && out_stride == x_stride);
            IAM_REQUIRE(in_place || !overlaps(part[i].p, part[i].bytes, part[j].p, part[j].bytes),
                        "rmsnorm_rows: an output overlaps another array");
        }
    }
    DeviceGuard on(c);
    NormArgs a{x, r, sum, gain, out, scale, x_stride, r_stride, out_stride, dim, group, groups, out_type, eps};
    auto move = [](auto* p, size_t bytes) { return p ? decltype(p)(const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(p)) + bytes) : p; };
    // at most 2^20 rows (2^30 threads) a launch
    constexpr int kSlice = 1 << 20;
    for (int r0 = 0; r0 < rows; r0 += kSlice) {
        const int some = std::min(kSlice, rows - r0);
        if (type == IAM_F32) IAM_TRY(norm_typed<float>(c, a, r_type, some));
        else if (type == IAM_F16) IAM_TRY(norm_typed<_Float16>(c, a, r_type, some));
        else IAM_TRY(norm_typed<__bf16>(c, a, r_type, some));
        a.x = move(a.x, kSlice * x_stride * xb);
        a.r = move(a.r, kSlice * r_stride * rb);
        a.sum = move(a.sum, kSlice * r_stride * rb);
        a.out = move(a.out, kSlice * out_stride * ob);
        a.scale = move(a.scale, (size_t)kSlice * groups * 4);
    }
    return IAM_OK;
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
    const int parts = (dim + kReadThreads * 8 - 1) / (kReadThreads * 8);
    // at most 2^22 workgroups (2^30 threads) a launch
    const int most = (1 << 22) / parts;
    for (int r0 = 0; r0 < rows; r0 += most) {
        const Read8Args a{reinterpret_cast<const uint8_t*>(x) + (size_t)r0 * stride, scale + (size_t)r0 * groups, out + (size_t)r0 * d, stride, dim, group,
                          groups, type, parts};
        IAM_TRY(launch(c, "rows8_read", k_rows8_read, dim3((unsigned)(std::min(most, rows - r0) * parts)), dim3(kReadThreads), 0, a));
    }
    return IAM_OK;
}

}  // extern "C"
