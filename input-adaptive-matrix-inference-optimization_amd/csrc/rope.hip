// Rotary positions of many tokens: the table with its scalings for long
// contexts, and the rotation in both pair layouts, of the whole head or of its
// first part.
#include <cmath>

#include "layer_ops.h"
#include "numbers.h"

namespace iam {

// ------------------------------------------------------------- the table ---
constexpr int kMaxPairs = 512;

struct RopeFreqs {
    double f[kMaxPairs];
};

// One thread per position and pair.  The angle, its cosine and its sine in
// fp64: at position 1e5 an fp32 angle is off by up to 4e-3 radians.
__global__ __launch_bounds__(256) void k_rope_table(const double* __restrict__ freqs, int pairs, int max_pos,
                                                    double magnitude, float2* __restrict__ table)
{
    const size_t n = (size_t)pairs * max_pos;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t pos = i / (unsigned)pairs;
        const double angle = (double)pos * freqs[i - pos * pairs];
        double s, c;
        sincos(angle, &s, &c);
        table[i] = make_float2((float)(c * magnitude), (float)(s * magnitude));
    }
}

// the angle of each pair for one position, and the rotation's factor
static void rope_freqs(double theta, int rot, const iam_rope_scaling& r, double* f, double* magnitude)
{
    const int pairs = rot / 2;
    const double two_pi = 2.0 * M_PI;
    double base = theta;
    if (r.kind == IAM_ROPE_SCALE_BASE && rot > 2) base = theta * std::pow(r.factor, (double)rot / (rot - 2));
    double lo = 0.0, hi = 0.0;   // RAMP: the pairs between which the mix runs
    if (r.kind == IAM_ROPE_SCALE_RAMP) {
        auto place = [&](double turns) {
            return rot * std::log(r.original_ctx / (two_pi * turns)) / (2.0 * std::log(theta));
        };
        lo = std::max(std::floor(place(r.high)), 0.0);
        hi = std::min(std::ceil(place(r.low)), rot - 1.0);
    }
    for (int i = 0; i < pairs; i++) {
        const double fi = std::pow(base, -2.0 * i / rot);
        double keep = 1.0;   // the share of the unscaled frequency
        if (r.kind == IAM_ROPE_SCALE_LINEAR) keep = 0.0;
        if (r.kind == IAM_ROPE_SCALE_BANDS)
            keep = std::min(std::max((r.original_ctx * fi / two_pi - r.low) / (r.high - r.low), 0.0), 1.0);
        if (r.kind == IAM_ROPE_SCALE_RAMP)
            keep = 1.0 - std::min(std::max((i - lo) / std::max(hi - lo, 1e-3), 0.0), 1.0);
        f[i] = keep == 1.0 ? fi : fi * keep + fi / r.factor * (1.0 - keep);
    }
    *magnitude = r.magnitude != 0.0 ? r.magnitude : r.kind == IAM_ROPE_SCALE_RAMP ? 0.1 * std::log(r.factor) + 1.0 : 1.0;
}

// ---------------------------------------------------------- the rotation ---
// Memory bound: every value is read and written once, a token's table row
// (rot/2 pairs of fp32) serves all its heads from the caches.  A thread takes
// VEC pairs of one head (its two runs of VEC values, or 2 * VEC neighbours)
// or, past the rotated part, 2 * VEC values to copy.  VEC makes a run 16
// bytes where the addresses allow it, else it is 1.  The arithmetic is
// rope_mx's (aux.cl:227-248), one IEEE operation at a time, so that a half
// layout over the whole head equals iam_rope bit for bit.
struct RopeArgs {
    const void* x;
    void* out;
    const float* table;
    const int* pos;
    size_t x_stride, out_stride;   // values between rows
    int tokens, head_dim, rot, max_pos;
    int units;        // threads per token: heads * head_dim / (2 * VEC)
    int per_head;     // of them per head
    int slice;        // tokens per grid row (slice * units < 2^31)
    int copy;         // the part that is not rotated is copied (not in place)
};

template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_rope_tokens(RopeArgs a)
{
#pragma clang fp contract(off)
    const unsigned n = blockIdx.x * 256u + threadIdx.x;
    const unsigned in_slice = n / (unsigned)a.units;
    const unsigned token = blockIdx.y * (unsigned)a.slice + in_slice;
    if (in_slice >= (unsigned)a.slice || token >= (unsigned)a.tokens) return;
    const unsigned u = n - in_slice * (unsigned)a.units;
    const unsigned head = u / (unsigned)a.per_head, v = u - head * (unsigned)a.per_head;
    const int pos = a.pos[token];
    if (pos < 0 || pos >= a.max_pos) return;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)token * a.x_stride + (size_t)head * a.head_dim;
    T* out = reinterpret_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * a.head_dim;
    const int half = a.rot / 2, i = (int)v * VEC;
    if (i >= half) {
        if (!a.copy) return;
        const int d = 2 * i;   // past the rotated part
        *reinterpret_cast<Pack<T, 2 * VEC, VEC * (int)sizeof(T)>*>(out + d) =
            *reinterpret_cast<const Pack<T, 2 * VEC, VEC * (int)sizeof(T)>*>(x + d);
        return;
    }
    const Pack<float, 2 * VEC, VEC == 1 ? 8 : 16> cs =
        *reinterpret_cast<const Pack<float, 2 * VEC, VEC == 1 ? 8 : 16>*>(a.table + (size_t)pos * a.rot + 2 * i);
    using Run = Pack<T, VEC>;
    float p[VEC], q[VEC];
    if constexpr (INTERLEAVED) {
        const Run r0 = *reinterpret_cast<const Run*>(x + 2 * i), r1 = *reinterpret_cast<const Run*>(x + 2 * i + VEC);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const int k0 = 2 * e, k1 = 2 * e + 1;
            p[e] = to_f32(k0 < VEC ? r0.v[k0 % VEC] : r1.v[k0 % VEC]);
            q[e] = to_f32(k1 < VEC ? r0.v[k1 % VEC] : r1.v[k1 % VEC]);
        }
    } else {
        const Run r0 = *reinterpret_cast<const Run*>(x + i), r1 = *reinterpret_cast<const Run*>(x + half + i);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            p[e] = to_f32(r0.v[e]);
            q[e] = to_f32(r1.v[e]);
        }
    }
    Run o0, o1;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float c = cs.v[2 * e], s = cs.v[2 * e + 1];
        const T y0 = from_f32<T>(__fsub_rn(__fmul_rn(p[e], c), __fmul_rn(q[e], s)));
        const T y1 = from_f32<T>(__fadd_rn(__fmul_rn(q[e], c), __fmul_rn(p[e], s)));
        if constexpr (INTERLEAVED) {
            (2 * e < VEC ? o0 : o1).v[(2 * e) % VEC] = y0;
            (2 * e + 1 < VEC ? o0 : o1).v[(2 * e + 1) % VEC] = y1;
        } else {
            o0.v[e] = y0;
            o1.v[e] = y1;
        }
    }
    if constexpr (INTERLEAVED) {
        *reinterpret_cast<Run*>(out + 2 * i) = o0;
        *reinterpret_cast<Run*>(out + 2 * i + VEC) = o1;
    } else {
        *reinterpret_cast<Run*>(out + i) = o0;
        *reinterpret_cast<Run*>(out + half + i) = o1;
    }
}

template <typename T, int VEC>
static int rope_launch(Ctx* c, RopeArgs a, int heads, int layout)
{
    a.per_head = a.head_dim / (2 * VEC);
    a.units = heads * a.per_head;
    a.slice = (int)std::min<int64_t>(a.tokens, ((int64_t)1 << 30) / a.units);
    const dim3 grid((unsigned)(((int64_t)a.slice * a.units + 255) / 256), (unsigned)((a.tokens + a.slice - 1) / a.slice));
    return layout == IAM_ROPE_HALF ? launch(c, "rope_tokens", k_rope_tokens<T, VEC, false>, grid, dim3(256), 0, a)
                                   : launch(c, "rope_tokens", k_rope_tokens<T, VEC, true>, grid, dim3(256), 0, a);
}

template <typename T>
static int rope_typed(Ctx* c, const RopeArgs& a, int heads, int layout)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    constexpr size_t B = sizeof(T);
    const bool wide = (a.rot / 2) % VEC == 0 && a.head_dim % (2 * VEC) == 0 && a.x_stride % VEC == 0 &&
                      a.out_stride % VEC == 0 && aligned(a.x, VEC * B) && aligned(a.out, VEC * B) &&
                      aligned(a.table, 16);
    return wide ? rope_launch<T, VEC>(c, a, heads, layout) : rope_launch<T, 1>(c, a, heads, layout);
}

}  // namespace iam

using namespace iam;

extern "C" {

int iam_rope_scaled_table(iam_ctx* c, double theta, int rot, int max_pos, const iam_rope_scaling* scaling,
                          float* table)
{
    if (!c || !table) return fail(IAM_E_INVALID, "rope_scaled_table: null argument");
    IAM_REQUIRE(rot >= 2 && rot % 2 == 0 && rot <= 2 * kMaxPairs, "rope_scaled_table: rot_dim must be even, 2 to 1024");
    IAM_REQUIRE(max_pos >= 1 && theta > 1.0 && std::isfinite(theta), "rope_scaled_table: max_pos must be at least 1, theta above 1");
    IAM_REQUIRE(aligned(table, 8), "rope_scaled_table: the table must be 8-byte aligned");
    iam_rope_scaling r{};
    if (scaling) r = *scaling;
    IAM_REQUIRE(r.kind >= IAM_ROPE_SCALE_NONE && r.kind <= IAM_ROPE_SCALE_RAMP, "rope_scaled_table: unknown scaling");
    IAM_REQUIRE(r.kind == IAM_ROPE_SCALE_NONE || (r.factor >= 1.0 && std::isfinite(r.factor)),
                "rope_scaled_table: factor must be at least 1");
    IAM_REQUIRE(r.kind < IAM_ROPE_SCALE_BANDS ||
                    (r.original_ctx >= 1.0 && r.low > 0.0 && r.high > r.low && std::isfinite(r.high) && std::isfinite(r.original_ctx)),
                "rope_scaled_table: original_ctx must be at least 1 and 0 < low < high");
    IAM_REQUIRE(std::isfinite(r.magnitude), "rope_scaled_table: magnitude must be finite");
    const size_t n = (size_t)max_pos * (rot / 2);
    IAM_TRY(check_dev_range(c, table, n * 8, "rope_scaled_table table"));
    IAM_REQUIRE(!c->capturing, "rope_scaled_table: not allowed during graph capture");
    DeviceGuard on(c);
    RopeFreqs f;
    double magnitude;
    rope_freqs(theta, rot, r, f.f, &magnitude);
    void* dev = nullptr;
    IAM_TRY(ctx_alloc(c, sizeof(double) * (rot / 2), &dev));
    int rc = IAM_OK;
    if (hipMemcpyAsync(dev, f.f, sizeof(double) * (rot / 2), hipMemcpyHostToDevice, c->stream) != hipSuccess)
        rc = fail(IAM_E_HIP, "rope_scaled_table: copy failed");
    if (rc == IAM_OK)
        rc = launch(c, "rope_table", k_rope_table, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, (const double*)dev,
                    rot / 2, max_pos, magnitude, reinterpret_cast<float2*>(table));
    if (hipStreamSynchronize(c->stream) != hipSuccess && rc == IAM_OK) rc = fail(IAM_E_HIP, "rope_scaled_table: sync failed");
    (void)ctx_free(c, dev);
    return rc;
}

int iam_rope_tokens(iam_ctx* c, const void* x, int type, int n_tokens, int n_heads, int head_dim, int rot, int layout,
                    size_t x_stride, const float* table, int max_pos, const int* pos, void* out, size_t out_stride)
{
    if (!c || !x || !table || !pos || !out) return fail(IAM_E_INVALID, "rope_tokens: null argument");
    IAM_REQUIRE(type == IAM_F32 || type == IAM_F16 || type == IAM_BF16, "rope_tokens: unknown type");
    IAM_REQUIRE(layout == IAM_ROPE_HALF || layout == IAM_ROPE_INTERLEAVED, "rope_tokens: unknown layout");
    IAM_REQUIRE(n_tokens >= 0 && n_heads >= 1 && n_heads <= 65536, "rope_tokens: n_tokens must not be negative, n_heads 1 to 65536");
    IAM_REQUIRE(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 8192, "rope_tokens: head_dim must be even, 2 to 8192");
    IAM_REQUIRE(rot >= 2 && rot % 2 == 0 && rot <= head_dim, "rope_tokens: rot_dim must be even, 2 to head_dim");
    IAM_REQUIRE(max_pos >= 1, "rope_tokens: max_pos must be at least 1");
    const size_t width = (size_t)n_heads * head_dim, B = type_bytes(type);
    if (!x_stride) x_stride = width;
    if (!out_stride) out_stride = width;
    IAM_REQUIRE(x_stride >= width && out_stride >= width && x_stride < ((size_t)1 << 40) && out_stride < ((size_t)1 << 40),
                "rope_tokens: a stride is smaller than a row");
    IAM_REQUIRE(aligned(x, B) && aligned(out, B) && aligned(table, 8) && aligned(pos, 4),
                "rope_tokens: x and out must be aligned to their type, the table to 8 bytes");
    if (n_tokens == 0) return IAM_OK;
    const size_t xb = rows_bytes(n_tokens, width, x_stride, B), ob = rows_bytes(n_tokens, width, out_stride, B);
    IAM_TRY(check_dev_range(c, x, xb, "rope_tokens x"));
    IAM_TRY(check_dev_range(c, out, ob, "rope_tokens out"));
    IAM_TRY(check_dev_range(c, table, (size_t)max_pos * rot * 4, "rope_tokens table"));
    IAM_TRY(check_dev_range(c, pos, (size_t)n_tokens * 4, "rope_tokens pos"));
    const bool in_place = x == out && x_stride == out_stride;
    IAM_REQUIRE(in_place || !overlaps(x, xb, out, ob), "rope_tokens: x and out overlap without being the same rows");
    IAM_REQUIRE(!overlaps(table, (size_t)max_pos * rot * 4, out, ob) && !overlaps(pos, (size_t)n_tokens * 4, out, ob),
                "rope_tokens: out overlaps the table or the positions");
    DeviceGuard on(c);
    RopeArgs a{};
    a.x = x;
    a.out = out;
    a.table = table;
    a.pos = pos;
    a.x_stride = x_stride;
    a.out_stride = out_stride;
    a.tokens = n_tokens;
    a.head_dim = head_dim;
    a.rot = rot;
    a.max_pos = max_pos;
    a.copy = !in_place;
    if (type == IAM_F32) return rope_typed<float>(c, a, n_heads, layout);
    if (type == IAM_F16) return rope_typed<_Float16>(c, a, n_heads, layout);
    return rope_typed<__bf16>(c, a, n_heads, layout);
}

}  // extern "C"
