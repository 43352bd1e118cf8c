// Matrices of 4-bit weights: laying them out, rounding to them, reading them back.
#include "q4.h"

namespace iam {

constexpr int kQ4Threads = 256;

struct PackArgs {
    Q4 m;
    uint32_t* words;
    uint16_t* scales;
    uint8_t* zeros;
    const uint8_t* n;          // plain numbers, two a byte
    const uint16_t* scale;     // plain scales
    const uint8_t* zero;
};

// Eight inputs of a row are one word of the layout and four bytes of the plain
// rows.  A workgroup takes 512 inputs of 16 rows: 4 KB, each read as it lies
// (64 threads a row's 256 bytes) and written through LDS in whole lines.
__global__ __launch_bounds__(kQ4Threads) void k_q4_pack(PackArgs a)
{
    __shared__ uint32_t words[4 * kTile * kStrip / 8];
    const int strip = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    const int tiles = min(4, a.m.tiles - chunk * 4);
    const size_t row_bytes = (size_t)(a.m.in + 1) / 2;
    for (int i = tid; i < kStrip * 64; i += kQ4Threads) {
        const int r = i / 64, k = (i % 64) * 8, o = strip * kStrip + r;
        uint32_t w = 0;
        if (o < a.m.out) {
            const uint8_t* src = a.n + (size_t)o * row_bytes;
            for (int b = 0; b < 4; b++) {
                const int at = chunk * kChunk + k + 2 * b;
                const uint32_t two = at < a.m.in ? src[at / 2] : 0x88u;
                const uint32_t hi = at + 1 < a.m.in ? two >> 4 : 8u;
                w |= (two & 15u) << (4 * b) | hi << (16 + 4 * b);
            }
            w ^= 0x88888888u;
        }
        words[((k / kTile) * 64 + k % 32 / 8 * 16 + r) * 4 + k % kTile / 32] = w;
    }
    __syncthreads();
    uint32_t* out = a.words + ((size_t)strip * a.m.tiles + chunk * 4) * 256;
    for (int i = tid; i < tiles * 256; i += kQ4Threads) out[i] = words[i];
    const int per = kChunk / a.m.group, groups = (a.m.in + a.m.group - 1) / a.m.group;
    for (int i = tid; i < kStrip * per; i += kQ4Threads) {
        const int r = i / per, g = i % per, o = strip * kStrip + r, k = chunk * kChunk + g * a.m.group;
        const bool there = o < a.m.out && k < a.m.in;
        const size_t from = (size_t)o * groups + k / a.m.group;
        a.scales[q4_scale(a.m, o, k)] = there ? a.scale[from] : (uint16_t)0;
        if (a.zeros) a.zeros[q4_zero(a.m, o, k)] = there ? (uint8_t)min((int)a.zero[from], 15) : (uint8_t)0;
    }
}

struct QuantArgs {
    Q4 m;
    uint32_t* words;
    uint16_t* scales;
    uint8_t* zeros;
    const void* w;
    size_t stride;
};

// One thread rounds one group of a row.  Once for a matrix: not a hot path.
template <typename T>
__global__ __launch_bounds__(kQ4Threads) void k_q4_quantize(QuantArgs a)
{
    const int per = kChunk / a.m.group, all = a.m.chunks * per;
    const size_t i = (size_t)blockIdx.x * kQ4Threads + threadIdx.x;
    // neighbours are rows of a strip: their words lie side by side
    const int r = (int)(i % kStrip), o = (int)(i / kStrip / all) * kStrip + r, k0 = (int)(i / kStrip % all) * a.m.group;
    if (o >= q4_strips(a.m.out) * kStrip) return;
    const bool there = o < a.m.out && k0 < a.m.in;
    const int n = there ? min(a.m.group, a.m.in - k0) : 0;
    const T* w = reinterpret_cast<const T*>(a.w) + (there ? (size_t)o * a.stride + k0 : 0);
    float low = 0.0f, high = 0.0f;
    bool finite = true;
    for (int e = 0; e < n; e++) {
        const float v = to_f32(w[e]);
        finite = finite && fabsf(v) < INFINITY;
        low = fminf(low, v);
        high = fmaxf(high, v);
    }
    const _Float16 h = (_Float16)(a.zeros ? (high - low) / 15.0f : fmaxf(high, -low) / 7.0f);
    const float s = (float)h;
    finite = finite && s < INFINITY;
    const bool live = finite && s > 0.0f;
    const int zero = a.zeros ? (live ? (int)fminf(fmaxf(rintf(-low / s), 0.0f), 15.0f) : 0) : 8;
    a.scales[q4_scale(a.m, o, k0)] = there ? (finite ? __builtin_bit_cast(uint16_t, h) : (uint16_t)0x7e00) : (uint16_t)0;
    if (a.zeros) a.zeros[q4_zero(a.m, o, k0)] = (uint8_t)zero;
    for (int e = 0; e < a.m.group && k0 + e < a.m.tiles * kTile; e += 8) {
        uint32_t word = 0;
        for (int j = 0; j < 8; j++) {
            if (e + j >= n) continue;
            const int q = live ? (int)fminf(fmaxf(rintf(to_f32(w[e + j]) / s) + (float)zero, 0.0f), 15.0f) : zero;
            word |= (uint32_t)(q ^ 8) << q4_shift(j);
        }
        a.words[q4_word(a.m, o, k0 + e)] = word;
    }
}

__global__ __launch_bounds__(kQ4Threads) void k_q4_read(Q4 m, int first, size_t values, float* out)
{
    for (size_t i = (size_t)blockIdx.x * kQ4Threads + threadIdx.x; i < values; i += (size_t)gridDim.x * kQ4Threads) {
        const int o = first + (int)(i / m.in), k = (int)(i % m.in);
        const uint32_t w = reinterpret_cast<const uint32_t*>(m.numbers)[q4_word(m, o, k)];
        const int n = (int)(w >> q4_shift(k) & 15u) ^ 8, z = m.zeros ? m.zeros[q4_zero(m, o, k)] : 8;
        out[i] = (float)__builtin_bit_cast(_Float16, m.scales[q4_scale(m, o, k)]) * (float)(n - z);
    }
}

// ------------------------------------------------------------------ host ---
Q4Bytes q4_bytes(int out, int in, int group)
{
    const size_t strips = (size_t)q4_strips(out), chunks = (size_t)q4_chunks(in), per = (size_t)(kChunk / group);
    return {strips * q4_tiles(in) * 1024, strips * chunks * per * kStrip * 2, strips * chunks * per * kStrip};
}

static int q4_shape(int out, int in, int group)
{
    IAM_REQUIRE(out >= 1 && out <= (1 << 24) && in >= 1 && in <= (1 << 20), "q4: out_dim must be 1 to 2^24, in_dim 1 to 2^20");
    IAM_REQUIRE(group == 32 || group == 64 || group == 128, "q4: group must be 32, 64 or 128");
    return IAM_OK;
}

int q4_check(Ctx* c, const iam_q4_matrix* m, const char* what)
{
    if (!m->numbers || !m->scales) return fail(IAM_E_INVALID, std::string(what) + ": null part of the matrix");
    IAM_TRY(q4_shape(m->out_dim, m->in_dim, m->group));
    const Q4Bytes b = q4_bytes(m->out_dim, m->in_dim, m->group);
    IAM_REQUIRE(aligned(m->numbers, 16) && aligned(m->scales, 16) && aligned(m->zeros, 16),
                std::string(what) + ": the matrix's parts must be 16-byte aligned");
    IAM_TRY(check_dev_range(c, m->numbers, b.numbers, "q4 numbers"));
    IAM_TRY(check_dev_range(c, m->scales, b.scales, "q4 scales"));
    if (m->zeros) IAM_TRY(check_dev_range(c, m->zeros, b.zeros, "q4 zeros"));
    IAM_REQUIRE(!overlaps(m->numbers, b.numbers, m->scales, b.scales) &&
                    !(m->zeros && (overlaps(m->numbers, b.numbers, m->zeros, b.zeros) || overlaps(m->scales, b.scales, m->zeros, b.zeros))),
                std::string(what) + ": parts of the matrix overlap");
    return IAM_OK;
}

Q4 q4_of(const iam_q4_matrix* m)
{
    return {m->numbers, m->scales, m->zeros, m->out_dim, m->in_dim, m->group, q4_tiles(m->in_dim), q4_chunks(m->in_dim)};
}

bool q4_overlaps(const iam_q4_matrix* m, const void* p, size_t bytes)
{
    const Q4Bytes b = q4_bytes(m->out_dim, m->in_dim, m->group);
    return overlaps(m->numbers, b.numbers, p, bytes) || overlaps(m->scales, b.scales, p, bytes) ||
           (m->zeros && overlaps(m->zeros, b.zeros, p, bytes));
}

}  // namespace iam

using namespace iam;

extern "C" {

int iam_q4_size(int out, int in, int group, size_t* numbers, size_t* scales, size_t* zeros)
{
    IAM_TRY(q4_shape(out, in, group));
    const Q4Bytes b = q4_bytes(out, in, group);
    if (numbers) *numbers = b.numbers;
    if (scales) *scales = b.scales;
    if (zeros) *zeros = b.zeros;
    return IAM_OK;
}

int iam_q4_pack(iam_ctx* c, const iam_q4_matrix* m, const uint8_t* n, const uint16_t* scale, const uint8_t* zero)
{
    if (!c || !m || !n || !scale) return fail(IAM_E_INVALID, "q4_pack: null argument");
    IAM_TRY(q4_check(c, m, "q4_pack"));
    IAM_REQUIRE((m->zeros != nullptr) == (zero != nullptr), "q4_pack: zero points are given where the matrix has them");
    IAM_REQUIRE(aligned(scale, 2), "q4_pack: pointers must be aligned to their type");
    const size_t rows = (size_t)m->out_dim, groups = (size_t)(m->in_dim + m->group - 1) / m->group;
    struct {
        const void* p;
        size_t bytes;
        const char* what;
    } const part[] = {{n, rows * (((size_t)m->in_dim + 1) / 2), "q4_pack n"}, {scale, rows * groups * 2, "q4_pack scale"}, {zero, rows * groups, "q4_pack zero"}};
    for (const auto& s : part) {
        if (!s.p) continue;
        IAM_TRY(check_dev_range(c, s.p, s.bytes, s.what));
        IAM_REQUIRE(!q4_overlaps(m, s.p, s.bytes), "q4_pack: the matrix overlaps a source");
    }
    DeviceGuard on(c);
    PackArgs a{q4_of(m), reinterpret_cast<uint32_t*>(m->numbers), m->scales, m->zeros, n, scale, zero};
    // at most 2^22 workgroups (2^30 threads) a launch, 2^15 strips (of a grid's second dimension)
    const int strips = q4_strips(m->out_dim), most = std::min(1 << 15, (1 << 22) / a.m.chunks);
    for (int s0 = 0; s0 < strips; s0 += most) {
        PackArgs b = a;
        const size_t row0 = (size_t)s0 * kStrip;
        b.m.out -= (int)row0;
        b.words += (size_t)s0 * a.m.tiles * 256;
        b.scales += q4_scale(a.m, (int)row0, 0);
        if (b.zeros) b.zeros += q4_zero(a.m, (int)row0, 0);
        b.n += row0 * (((size_t)m->in_dim + 1) / 2);
        b.scale += row0 * groups;
        if (b.zero) b.zero += row0 * groups;
        IAM_TRY(launch(c, "q4_pack", k_q4_pack, dim3(a.m.chunks, std::min(most, strips - s0)), dim3(kQ4Threads), 0, b));
    }
    return IAM_OK;
}

int iam_q4_quantize(iam_ctx* c, const iam_q4_matrix* m, const void* w, int type, size_t stride)
{
    if (!c || !m || !w) return fail(IAM_E_INVALID, "q4_quantize: null argument");
    IAM_TRY(q4_check(c, m, "q4_quantize"));
    IAM_REQUIRE(is_float_type(type), "q4_quantize: unknown type");
    if (!stride) stride = (size_t)m->in_dim;
    IAM_REQUIRE(stride >= (size_t)m->in_dim && stride < ((size_t)1 << 40), "q4_quantize: the stride is smaller than a row");
    IAM_REQUIRE(aligned(w, type_bytes(type)), "q4_quantize: pointers must be aligned to their type");
    const size_t bytes = rows_bytes((size_t)m->out_dim, (size_t)m->in_dim, stride, type_bytes(type));
    IAM_TRY(check_dev_range(c, w, bytes, "q4_quantize w"));
    IAM_REQUIRE(!q4_overlaps(m, w, bytes), "q4_quantize: the matrix overlaps its source");
    DeviceGuard on(c);
    const QuantArgs a{q4_of(m), reinterpret_cast<uint32_t*>(m->numbers), m->scales, m->zeros, w, stride};
    // at most 2^22 workgroups (2^30 threads) a launch: whole strips
    const size_t per_strip = (size_t)a.m.chunks * (kChunk / m->group) * kStrip;
    const int strips = q4_strips(m->out_dim), most = (int)std::max<size_t>(1, ((size_t)1 << 30) / per_strip);
    for (int s0 = 0; s0 < strips; s0 += most) {
        QuantArgs b = a;
        const int n = std::min(most, strips - s0);
        const size_t row0 = (size_t)s0 * kStrip;
        b.m.out = std::min(a.m.out - (int)row0, n * kStrip);
        b.words += (size_t)s0 * a.m.tiles * 256;
        b.scales += q4_scale(a.m, (int)row0, 0);
        if (b.zeros) b.zeros += q4_zero(a.m, (int)row0, 0);
        b.w = reinterpret_cast<const uint8_t*>(w) + row0 * stride * type_bytes(type);
        const dim3 grid((unsigned)((per_strip * n + kQ4Threads - 1) / kQ4Threads));
        if (type == IAM_F32) IAM_TRY(launch(c, "q4_quantize", k_q4_quantize<float>, grid, dim3(kQ4Threads), 0, b));
        else if (type == IAM_F16) IAM_TRY(launch(c, "q4_quantize", k_q4_quantize<_Float16>, grid, dim3(kQ4Threads), 0, b));
        else IAM_TRY(launch(c, "q4_quantize", k_q4_quantize<__bf16>, grid, dim3(kQ4Threads), 0, b));
    }
    return IAM_OK;
}

int iam_q4_read(iam_ctx* c, const iam_q4_matrix* m, int first, int rows, float* out)
{
    if (!c || !m || !out) return fail(IAM_E_INVALID, "q4_read: null argument");
    IAM_TRY(q4_check(c, m, "q4_read"));
    IAM_REQUIRE(first >= 0 && rows >= 0 && first <= m->out_dim && rows <= m->out_dim - first, "q4_read: rows outside the matrix");
    IAM_REQUIRE(aligned(out, 4), "q4_read: pointers must be aligned to their type");
    if (rows == 0) return IAM_OK;
    const size_t values = (size_t)rows * m->in_dim;
    IAM_TRY(check_dev_range(c, out, values * 4, "q4_read out"));
    IAM_REQUIRE(!q4_overlaps(m, out, values * 4), "q4_read: out overlaps the matrix");
    DeviceGuard on(c);
    const size_t blocks = std::min<size_t>((values + kQ4Threads - 1) / kQ4Threads, 16384);
    return launch(c, "q4_read", k_q4_read, dim3((unsigned)blocks), dim3(kQ4Threads), 0, q4_of(m), first, values, out);
}

}  // extern "C"
