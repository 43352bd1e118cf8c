// Products of a few rows (single tokens, drafted ones) with 4-bit weights.
//
// With the rows of x as whole numbers n = sum over d of 256^d n_d, the digits n_d
// signed bytes, and one power of two for each row and tile of 128 inputs:
//   y[r][o] = sum over d of 256^d  sum over tiles, groups of
//             (2^e[r][tile] scale[o][group]) * (sum over the group of n_d[r][k] (w[o][k] - zero))
// The innermost sums are exact, on the 8-bit matrix instructions, whose 16
// columns are the rows' digits: three of a row in 16 bits or e4m3 (22 bits of the
// tile's largest value and its sign), four of an fp32 row (30 bits: values from
// 2^-6 of the largest on enter whole), one of an int8 row.  4-bit weights become
// bytes with three instructions for eight of them, and four or five rows take no
// more matrix instructions than one.  One row of 28672 x 4096 (groups of 64, zero
// points) takes 13.0 us, 4.9 TB/s; bound by reads, and where there are few of them
// by the chain of x's loads, its digits, the weights' use and the waves' joining
// (4.3 us).  Four fp32 rows of 6144 x 4096 take 7.7 us.
#include "accum.h"
#include "q4_mul.h"

namespace iam {

struct FewArgs {
    MulArgs u;
    int waves;      // of a workgroup
    int rows;       // of a workgroup
    // the inputs cut into parts for more workgroups, whose sums the last one to arrive joins
    int splits;
    float* sums;
    uint32_t* ctr;  // zero on entry (left zero)
};

constexpr int kFewMaxWaves = 16;
constexpr int kFewCols = 16;
constexpr int kFewSplits = 8;
constexpr int kFewLds = 160 * 1024;

// A strip's words of a chunk, its scales and zero points, in a lane's registers.
template <int GROUP, bool ZEROS>
struct FewWeights {
    static constexpr int PER = kChunk / GROUP;
    uint4 w[4];
    uint4 s[PER / 2];                 // [PER][4] halves
    uint32_t z[ZEROS ? PER / 4 : 1];  // [PER] bytes of the lane's row, 16 - zero

    // tile t's words, and the scales and zero points whose last one is the tile's:
    // what an earlier strip had there has been used
    __device__ __forceinline__ void load(const Q4& m, int strip, int chunk, int lane, int t)
    {
        constexpr int S_TILES = PER > 8 ? 1 : 8 / PER, Z_TILES = 16 / PER;   // tiles of an s (two for 32), of a z
        if (chunk * 4 + t < m.tiles) w[t] = reinterpret_cast<const uint4*>(m.numbers)[((size_t)strip * m.tiles + chunk * 4 + t) * 64 + lane];
        const size_t cell = (size_t)strip * m.chunks + chunk;
        if ((t + 1) % S_TILES == 0) {
            const uint4* q = reinterpret_cast<const uint4*>(m.scales) + (cell * 4 + (lane >> 4)) * (PER / 2);
            constexpr int N = PER > 8 ? 2 : 1;
#pragma unroll
            for (int i = 0; i < N; i++) s[t / S_TILES * N + i] = q[t / S_TILES * N + i];
        }
        if constexpr (ZEROS)
            if ((t + 1) % Z_TILES == 0) {
                const uint32_t* r = reinterpret_cast<const uint32_t*>(m.zeros) + (cell * kStrip + (lane & 15)) * (PER / 4);
                z[t / Z_TILES] = 0x10101010u - r[t / Z_TILES];
            }
    }
};

// Eight weights as signed bytes: without zero points 16 (n - 8) (the stored four
// bits are n - 8 in two's complement, at the top of a byte 16 times that),
// with them n - zero + 16 (16 times the sum of x's digits is taken off by an
// instruction of its own, on the matrix units that have the time).
template <bool ZEROS>
__device__ __forceinline__ void widen8(uint32_t w, uint32_t zero4, uint32_t& lo, uint32_t& hi)
{
    if constexpr (ZEROS) {
        lo = ((w & 0x0f0f0f0fu) ^ 0x08080808u) + zero4;
        hi = ((w >> 4 & 0x0f0f0f0fu) ^ 0x08080808u) + zero4;
    } else {
        lo = w << 4 & 0xf0f0f0f0u;
        hi = w & 0xf0f0f0f0u;
    }
}

// Columns are an odd number of 16 bytes apart in LDS: lanes that write a column's
// next inputs meet other banks.
__host__ __device__ constexpr int few_pitch(int cols) { return cols | 1; }

// the largest of 16 neighbouring lanes', in each of them
__device__ __forceinline__ uint32_t max16(uint32_t v)
{
    v = max(v, dpp_t<0x128>(v, v));
    v = max(v, dpp_t<0x124>(v, v));
    v = max(v, dpp_t<0x122>(v, v));
    return max(v, dpp_t<0x121>(v, v));
}

// A workgroup takes S strips of 16 rows of the matrix; its waves deal the chunks
// of 512 inputs among themselves.  A wave brings the rows' 512 values into its
// own part of LDS as digits in the operands' order (16 lanes a tile, 8 values
// each) while the first strip's weights are on their way (a strip's tile comes as
// soon as the one before has been computed), and needs no other wave until the
// sums are joined.
template <int D, bool E4M3, int GROUP, bool ZEROS, int S>
__global__ __launch_bounds__(64 * kFewMaxWaves) void k_q4_few(FewArgs a)
{
    extern __shared__ uint4 lds[];
    constexpr bool SCALED = D == 1 || E4M3;
    const int x_type = D == 1 ? IAM_I8 : D == 4 ? IAM_F32 : E4M3 ? IAM_E4M3 : a.u.x_type;
    MulArgs u = a.u;
    if (D == 4 && gridDim.y > 1) {       // (else there is one part)
        const int r0 = blockIdx.y * a.rows;
        u.rows = min(a.rows, u.rows - r0);
        u.x = reinterpret_cast<const float*>(u.x) + (size_t)r0 * u.x_stride;
        u.y = reinterpret_cast<uint8_t*>(u.y) + (size_t)r0 * u.y_stride * (u.y_type == IAM_F32 ? 4 : 2);
    }
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int last = q4_strips(u.m.out) - 1, groups = (last + S) / S, id = xcd_remap(blockIdx.x, gridDim.x);
    const int split = id / groups, group = id - split * groups, strip0 = group * S, cols = u.rows * D;
    const int pitch = few_pitch(cols);
    uint4* digits = lds + wave * (32 * pitch);                                      // [tile][step][g][col] 16 bytes
    float* factor = reinterpret_cast<float*>(lds + a.waves * (32 * pitch)) + wave * 4 * kFewCols;   // [tile][row]
    const int col = min(c, cols - 1), mine = col / D;
    // What a tile's sums are times: the digit's place, less the weights' 16 and
    // e4m3 numbers' 2^13.  (At the end alone, the sums of digits of the smallest
    // results would be subnormal and those of the largest infinite.)  A power of
    // two takes it exactly, a scale might not: 8-bit rows' sums are times it first.
    const float place = ldexpf(1.0f, 8 * (col - mine * D) - (ZEROS ? 0 : 4) - (E4M3 ? 13 : 0));
    floatx4 acc[S];
#pragma unroll
    for (int s = 0; s < S; s++) acc[s] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    FewWeights<GROUP, ZEROS> now;
    for (int chunk = split * a.waves + wave; chunk < u.m.chunks; chunk += a.splits * a.waves) {
        const int t16 = lane >> 4, k8 = lane & 15, k = chunk * kChunk + t16 * kTile + k8 * 8;
        Raw8 raw = load_raw8(u.x, x_type, 0, k, u.m.in);
        float xs = SCALED ? u.x_scale[u.x_groups > 1 ? min(chunk * 4 + t16, u.x_groups - 1) : 0] : 1.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) now.load(u.m, strip0, chunk, lane, t);
        uint2* to = reinterpret_cast<uint2*>(digits + ((t16 * 2 + (k8 >> 3)) * 4 + (k8 & 3)) * pitch) + (k8 >> 2 & 1);
        for (int r = 0; r < u.rows; r++) {
            const Raw8 mine8 = raw;
            const float scale = xs;
            if (r + 1 < u.rows) {
                raw = load_raw8(u.x, x_type, (size_t)(r + 1) * u.x_stride, k, u.m.in);
                if constexpr (SCALED)
                    xs = u.x_scale[(size_t)(r + 1) * u.x_groups + (u.x_groups > 1 ? min(chunk * 4 + t16, u.x_groups - 1) : 0)];
            }
            if constexpr (D == 1) {
                const uint32_t p = mine8.a.x, q = mine8.a.y;
                to[r * 2] = {__builtin_amdgcn_perm(q, p, 0x05010400u), __builtin_amdgcn_perm(q, p, 0x07030602u)};
                if (k8 == 0) factor[t16 * kFewCols + r] = scale;
            } else {
                float v[8];
                values8(mine8, x_type, v);
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
                top = max16(top);
                // n = round(v 2^(148 - e)), below 2^22; 2^(e - 148) back (NaN
                // where a value is not finite).  Tiles below 2^-102 count as if
                // they were that large; e4m3 numbers, at most 448 and whole multiples
                // of 2^-9, have one power, which goes to `place` so that the smallest
                // scales keep their bits.  fp32: 2^(156 - e), below 2^30, from 2^-96 on.
                const uint32_t e8 = E4M3 ? 135u : max(top >> 23, D == 4 ? 30u : 24u);
                const float up = __uint_as_float(((D == 4 ? 283u : 275u) - e8) << 23);
                uint32_t n[8];               // 128 more in each digit makes them whole bytes
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if constexpr (D == 4) n[e] = (uint32_t)(int)(v[e] * up) + 0x80808080u;
                    else n[e] = __float_as_uint(__builtin_fmaf(v[e], up, 12582912.0f)) + (0x00808080u - 0x4b400000u);   // 1.5 2^23 + n has n in its low bits
                }
                // digits d and d + 1 of two values, then each of four
                auto two = [&](int lo, int hi, uint32_t sel) { return __builtin_amdgcn_perm(n[hi], n[lo], sel); };
                uint2* at = to + r * 2 * D;
#pragma unroll
                for (int d = 0; d < D; d += 2) {
                    const uint32_t sel = d == 0 ? 0x05010400u : D == 4 ? 0x07030602u : 0x0c0c0602u;
                    const uint32_t a0 = two(0, 4, sel), a1 = two(1, 5, sel), b0 = two(2, 6, sel), b1 = two(3, 7, sel);
                    at[2 * d] = {__builtin_amdgcn_perm(a1, a0, 0x05040100u) ^ 0x80808080u, __builtin_amdgcn_perm(b1, b0, 0x05040100u) ^ 0x80808080u};
                    if (d + 1 < D) at[2 * d + 2] = {__builtin_amdgcn_perm(a1, a0, 0x07060302u) ^ 0x80808080u, __builtin_amdgcn_perm(b1, b0, 0x07060302u) ^ 0x80808080u};
                }
                if (k8 == 0) factor[t16 * kFewCols + r] = top >= 0x7f800000u ? NAN : E4M3 ? scale : __uint_as_float((e8 - (D == 4 ? 29u : 21u)) << 23);
            }
        }
        wave_sync();
        const int tiles = min(4, u.m.tiles - chunk * 4);
#pragma unroll
        for (int sn = 0; sn < S; sn++) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (t < tiles) {
                    const float f = SCALED ? factor[t * kFewCols + mine] : factor[t * kFewCols + mine] * place;
                    const uint32_t wd[4] = {now.w[t].x, now.w[t].y, now.w[t].z, now.w[t].w};
                    intx4 sum = {0, 0, 0, 0};
                    floatx4 part = {0.0f, 0.0f, 0.0f, 0.0f};   // of the tile, without f
#pragma unroll
                    for (int step = 0; step < 2; step++) {
                        const uint4 b = digits[((t * 2 + step) * 4 + g) * pitch + col];
                        uint32_t lo[2], hi[2];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const int grp = (t * kTile + (step * 2 + j) * 32) / GROUP;
                            uint32_t z4 = 0;
                            if constexpr (ZEROS) z4 = __builtin_amdgcn_perm(0u, now.z[grp / 4], 0x01010101u * (grp % 4));
                            widen8<ZEROS>(wd[step * 2 + j], z4, lo[j], hi[j]);
                        }
                        auto join = [&](int grp) {
                            const uint32_t s0 = grp % 2 ? now.s[grp / 2].z : now.s[grp / 2].x, s1 = grp % 2 ? now.s[grp / 2].w : now.s[grp / 2].y;
                            const half4 s = __builtin_bit_cast(half4, (uint64_t)s1 << 32 | s0);
#pragma unroll
                            for (int i = 0; i < 4; i++) part[i] = __builtin_fmaf((float)sum[i], (float)s[i], part[i]);
                            sum = intx4{0, 0, 0, 0};
                        };
                        if constexpr (GROUP == 32) {
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const long x8 = (long)((uint64_t)(j ? b.w : b.y) << 32 | (j ? b.z : b.x));
                                if constexpr (ZEROS) sum = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)0xf0f0f0f0f0f0f0f0ull, x8, sum, 0, 0, 0);
                                sum = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)((uint64_t)hi[j] << 32 | lo[j]), x8, sum, 0, 0, 0);
                                join(t * 4 + step * 2 + j);
                            }
                        } else {
                            constexpr int less = (int)0xf0f0f0f0u;   // -16, four times
                            const intx4 w8 = {(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
                            if constexpr (ZEROS) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(intx4{less, less, less, less}, __builtin_bit_cast(intx4, b), sum, 0, 0, 0);
                            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(w8, __builtin_bit_cast(intx4, b), sum, 0, 0, 0);
                            if constexpr (GROUP == 64) join(t * 2 + step);
                            else if (step == 1) join(t);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[sn][i] = __builtin_fmaf(SCALED && !(D == 1 && ZEROS) ? part[i] * place : part[i], f, acc[sn][i]);
                }
                if (sn + 1 < S) now.load(u.m, min(strip0 + sn + 1, last), chunk, lane, t);
            }
        }
        wave_sync();
    }
    // the waves' sums: [wave][strip][col][16]
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
    if (c < cols)
#pragma unroll
        for (int s = 0; s < S; s++) *reinterpret_cast<floatx4*>(part + ((wave * S + s) * cols + c) * 16 + 4 * g) = acc[s];
    __syncthreads();
    const int values = S * u.rows * 16;
    auto put = [&](int i, float y) {
        const int r = i / (S * 16), o = (strip0 + i / 16 % S) * kStrip + (i & 15);
        if (o < u.m.out) put_value(u.y, u.y_type, (size_t)r * u.y_stride + o, y);
    };
    const size_t cell = (size_t)blockIdx.y * groups + group;
    float* sums = a.sums + cell * a.splits * (S * a.rows * 16);
    for (int i = tid; i < values; i += a.waves * 64) {
        const int r = i / (S * 16), s = i / 16 % S;
        float y = 0.0f;
#pragma unroll
        for (int d = D - 1; d >= 0; d--) {
            float sum = 0.0f;
            for (int w = 0; w < a.waves; w++) sum += part[((w * S + s) * cols + r * D + d) * 16 + (i & 15)];
            y += sum;
        }
        if (a.splits == 1) put(i, y);
        else acc_put(sums + split * values + i, y);
    }
    if (a.splits == 1) return;
    __shared__ int arrived;
    if (!acc_arrive(a.ctr + cell, (uint32_t)a.splits, &arrived)) return;
    if (tid == 0) a.ctr[cell] = 0u;
    for (int i = tid; i < values; i += a.waves * 64) {
        float each[kFewSplits], y = 0.0f;
#pragma unroll
        for (int q = 0; q < kFewSplits; q++) each[q] = acc_peek(sums + min(q, a.splits - 1) * values + i);
#pragma unroll
        for (int q = 0; q < kFewSplits; q++) y += q < a.splits ? each[q] : 0.0f;
        put(i, y);
    }
}

// ------------------------------------------------------------------ host ---
static int digits_of(int x_type) { return x_type == IAM_I8 ? 1 : x_type == IAM_F32 ? 4 : 3; }

// How a call's rows, strips and chunks are dealt.
struct FewPlan {
    int digits, rows, row_parts;   // rows of a workgroup, and in how many of these the rows are
    int together;                  // strips of a workgroup
    int splits, waves;
    size_t lds;
};
static FewPlan few_plan(const MulArgs& u)
{
    FewPlan p{};
    p.digits = digits_of(u.x_type);
    p.row_parts = (u.rows * p.digits + kFewCols - 1) / kFewCols;
    p.rows = (u.rows + p.row_parts - 1) / p.row_parts;
    // Several strips share the rows' digits, and a strip's weights come while the
    // one before is computed, where there are enough for the card all the same
    // (one bf16 row, 28672 x 4096 with groups of 64 and zero points: 17.3 us by single
    // strips, 15.1 by two, 13.1 by four, 23.8 by eight; five rows 26.1, 20.0 and 15.6;
    // 8192 x 8192 with groups of 128 11.0, 9.4 and 9.1, 6144 x 4096 5.7, 6.2 and 7.1).
    // Groups of 32 with zero points and four strips do not fit the registers (28672 x
    // 4096: 20.1, 17.4 and 23.0).
    const int strips = q4_strips(u.m.out);
    p.together = strips < 512 ? 1 : u.m.group == 32 ? 2 : 4;
    // A wave for each chunk, as many as 160 KB of LDS hold digits of (512 bytes
    // a column and 256 of factors each).
    const int cols = p.rows * p.digits, most = std::min(kFewMaxWaves, kFewLds / (512 * few_pitch(cols) + 256));
    // Where a workgroup's waves would take several turns the inputs are cut, for
    // about a workgroup a CU (four fp32 rows, 1024 x 14336: 11.0 us whole, 8.6 cut;
    // 1024 x 8192 in one turn 7.2 and 7.2; one row of 1024 x 14336 7.3 and 6.6, but 7.7
    // and 8.1 of 2048 x 14336 in two).
    const int fit = 256 / strips;
    p.splits = u.m.chunks > most && fit > (u.rows > 1 ? 1 : 2) ? std::min({fit, kFewSplits, u.m.chunks / 4}) : 1;
    const int each = (u.m.chunks + p.splits - 1) / p.splits, rounds = (each + most - 1) / most;
    p.waves = (each + rounds - 1) / rounds;
    const size_t stage = (size_t)p.waves * (512 * few_pitch(cols) + 256), join = (size_t)p.waves * p.together * cols * 64;
    p.lds = std::max(stage, join);
    return p;
}

bool q4_takes_few(const MulArgs& u)
{
    if ((int64_t)u.rows * digits_of(u.x_type) <= kFewCols) return true;
    if (u.x_type != IAM_F32 || u.rows > 5) return false;
    // Five fp32 rows, as three and two: where the workgroups of both run in one round
    // and a half at most (6144 x 4096 9.3 us, 12.3 with fp16 parts; 14336 x 4096 10.2
    // and 15.2; 4096 x 14336 and 32000 x 4096, in two rounds, 19.1 and 24.3, but 17.3 and 21.6).
    const FewPlan p = few_plan(u);
    const int64_t all = (int64_t)((q4_strips(u.m.out) + p.together - 1) / p.together) * p.splits * p.row_parts;
    return 2 * all <= 3 * 256 * (int64_t)std::min<size_t>(kFewLds / p.lds, 32 / p.waves);
}

template <int D, bool E4M3, int GROUP, int S>
static int few_launch(Ctx* c, const FewArgs& a, const FewPlan& p)
{
    const dim3 grid((unsigned)((q4_strips(a.u.m.out) + S - 1) / S * a.splits), (unsigned)p.row_parts), block((unsigned)a.waves * 64);
    return a.u.m.zeros ? launch(c, "q4_mul.few", k_q4_few<D, E4M3, GROUP, true, S>, grid, block, p.lds, a)
                       : launch(c, "q4_mul.few", k_q4_few<D, E4M3, GROUP, false, S>, grid, block, p.lds, a);
}

template <int D, bool E4M3, int GROUP>
static int few_sized(Ctx* c, const FewArgs& a, const FewPlan& p)
{
    return p.together == 1 ? few_launch<D, E4M3, GROUP, 1>(c, a, p) : few_launch<D, E4M3, GROUP, GROUP == 32 ? 2 : 4>(c, a, p);
}

template <int D, bool E4M3>
static int few_grouped(Ctx* c, const FewArgs& a, const FewPlan& p)
{
    if (a.u.m.group == 32) return few_sized<D, E4M3, 32>(c, a, p);
    if (a.u.m.group == 64) return few_sized<D, E4M3, 64>(c, a, p);
    return few_sized<D, E4M3, 128>(c, a, p);
}

int q4_mul_few(Ctx* c, const MulArgs& u)
{
    const FewPlan p = few_plan(u);
    FewArgs a{};
    a.u = u;
    a.rows = p.rows;
    a.waves = p.waves;
    a.splits = p.splits;
    if (p.splits > 1) {
        const size_t cells = (size_t)q4_strips(u.m.out) * p.row_parts;    // (single strips)
        IAM_TRY(ensure_q4_sums(c, cells * p.splits * p.rows * kStrip, cells));
        a.sums = c->q4_sums;
        a.ctr = c->q4_ctr;
    }
    if (p.digits == 1) return few_grouped<1, false>(c, a, p);
    if (p.digits == 4) return few_grouped<4, false>(c, a, p);
    return u.x_type == IAM_E4M3 ? few_grouped<3, true>(c, a, p) : few_grouped<3, false>(c, a, p);
}

}  // namespace iam
