// Products of many rows (batches, prompts) with 4-bit weights, on the fp16 matrix
// instructions, and those of more than 64 rows in int8 on the 8-bit ones.
//
// A launch of its own brings x into the instructions' order, bytes as they are,
// the rest as fp16: one part of values that fp16 holds (fp16 and 8-bit numbers;
// bf16 of a tile of 128 after a power of two where its largest value lies outside
// [2^-2, 2^15)), two, high and low, of fp32 (22 bits).  4-bit weights become fp16 under the exponents of
// 1024 and 64, n - zero exactly.  Products are then exact; a group's are added
// in fp32 by the instructions and go to the row's sum with the group's scale and
// that power: times the scale first, as a sum of large x times the power alone
// may pass fp32's range, and so may the two together at either end.
#include "accum.h"
#include "q4_mul.h"

namespace iam {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef unsigned long long ull2 __attribute__((ext_vector_type(2)));

// ---- x in the operands' order
// parts  fp16 [part][block of 16 rows][tile][j][lane 16 g + row][8]: inputs
//        32 j + 8 g and on of the tile.  Or int8 [block of 16 rows][tile][j][lane
//        16 half + row][16]: eight inputs from 32 j + 8 half on, eight from 16 further on
// factor fp32 [block][tile][16]: what the tile's values were divided by
// scaled [block][tile]: kScaled if any of these is not 1, kFar too if one is far from it
constexpr uint8_t kScaled = 1, kFar = 2;
// A factor up to 2^64 times a weights' scale (below 2^16) and a sum (below 2^27 a
// tile, 2^13 tiles) stays in fp32's range, and one from 2^-100 on times a scale
// (from 2^-24 on) keeps its bits.
__device__ __forceinline__ bool is_far(float f) { return f != 0.0f && !(fabsf(f) >= 0x1p-100f && fabsf(f) <= 0x1p64f); }
struct PrepArgs {
    const void* x;
    int type;
    size_t stride;
    const float* x_scale;    // with a scale for each tile (else null)
    int rows, in, tiles;
    _Float16* parts;
    size_t part_stride;      // values of a part
    float* factor;
    uint8_t* scaled;
    int parts_n;             // 0: 8-bit rows as they are
};

constexpr int kPrepThreads = 256;

// A wave takes a tile of a block of 16 rows: lane (g, c) 32 values of row c.
__global__ __launch_bounds__(kPrepThreads) void k_q4_prep(PrepArgs a)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int tile = blockIdx.x * (kPrepThreads / 64) + (threadIdx.x >> 6), block = blockIdx.y;
    if (tile >= a.tiles) return;
    const int row = block * 16 + c;
    const bool there = row < a.rows;
    float v[4][8];
    uint2 bytes[4];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const Raw8 r = load_raw8(a.x, a.type, (size_t)(there ? row : 0) * a.stride, tile * kTile + 32 * j + 8 * g, there ? a.in : 0);
        values8(r, a.type, v[j]);
        bytes[j] = {r.a.x, r.a.y};
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(v[j][e]) & 0x7fffffffu);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    float up = 1.0f, f = 1.0f;
    if (a.type == IAM_F32 || a.type == IAM_BF16) {
        // exponents -2 .. 14 (and 0) stay; else the largest value goes to [2^14, 2^15)
        const int e = (int)(top >> 23) - 127;
        if (top != 0u && e < 128 && (e < -2 || e > 14)) {
            const int sh = min(14 - e, 126);
            up = ldexpf(1.0f, sh);
            f = ldexpf(1.0f, -sh);
        }
    }
    if (a.x_scale) f = there ? a.x_scale[(size_t)row * a.tiles + tile] : 1.0f;
    const size_t at = ((size_t)block * a.tiles + tile) * 4 * 64 * 8;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (a.parts_n == 0) {
            // as the bytes of widened weights lie
            const uint32_t p = bytes[j].x, q = bytes[j].y;
            *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.parts) + at + ((j * 32 + (g & 1) * 16 + c) * 16 + (g >> 1) * 8)) =
                uint2{__builtin_amdgcn_perm(q, p, 0x05010400u), __builtin_amdgcn_perm(q, p, 0x07030602u)};
            continue;
        }
        half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = v[j][e] * up;
            h[e] = (_Float16)y;
            l[e] = fabsf((float)h[e]) < INFINITY ? (_Float16)(y - (float)h[e]) : (_Float16)0.0f;
        }
        *reinterpret_cast<half8*>(a.parts + at + (j * 64 + lane) * 8) = h;
        if (a.parts_n == 2) *reinterpret_cast<half8*>(a.parts + a.part_stride + at + (j * 64 + lane) * 8) = l;
    }
    const size_t cell = (size_t)block * a.tiles + tile;
    if (g == 0) a.factor[cell * 16 + c] = f;
    const bool scaled = __any(f != 1.0f), far = __any(is_far(f));
    if (lane == 0) a.scaled[cell] = (scaled ? kScaled : 0) | (far ? kFar : 0);
}

// ---- the products
struct RowsArgs {
    MulArgs u;
    const _Float16* parts;
    size_t part_stride;
    const float* factor;
    const uint8_t* scaled;    // null: no factor can be anything but 1
    const float* row_scale;   // of a whole row, or null
    bool bytes;               // parts in 8 bits
    int blocks;               // of 16 rows
    int waves;
    // the inputs cut into parts for more workgroups, whose sums the last one to arrive joins
    int splits;
    float* sums;
    uint32_t* ctr;            // zero on entry (left zero)
};

constexpr int kMaxSplits = 8;

// Eight weights as fp16, n - zero: under the exponent of 1024 a number's step is
// 1, under that of 64 it is 1/16.
__device__ __forceinline__ half8 widen_half(uint32_t w, uint32_t minus1024, uint32_t minus64)
{
    const uint32_t v = w >> 8;
    const half2v a = __builtin_bit_cast(half2v, (w & 0x000f000fu) ^ 0x64086408u) + __builtin_bit_cast(half2v, minus1024);
    const half2v b = __builtin_bit_cast(half2v, (w & 0x00f000f0u) ^ 0x54805480u) + __builtin_bit_cast(half2v, minus64);
    const half2v c = __builtin_bit_cast(half2v, (v & 0x000f000fu) ^ 0x64086408u) + __builtin_bit_cast(half2v, minus1024);
    const half2v d = __builtin_bit_cast(half2v, (v & 0x00f000f0u) ^ 0x54805480u) + __builtin_bit_cast(half2v, minus64);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four weights as signed bytes (of the word's low or high halves of bytes): without
// zero points 16 (n - 8), with them n - zero.
template <bool ZEROS>
__device__ __forceinline__ uint32_t widen_low(uint32_t w, uint32_t zero4)
{
    return ZEROS ? (((w & 0x0f0f0f0fu) ^ 0x88888888u) - zero4) ^ 0x80808080u : w << 4 & 0xf0f0f0f0u;   // 128 + n - zero: no borrows
}
template <bool ZEROS>
__device__ __forceinline__ uint32_t widen_high(uint32_t w, uint32_t zero4)
{
    return ZEROS ? widen_low<true>(w >> 4, zero4) : w & 0xf0f0f0f0u;
}

// what is subtracted for a zero point: -(1024 + zero) and -(64 + zero), twice
struct Minus {
    uint32_t k1024, k64;
};
__device__ __forceinline__ Minus minus_of(uint32_t zero)
{
    const uint32_t two = zero | zero << 16;
    return {0xe400e400u | two, 0xd400d400u | two << 4};
}

__device__ __forceinline__ floatx4 mfma_f16(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// four results of row r, outputs o and on
__device__ __forceinline__ void put_four(const MulArgs& u, int r, int o, floatx4 v)
{
    const size_t at = (size_t)r * u.y_stride + o;
    if (o + 4 <= u.m.out) {
        if (u.y_type == IAM_F32) {
            *reinterpret_cast<Pack<float, 4, 4>*>(reinterpret_cast<float*>(u.y) + at) = {v[0], v[1], v[2], v[3]};
        } else if (u.y_type == IAM_F16) {
            *reinterpret_cast<Pack<_Float16, 4, 2>*>(reinterpret_cast<_Float16*>(u.y) + at) = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        } else {
            *reinterpret_cast<Pack<__bf16, 4, 2>*>(reinterpret_cast<__bf16*>(u.y) + at) = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (o + i < u.m.out) put_value(u.y, u.y_type, at + i, v[i]);
}

// eight of them in 16 bits, from o on
__device__ __forceinline__ void put_eight(const MulArgs& u, int r, int o, floatx4 v, floatx4 w)
{
    const size_t at = (size_t)r * u.y_stride + o;
    if (o + 8 <= u.m.out) {
        if (u.y_type == IAM_F16)
            *reinterpret_cast<Pack<_Float16, 8, 2>*>(reinterpret_cast<_Float16*>(u.y) + at) = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3],
                                                                                              (_Float16)w[0], (_Float16)w[1], (_Float16)w[2], (_Float16)w[3]};
        else
            *reinterpret_cast<Pack<__bf16, 8, 2>*>(reinterpret_cast<__bf16*>(u.y) + at) = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3],
                                                                                          (__bf16)w[0], (__bf16)w[1], (__bf16)w[2], (__bf16)w[3]};
        return;
    }
    put_four(u, r, o, v);
    if (o + 4 < u.m.out) put_four(u, r, o + 4, w);
}

// A workgroup takes S strips of the matrix and NB blocks of 16 rows; its waves
// deal the tiles of 128 inputs among themselves and join their sums in LDS.
// Every operand comes straight from memory in the order in which it is used.  32
// bf16 rows of 4096 x 14336 take 12.5 us: 31 MB of weights (4.9 at a streaming
// read's rate), x's parts 117 MB from the L2 caches; the next tile's operands in
// registers ahead of their use change nothing.
template <int PARTS, int GROUP, int S, int NB, int MOST>
__global__ __launch_bounds__(64 * MOST) void k_q4_batch(RowsArgs a)
{
    extern __shared__ floatx4 join[];
    constexpr int GT = kTile / GROUP;      // groups of a tile
    const MulArgs& u = a.u;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int strips = q4_strips(u.m.out), groups = (strips + S - 1) / S, id = xcd_remap(blockIdx.x, gridDim.x);
    const int split = id / groups, group = id - split * groups, s0 = group * S, b0 = blockIdx.y * NB;
    floatx4 acc[S][NB];
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int n = 0; n < NB; n++) acc[s][n] = floatx4{0, 0, 0, 0};
    const uint4* words[S];
    int strip[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
        strip[s] = min(s0 + s, strips - 1);
        words[s] = reinterpret_cast<const uint4*>(u.m.numbers) + (size_t)strip[s] * u.m.tiles * 64 + lane;
    }
    // a tile's operands, scales and zero points
    struct Tile {
        half8 x[PARTS][NB][4];
        float f[NB];
        uint4 w[S];
        half4 sc[S][GT];
        uint32_t zero[S];
    };
    auto load = [&](Tile& o, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            o.w[s] = words[s][(size_t)t * 64];
            const size_t cell = (size_t)strip[s] * u.m.chunks + (t >> 2);
            const half4* q = reinterpret_cast<const half4*>(u.m.scales) + (cell * 4 + g) * (4 * GT) + (t & 3) * GT;
#pragma unroll
            for (int i = 0; i < GT; i++) o.sc[s][i] = q[i];
            o.zero[s] = 0x08080808u;
            if (u.m.zeros) {
                const uint8_t* z = u.m.zeros + (cell * kStrip + c) * (4 * GT) + (t & 3) * GT;
                if constexpr (GT == 1) o.zero[s] = *z;
                else if constexpr (GT == 2) o.zero[s] = *reinterpret_cast<const uint16_t*>(z);
                else o.zero[s] = *reinterpret_cast<const uint32_t*>(z);
            }
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const size_t cell = (size_t)min(b0 + n, a.blocks - 1) * u.m.tiles + t;
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int j = 0; j < 4; j++) o.x[p][n][j] = *reinterpret_cast<const half8*>(a.parts + p * a.part_stride + (cell * 4 + j) * 512 + lane * 8);
            o.f[n] = a.factor[cell * 16 + c];
        }
    };
    auto compute = [&](const Tile& o) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            const uint32_t wd[4] = {o.w[s].x, o.w[s].y, o.w[s].z, o.w[s].w};
            half8 wide[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const Minus m = minus_of(o.zero[s] >> (8 * (j * 32 / GROUP)) & 255u);
                wide[j] = widen_half(wd[j], m.k1024, m.k64);
            }
#pragma unroll
            for (int i = 0; i < GT; i++) {
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    floatx4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int j = i * 4 / GT; j < (i + 1) * 4 / GT; j++)
#pragma unroll
                        for (int p = 0; p < PARTS; p++) d = mfma_f16(wide[j], o.x[p][n][j], d);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[s][n][e] = __builtin_fmaf(d[e] * (float)o.sc[s][i][e], o.f[n], acc[s][n][e]);
                }
            }
        }
    };
    for (int t = split * a.waves + wave; t < u.m.tiles; t += a.splits * a.waves) {
        Tile o;
        load(o, t);
        // all loads before any use: left to itself the compiler saved registers and
        // waited for a few at a time (32 fp32 rows, 4096 x 14336: 27 us against 17)
        __builtin_amdgcn_sched_barrier(0);
        compute(o);
    }
    if (a.waves > 1) {
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int n = 0; n < NB; n++) join[(wave * S * NB + s * NB + n) * 64 + lane] = acc[s][n];
        __syncthreads();
    }
    // value e of a lane is row 4 g + e of strip s, row c of block n
    auto put = [&](int s, int n, floatx4 v) __attribute__((always_inline)) {
        const int r = (b0 + n) * 16 + c;
        if (s0 + s >= strips || r >= u.rows) return;
        if (a.row_scale) v *= a.row_scale[r];
        put_four(u, r, (s0 + s) * kStrip + 4 * g, v);
    };
    // the splits' sums: [group of strips][group of blocks][split][S * NB][lane] four floats
    const size_t cell = (size_t)blockIdx.y * groups + group;
    float* sums = a.sums + cell * a.splits * (S * NB * 256);
#pragma unroll
    for (int i = 0; i < S * NB; i++) {
        if (i % a.waves != wave) continue;
        floatx4 v = acc[i / NB][i % NB];
        if (a.waves > 1) {
            v = join[i * 64 + lane];
            for (int q = 1; q < a.waves; q++) v += join[(q * S * NB + i) * 64 + lane];
        }
        if (a.splits == 1) {
            put(i / NB, i % NB, v);
        } else {
            const ull2 two = __builtin_bit_cast(ull2, v);
            unsigned long long* to = reinterpret_cast<unsigned long long*>(sums + ((size_t)split * (S * NB) + i) * 256 + lane * 4);
            acc_put(to, two[0]);
            acc_put(to + 1, two[1]);
        }
    }
    if (a.splits == 1) return;
    __shared__ int last;
    if (!acc_arrive(a.ctr + cell, (uint32_t)a.splits, &last)) return;
    if (threadIdx.x == 0) a.ctr[cell] = 0u;
    for (int i = wave; i < S * NB; i += a.waves) {
        // all of them on the way at once
        ull2 two[kMaxSplits];
#pragma unroll
        for (int q = 0; q < kMaxSplits; q++) {
            unsigned long long* from = reinterpret_cast<unsigned long long*>(sums + ((size_t)min(q, a.splits - 1) * (S * NB) + i) * 256 + lane * 4);
            two[q][0] = acc_peek(from);
            two[q][1] = acc_peek(from + 1);
        }
        floatx4 v = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < kMaxSplits; q++)
            if (q < a.splits) v += __builtin_bit_cast(floatx4, two[q]);
        put(i / NB, i % NB, v);
    }
}

// Many rows: a workgroup takes 64 WO rows of the matrix and 32 NB of x, its
// waves WO by two 64 x 16 NB of them.  What a tile of 128 inputs needs goes to
// LDS past the registers, STAGES - 1 tiles ahead: x's operands and the strips'
// words in runs of 1 KB, a share for each wave, then scales and zero points.  4096
// bf16 rows of 14336 x 4096 take 450 to 490 us (980 to 1070 TFLOP/s; a matrix product
// of bf16 weights from the library 415): a tile of 256 x 128 products reads 240 KB
// of LDS, 1.9 thousand of its 3.5 thousand clocks, and the matrix instructions, busy
// 46% of the time, wait where the groups change.  In int8 343 us, bound by the
// vector instructions (11 and more for each matrix instruction of 32 clocks).
constexpr int kGemmStrips = 4;     // of a wave
constexpr int kGemmPanel = 8;      // workgroups side by side along x's rows that run together

// PARTS: of x in fp16; 0 and -1: x in 8 bits, with weights that have zero points (-1) or none.
template <int PARTS, int GROUP, int NB, int WO, int STAGES>
struct Gemm {
    static constexpr bool BYTE = PARTS <= 0;
    static constexpr int BLOCK = BYTE ? 2 : 4;     // KB of a tile of 16 rows
    static constexpr int GT = kTile / GROUP, S = kGemmStrips, WAVES = 2 * WO, STRIPS = S * WO;
    static constexpr int X = (BYTE ? 1 : PARTS) * 2 * NB * BLOCK, RUNS = X + STRIPS, SHARE = RUNS / WAVES;
    static constexpr int SCALES = RUNS * 1024;                      // [group][strip][g] four halves
    static constexpr int ZEROS = SCALES + GT * STRIPS * 32;         // [strip][row] words
    static constexpr int BYTES = ZEROS + STRIPS * 64;
    static constexpr int PER_GROUP = STRIPS / 8, SMALL = GT * PER_GROUP + STRIPS / 4;   // loads of 256 bytes
    static_assert(RUNS % WAVES == 0, "every wave brings as many runs");
    uint4 at[STAGES][BYTES / 16];
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx16 __attribute__((ext_vector_type(16)));

// LDS reads in one piece of assembly with their wait: the compiler, which
// cannot tell the stages apart, would wait for all loads in flight to LDS
// before any of them.
// x's operands of 32 rows (two blocks): (j, p) at 1024 j + 512 p
__device__ __forceinline__ void read_rows32(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:512\n\tds_read_b128 %2, %8 offset:1024\n\tds_read_b128 %3, %8 offset:1536\n\t"
        "ds_read_b128 %4, %8 offset:2048\n\tds_read_b128 %5, %8 offset:2560\n\tds_read_b128 %6, %8 offset:0xc00\n\tds_read_b128 %7, %8 offset:3584\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(at)
        : "memory");
}
// and of 64 rows
__device__ __forceinline__ void read_rows64(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %16\n\tds_read_b128 %1, %16 offset:512\n\tds_read_b128 %2, %16 offset:1024\n\tds_read_b128 %3, %16 offset:1536\n\t"
        "ds_read_b128 %4, %16 offset:2048\n\tds_read_b128 %5, %16 offset:2560\n\tds_read_b128 %6, %16 offset:0xc00\n\tds_read_b128 %7, %16 offset:3584\n\t"
        "ds_read_b128 %8, %16 offset:8192\n\tds_read_b128 %9, %16 offset:8704\n\tds_read_b128 %10, %16 offset:9216\n\tds_read_b128 %11, %16 offset:9728\n\t"
        "ds_read_b128 %12, %16 offset:10240\n\tds_read_b128 %13, %16 offset:10752\n\tds_read_b128 %14, %16 offset:11264\n\tds_read_b128 %15, %16 offset:11776\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]), "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]),
          "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
        : "v"(at)
        : "memory");
}
// 32 rows in 8 bits: j at 512 j
__device__ __forceinline__ void read_bytes32(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:512\n\tds_read_b128 %2, %4 offset:1024\n\tds_read_b128 %3, %4 offset:1536\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(at)
        : "memory");
}
// and 64
__device__ __forceinline__ void read_bytes64(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:512\n\tds_read_b128 %2, %8 offset:1024\n\tds_read_b128 %3, %8 offset:1536\n\t"
        "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %8 offset:4608\n\tds_read_b128 %6, %8 offset:5120\n\tds_read_b128 %7, %8 offset:5632\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(at)
        : "memory");
}
// two pairs of strips: words (pair, p) at 2048 pair + 512 p, zero points, scales of the first group
__device__ __forceinline__ void read_words(uint32_t words, uint32_t zeros, uint32_t scales, u32x4* w, uint32_t* z, u32x4* s)
{
    asm volatile(
        "ds_read_b128 %0, %10\n\tds_read_b128 %1, %10 offset:512\n\tds_read_b128 %2, %10 offset:2048\n\tds_read_b128 %3, %10 offset:2560\n\t"
        "ds_read_b32 %4, %11\n\tds_read_b32 %5, %11 offset:128\n\t"
        "ds_read2_b64 %6, %12 offset0:0 offset1:2\n\tds_read2_b64 %7, %12 offset0:4 offset1:6\n\t"
        "ds_read2_b64 %8, %12 offset0:8 offset1:10\n\tds_read2_b64 %9, %12 offset0:12 offset1:14\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(z[0]), "=&v"(z[1]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(words), "v"(zeros), "v"(scales)
        : "memory");
}
// their scales of a group: rows 8 i .. 8 i + 7 of a pair are in half i % 2 of s[2 pair + i / 2]
__device__ __forceinline__ void read_scales(uint32_t at, u32x4* s)
{
    asm volatile(
        "ds_read2_b64 %0, %4 offset0:0 offset1:2\n\tds_read2_b64 %1, %4 offset0:4 offset1:6\n\t"
        "ds_read2_b64 %2, %4 offset0:8 offset1:10\n\tds_read2_b64 %3, %4 offset0:12 offset1:14\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(at)
        : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }

// Tiles of a workgroup's products, without x's factors (they are all 1), with
// their products with the weights' scales, or with the two apart (some are far
// from 1; 4096 int8 rows of 14336 x 4096 in tiles of their own scale: 383 us, 361 with
// the products, which need not wait for the matrix instructions).
// Each is a loop of its own: no branch may lie between a matrix
// instruction and its results' first use, where the compiler leaves out the
// wait states of the edge that jumps.
enum class Factors { none, with_scales, apart };
template <int PARTS, int GROUP, int NB, int WO, int STAGES, Factors FACTORS, bool SECOND>
__device__ __forceinline__ void gemm_tiles(const RowsArgs& a, Gemm<PARTS, GROUP, NB, WO, STAGES>& stage, int s0, int b0, int t0, int t1, floatx16 (&acc)[2][NB / 2])
{
    typedef Gemm<PARTS, GROUP, NB, WO, STAGES> G;
    constexpr int GT = G::GT, S = G::S, N = NB / 2;
    constexpr int P = G::BYTE ? 1 : PARTS, OPS = G::BYTE ? 4 : 8;    // parts, matrix instructions of 32 rows and a pair of strips
    const MulArgs& u = a.u;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int c = lane & 15, side = lane >> 4 & 1, half = lane >> 5;   // row (of x or the matrix) 16 side + c, inputs 8 half and on of 16
    const int wo = wave >> 1, wx = wave & 1, last = q4_strips(u.m.out) - 1;
    typedef const __attribute__((address_space(1))) void* From;
    typedef __attribute__((address_space(3))) void* To;
    // A wave brings every WAVES-th run, (part, block, j) of x and then one a strip,
    // and every WAVES-th of the small loads: scales (group, eight strips), 8
    // lanes a strip, two a g; zero points (the word with the tile's) of four
    // strips' 16 rows.
    constexpr int SLOTS = (G::SMALL + G::WAVES - 1) / G::WAVES, N_SCALES = GT * G::PER_GROUP;
    const uint32_t lane16 = (uint32_t)lane * 16u;
    const uint8_t* run[G::SHARE];
    const uint8_t* small[SLOTS];
#pragma unroll
    for (int q = 0; q < G::SHARE; q++) {
        const int i = wave + G::WAVES * q;
        if ((q + 1) * G::WAVES <= G::X) {
            const int b = min(b0 + i / G::BLOCK % (2 * NB), a.blocks - 1), p = i / G::BLOCK / (2 * NB);
            run[q] = reinterpret_cast<const uint8_t*>(a.parts + p * a.part_stride) + ((size_t)b * u.m.tiles * G::BLOCK + i % G::BLOCK) * 1024;
        } else {
            run[q] = u.m.numbers + (size_t)min(s0 + i - G::X, last) * u.m.tiles * 1024;
        }
    }
#pragma unroll
    for (int k = 0; k < SLOTS; k++) {
        const int i = wave + G::WAVES * k, z = i - N_SCALES;
        if (z < 0) {
            const int strip = i % G::PER_GROUP * 8 + (lane >> 3);
            small[k] = reinterpret_cast<const uint8_t*>(u.m.scales) +
                       (((size_t)min(s0 + strip, last) * u.m.chunks * 4 + (lane >> 1 & 3)) * (4 * GT) + i / G::PER_GROUP) * 8 + (lane & 1) * 4;
        } else {
            const int strip = z * 4 + (lane >> 4);
            small[k] = u.m.zeros + ((size_t)min(s0 + strip, last) * u.m.chunks * kStrip + (lane & 15)) * (4 * GT);
        }
    }
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        char* to = reinterpret_cast<char*>(stage.at[buf]);
#pragma unroll
        for (int q = 0; q < G::SHARE; q++) {
            const uint8_t* src = run[q] + (uint32_t)t * ((q + 1) * G::WAVES <= G::X ? G::BLOCK * 1024u : 1024u);
            __builtin_amdgcn_global_load_lds((From)(src + lane16), (To)(to + (wave + G::WAVES * q) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < SLOTS; k++) {
            const int i = wave + G::WAVES * k;
            if (i < N_SCALES) {
                __builtin_amdgcn_global_load_lds((From)(small[k] + (uint32_t)((t >> 2) * (128 * GT) + (t & 3) * (8 * GT))), (To)(to + G::SCALES + i * 256), 4, 0, 0);
            } else if (i < G::SMALL && u.m.zeros) {
                __builtin_amdgcn_global_load_lds((From)(small[k] + (uint32_t)((t >> 2) * (64 * GT) + (t & 3) * GT / 4 * 4)),
                                                 (To)(to + G::ZEROS + (i - N_SCALES) * 256), 4, 0, 0);
            }
        }
    };
    float f[N];
    auto load_factors = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < N; n++) f[n] = a.factor[((size_t)min(b0 + wx * NB + 2 * n + side, a.blocks - 1) * u.m.tiles + t) * 16 + c];
    };
    if constexpr (FACTORS != Factors::none) load_factors(t0);
#pragma unroll
    for (int t = 0; t < STAGES - 1; t++) fetch(min(t0 + t, t1 - 1), t);
    int buf = 0, free_buf = STAGES - 1;
    const uint32_t base = lds_address(stage.at);
    // A wave's loads of a tile are done when no more are in flight than the
    // newer tiles' runs alone.
    auto arrived = [&] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * G::SHARE) : "memory"); };
    auto meet = [&] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // Two groups of four waves, one of each on a SIMD, take turns: one reads its
    // operands while the other computes.  (All in step read together, with the
    // matrix instructions idle, 4096 rows of 14336 x 4096 took 534 us against 479.)
    constexpr bool TURNS = G::WAVES == 8;
    arrived();
    meet();
    if constexpr (SECOND) meet();
#pragma unroll 1
    for (int t = t0; t < t1; t++) {
        // Every wave's loads of this tile have arrived, and every wave has read
        // the tile before, whose place the newest tile takes.
        float fn[N];
        if constexpr (FACTORS != Factors::none) {
#pragma unroll
            for (int n = 0; n < N; n++) fn[n] = f[n];
            load_factors(min(t + 1, t1 - 1));
        }
        fetch(min(t + STAGES - 1, t1 - 1), free_buf);   // behind the last tile, the last one again
        const uint32_t at = base + buf * G::BYTES;
        free_buf = buf;
        buf = buf + 1 == STAGES ? 0 : buf + 1;
        u32x4 x[P][N * OPS], w[4], sc[GT][4];
        uint32_t zero[2];
        const uint32_t mine = (uint32_t)(half * 16 + c) * 16u;
        read_words(at + (G::X + wo * S + side) * 1024 + mine, at + G::ZEROS + (wo * S + side) * 64 + c * 4, at + G::SCALES + wo * S * 32 + half * 8, w, zero, sc[0]);
#pragma unroll
        for (int i = 1; i < GT; i++) read_scales(at + G::SCALES + i * G::STRIPS * 32 + wo * S * 32 + half * 8, sc[i]);
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint32_t from = at + ((p * 2 + wx) * NB + side) * (G::BLOCK * 1024) + mine;
            if constexpr (G::BYTE && N == 2) read_bytes64(from, x[p]);
            else if constexpr (G::BYTE) read_bytes32(from, x[p]);
            else if constexpr (N == 2) read_rows64(from, x[p]);
            else read_rows32(from, x[p]);
        }
        // the next tile's loads, as late as the other group's turn allows
        if constexpr (SECOND) arrived();
        if constexpr (TURNS) meet();
#pragma unroll
        for (int s = 0; s < 2; s++) {       // pairs of strips
#pragma unroll
            for (int i = 0; i < GT; i++) {
                const uint32_t z = !u.m.zeros ? 8u
                                   : GT == 1  ? zero[s] >> (8 * (t & 3))
                                   : GT == 2  ? zero[s] >> (16 * (t & 1) + 8 * i)
                                              : zero[s] >> (8 * i);
                std::conditional_t<G::BYTE, intx16, floatx16> d[P][N];
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int n = 0; n < N; n++)
#pragma unroll
                        for (int e = 0; e < 16; e++) d[p][n][e] = 0;
                if constexpr (G::BYTE) {
                    const uint32_t z4 = (z & 255u) * 0x01010101u;
#pragma unroll
                    for (int j = i * 4 / GT; j < (i + 1) * 4 / GT; j++) {      // 32 inputs: word j of g = half and 2 + half
                        intx4 wide;
                        wide[0] = (int)widen_low<(PARTS < 0)>(w[s * 2][j], z4);
                        wide[1] = (int)widen_high<(PARTS < 0)>(w[s * 2][j], z4);
                        wide[2] = (int)widen_low<(PARTS < 0)>(w[s * 2 + 1][j], z4);
                        wide[3] = (int)widen_high<(PARTS < 0)>(w[s * 2 + 1][j], z4);
#pragma unroll
                        for (int n = 0; n < N; n++)
                            d[0][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wide, __builtin_bit_cast(intx4, x[0][n * 4 + j]), d[0][n], 0, 0, 0);
                    }
                } else {
                    const Minus m = minus_of(z & 255u);
#pragma unroll
                    for (int k = i * 8 / GT; k < (i + 1) * 8 / GT; k++) {      // 16 inputs: word k / 2, g = 2 (k % 2) + half
                        const half8 wide = widen_half(w[s * 2 + k % 2][k / 2], m.k1024, m.k64);
#pragma unroll
                        for (int p = 0; p < P; p++)
#pragma unroll
                            for (int n = 0; n < N; n++)
                                d[p][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wide, __builtin_bit_cast(half8, x[p][n * 8 + k]), d[p][n], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int n = 0; n < N; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const half8 scale = __builtin_bit_cast(half8, sc[i][s * 2 + e / 8]);
                        float v = (float)d[0][n][e];
                        if constexpr (P == 2) v += d[1][n][e];
                        float by = (float)scale[e % 8];
                        if constexpr (FACTORS == Factors::with_scales) by *= fn[n];
                        if constexpr (FACTORS == Factors::apart) {
                            v *= PARTS == 0 ? by * 0.0625f : by;
                            by = fn[n];
                        }
                        acc[s][n][e] = __builtin_fmaf(v, by, acc[s][n][e]);
                    }
            }
            if constexpr (GT > 1) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (GT == 1) {
            // the widening of the next inputs and the sums of the last pair between
            // the matrix instructions (smaller groups would spill); with 8 for 7 4096 rows
            // of 14336 x 4096 took 481 us for 478, with 14 for 11 389 int8 rows 28.5 for 27.5,
            // with 11 for 14 4096 of them 328 for 309
            constexpr int BETWEEN = !G::BYTE ? 7 : NB == 2 ? 11 : 14;
            __builtin_amdgcn_sched_group_barrier(0x2, 20, 0);
#pragma unroll
            for (int i = 0; i < 2 * OPS * N * P; i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, BETWEEN, 0);
            }
        }
        if constexpr (!SECOND) arrived();
        meet();
    }
    if constexpr (TURNS && !SECOND) meet();
    // the last loads are over before their places are another's
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <int PARTS, int GROUP, int NB, int WO, int STAGES>
__global__ __launch_bounds__(128 * WO, 2) void k_q4_gemm(RowsArgs a)
{
    constexpr int S = kGemmStrips, STRIPS = S * WO;
    __shared__ Gemm<PARTS, GROUP, NB, WO, STAGES> stage;
    __shared__ float rest;    // what the weights' 16 times leave to the end (in a register it cost 389 int8 rows 0.9 us)
    const MulArgs& u = a.u;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int strips = q4_strips(u.m.out);
    // panels of kGemmPanel along x's rows, the matrix's rows outermost in a panel
    const int along = (a.blocks + 2 * NB - 1) / (2 * NB), across = (strips + STRIPS - 1) / STRIPS;
    const int all = xcd_remap(blockIdx.x, gridDim.x), split = all / (along * across), id = all - split * along * across;
    const int panel = id / (kGemmPanel * across), p0 = panel * kGemmPanel;
    const int width = min(kGemmPanel, along - p0), in_panel = id - panel * kGemmPanel * across;
    const int xt = p0 + in_panel % width, ot = in_panel / width;
    const int s0 = ot * STRIPS, b0 = xt * 2 * NB;
    const int each = (u.m.tiles + a.splits - 1) / a.splits, t0 = split * each, t1 = min(t0 + each, u.m.tiles);
    uint32_t factors = 0;
    if (a.scaled) {
        uint32_t mine = 0;
        for (int i = threadIdx.x; i < min(2 * NB, a.blocks - b0) * u.m.tiles; i += 128 * WO) mine |= a.scaled[(size_t)b0 * u.m.tiles + i];
        uint32_t* any = reinterpret_cast<uint32_t*>(&stage);   // nothing else is there yet
        mine = (__any(mine & kScaled) ? kScaled : 0u) | (__any(mine & kFar) ? kFar : 0u);
        if (lane == 0) any[wave] = mine;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < 2 * WO; i++) all |= any[i];
        factors = __builtin_amdgcn_readfirstlane(all);
        __syncthreads();
    }
    if (PARTS == 0 && threadIdx.x == 0) rest = factors & kFar ? 1.0f : 0.0625f;
    floatx16 acc[2][NB / 2];
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int n = 0; n < NB / 2; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[s][n][e] = 0.0f;
    auto tiles = [&](auto with_factors) __attribute__((always_inline)) {
        constexpr Factors F = decltype(with_factors)::value;
        if (WO == 4 && wave >= 4) gemm_tiles<PARTS, GROUP, NB, WO, STAGES, F, WO == 4>(a, stage, s0, b0, t0, t1, acc);
        else gemm_tiles<PARTS, GROUP, NB, WO, STAGES, F, false>(a, stage, s0, b0, t0, t1, acc);
    };
    if (factors & kFar) tiles(std::integral_constant<Factors, Factors::apart>{});
    else if (factors) tiles(std::integral_constant<Factors, Factors::with_scales>{});
    else tiles(std::integral_constant<Factors, Factors::none>{});
    if (a.splits > 1) {
        // the splits' sums: [workgroup's place][split][four values][thread], past the
        // XCD's L2, joined in the splits' order by the last one to arrive
        constexpr int FOURS = 2 * (NB / 2) * 4, THREADS = 128 * WO, SOME = 8, ROUND = 4;
        constexpr int SC1 = 16;   // cache policy: at the point of coherence of the card
        const auto place = __builtin_amdgcn_make_buffer_rsrc(a.sums + (size_t)id * a.splits * (FOURS * THREADS * 4), 0, a.splits * (FOURS * THREADS * 16), 0x00020000);
        const int mine = (int)threadIdx.x * 16;
#pragma unroll
        for (int i = 0; i < FOURS; i++) {
            floatx16& v = acc[i / (NB * 2)][i / 4 % (NB / 2)];
            const floatx4 four = {v[i % 4 * 4], v[i % 4 * 4 + 1], v[i % 4 * 4 + 2], v[i % 4 * 4 + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, four), place, mine, (split * FOURS + i) * (THREADS * 16), SC1);
            v[i % 4 * 4] = v[i % 4 * 4 + 1] = v[i % 4 * 4 + 2] = v[i % 4 * 4 + 3] = 0.0f;
        }
        if (!acc_arrive(a.ctr + id, (uint32_t)a.splits, reinterpret_cast<int*>(&stage))) return;
        __syncthreads();   // every wave has read the answer, whose place is another's
        if (threadIdx.x == 0) a.ctr[id] = 0u;
#pragma unroll
        for (int i0 = 0; i0 < FOURS; i0 += SOME)
            for (int q = 0; q < a.splits; q += ROUND) {
                u32x4 v[ROUND][SOME];
#pragma unroll
                for (int j = 0; j < ROUND; j++)
#pragma unroll
                    for (int i = 0; i < SOME; i++)
                        v[j][i] = __builtin_amdgcn_raw_buffer_load_b128(place, mine, (min(q + j, a.splits - 1) * FOURS + i0 + i) * (THREADS * 16), SC1);
#pragma unroll
                for (int j = 0; j < ROUND; j++)
#pragma unroll
                    for (int i = 0; i < SOME; i++) {
                        const floatx4 four = __builtin_bit_cast(floatx4, v[j][i]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[(i0 + i) / (NB * 2)][(i0 + i) / 4 % (NB / 2)][(i0 + i) % 4 * 4 + e] += q + j < a.splits ? four[e] : 0.0f;
                    }
            }
    }
    // Value 4 i + e of a lane is row 8 i + 4 (lane / 32) + e of the pair of strips.
    // 32 rows of x at a time turn in the wave's own part of LDS, for whole lines of
    // y (64 results of a row): pieces of 16 bytes, as the registers hold them, took 2
    // us more (389 rows, 6144 x 4096).
    constexpr int ROW = S * kStrip + 4;    // floats of a row in LDS
    float* turn = reinterpret_cast<float*>(&stage) + wave * (32 * ROW);
    static_assert(sizeof(stage) >= 2 * WO * 32 * ROW * 4, "32 rows of every wave");
    const int o0 = (s0 + (wave >> 1) * S) * kStrip, there = min(u.m.out - o0, S * kStrip);
#pragma unroll
    for (int n = 0; n < NB / 2; n++) {
        const int r0 = (b0 + (wave & 1) * NB + 2 * n) * 16;
        const float rs = a.row_scale ? a.row_scale[min(r0 + (lane & 31), u.rows - 1)] : 1.0f;
        const float first = PARTS == 0 ? rest : 1.0f;    // before the row's scale, which may be among the smallest numbers
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<floatx4*>(turn + (lane & 31) * ROW + 32 * s + 8 * i + 4 * (lane >> 5)) =
                    floatx4{acc[s][n][4 * i], acc[s][n][4 * i + 1], acc[s][n][4 * i + 2], acc[s][n][4 * i + 3]} * first * rs;
        wave_sync();
        // four or eight results a lane
        auto at = [&](int r, int o) { return *reinterpret_cast<const floatx4*>(turn + r * ROW + o); };
        if (u.y_type == IAM_F32) {
            const int o = (lane & 15) * 4;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = i * 4 + (lane >> 4);
                if (r0 + r < u.rows && o < there) put_four(u, r0 + r, o0 + o, at(r, o));
            }
        } else {
            const int o = (lane & 7) * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = i * 8 + (lane >> 3);
                if (r0 + r < u.rows && o < there) put_eight(u, r0 + r, o0 + o, at(r, o), at(r, o + 4));
            }
        }
        wave_sync();
    }
}

// ------------------------------------------------------------------ host ---
template <int PARTS, int GROUP, int S, int NB, int MOST>
static int batch_launch(Ctx* c, RowsArgs a)
{
    const int groups = (q4_strips(a.u.m.out) + S - 1) / S, across = (a.blocks + NB - 1) / NB;
    // The inputs are cut for about a workgroup a CU: by 16 tiles and more (64 bf16
    // rows, 1024 x 14336: 10.6 us, 13.0 by 32), from four operands of x a tile on by 8
    // (64 bf16 rows, 1024 x 4096: 7.6 us, 9.0 by 16; 32 fp32 rows 6.3 and 8.4, but 64 of
    // 1024 x 2048 7.6 and 6.7), single strips of fewer not at all (8 rows: 4.4 whole, 5.1 by 16).
    constexpr bool MANY = PARTS * NB >= 4;
    const int parts = MANY ? a.u.m.tiles >= 32 ? a.u.m.tiles / 8 : 1 : S == 1 ? 1 : a.u.m.tiles / 16;
    a.splits = std::max(1, std::min({256 / (groups * across), kMaxSplits, parts}));
    // waves share a workgroup's tiles evenly
    const int each = (a.u.m.tiles + a.splits - 1) / a.splits, rounds = (each + MOST - 1) / MOST;
    a.waves = (each + rounds - 1) / rounds;
    if (a.splits > 1) {
        IAM_TRY(ensure_q4_sums(c, (size_t)groups * across * a.splits * (S * NB * 256), (size_t)groups * across));
        a.sums = c->q4_sums;
        a.ctr = c->q4_ctr;
    }
    return launch(c, "q4_mul.batch", k_q4_batch<PARTS, GROUP, S, NB, MOST>, dim3((unsigned)(groups * a.splits), (unsigned)across),
                  dim3((unsigned)a.waves * 64), (size_t)a.waves * S * NB * 1024, a);
}

template <int PARTS, int GROUP, int S, int MOST>
static int batch_blocks(Ctx* c, const RowsArgs& a)
{
    // (two parts of four blocks would not fit the registers)
    if (a.blocks == 1) return batch_launch<PARTS, GROUP, S, 1, MOST>(c, a);
    if (a.blocks == 2) return batch_launch<PARTS, GROUP, S, 2, MOST>(c, a);
    return batch_launch<PARTS, GROUP, S, PARTS == 2 || S == 1 ? 2 : 4, MOST>(c, a);
}

template <int PARTS, int GROUP, int NB, int WO, int STAGES>
static int gemm_launch(Ctx* c, RowsArgs a, int splits)
{
    const size_t along = (size_t)(a.blocks + 2 * NB - 1) / (2 * NB), across = (size_t)(q4_strips(a.u.m.out) + kGemmStrips * WO - 1) / (kGemmStrips * WO);
    a.splits = splits;
    if (splits > 1) {
        IAM_TRY(ensure_q4_sums(c, along * across * splits * (NB * WO * 2048), along * across));
        a.sums = c->q4_sums;
        a.ctr = c->q4_ctr;
    }
    return launch(c, "q4_mul.gemm", k_q4_gemm<PARTS, GROUP, NB, WO, STAGES>, dim3((unsigned)(along * across * splits)), dim3(128 * WO), 0, a);
}

// How long workgroups of 64 wo x 32 nb products take for all of them, with the
// inputs cut into the number of parts that is best: 5 us, what `round` says n
// workgroups' tiles of 128 inputs take on 256 CUs, and for several parts the
// join.  Fitted to measured times: of 64 x 128 (128 rows, 6144 x 4096) 29.3 us in one
// part and 21.9 in two, 256 x 64 35.2 and 26.1, 256 x 128 51.7 and 37.5; 389 rows 44.5 and
// 45.9, 39.7 and 53.5, 54.6 and 42.8; 4096 rows, 14336 x 4096 650, 608 and 494 in one;
// 128 rows, 1024 x 14336 90.7 in one, 22.1 in eight.  Rows in 8 bits: 389 of them 30.3
// and 29.8 by 64 x 128, 30.8 and 42.9, 41.2 and 37.5; 4096, 14336 x 4096 387, 453 and 350.
// fp32 rows, by 256 x 64 alone, only look for the number of parts: 128 rows, 6144 x 4096
// 31, 389 rows 62 (one round), 1024 rows 132 (two), 4096 rows, 14336 x 4096 915 (14).
struct GemmCost {
    double us;
    int splits;
};
template <typename F>
static GemmCost gemm_cost(const RowsArgs& a, int nb, int wo, F round)
{
    const int64_t cells = (int64_t)((a.blocks + 2 * nb - 1) / (2 * nb)) * ((q4_strips(a.u.m.out) + kGemmStrips * wo - 1) / (kGemmStrips * wo));
    GemmCost best{INFINITY, 1};
    // (more parts than give every CU four workgroups are not looked at)
    for (int s = 1; s <= kMaxSplits && (s == 1 || (s * cells <= 1024 && a.u.m.tiles >= 4 * s)); s++) {
        const int each = (a.u.m.tiles + s - 1) / s, splits = (a.u.m.tiles + each - 1) / each;
        const double mb = wo * nb * 8192e-6 * splits;   // of a place's sums
        const double us = 5.0 + each * round((int)(cells * splits)) + (s > 1 ? 2.0 + 10.0 * mb + 0.25 * mb * (double)cells : 0.0);
        if (us < best.us) best = {us, splits};
    }
    return best;
}

template <int PARTS, int GROUP>
static int gemm_sized(Ctx* c, const RowsArgs& a)
{
    // (groups of 32 have too many scales for the widest shape's registers; rows in
    // 8 bits were never best by 256 x 64)
    if constexpr (PARTS == 2) {
        return gemm_launch<PARTS, GROUP, 2, 4, 3>(c, a, gemm_cost(a, 2, 4, [](int n) { return 1.5 * ((n + 255) / 256); }).splits);
    } else if constexpr (PARTS <= 0) {
        const GemmCost small = gemm_cost(a, 2, 2, [](int n) { return n <= 256 ? 0.55 : n <= 512 ? 0.8 : 0.41 * ((n + 255) / 256); });
        const GemmCost wide = gemm_cost(a, 4, 4, [](int n) { return 1.45 * ((n - 1) / 256) + 1.0 + 0.4 * ((n - 1) % 256 + 1) / 256; });
        if constexpr (GROUP > 32)
            if (wide.us <= small.us) return gemm_launch<PARTS, GROUP, 4, 4, 3>(c, a, wide.splits);
        return gemm_launch<PARTS, GROUP, 2, 2, 3>(c, a, small.splits);
    } else {
        const GemmCost small = gemm_cost(a, 2, 2, [](int n) { return n <= 256 ? 0.76 : n <= 512 ? 1.24 : 0.72 * ((n + 255) / 256); });
        const GemmCost tall = gemm_cost(a, 2, 4, [](int n) { return 1.36 * ((n - 1) / 256) + 0.85 + 0.35 * ((n - 1) % 256 + 1) / 256; });
        const GemmCost wide = gemm_cost(a, 4, 4, [](int n) { return 2.0 * ((n - 1) / 256) + 1.45 + 0.55 * ((n - 1) % 256 + 1) / 256; });
        if constexpr (GROUP > 32)
            if (wide.us <= small.us && wide.us <= tall.us) return gemm_launch<PARTS, GROUP, 4, 4, 3>(c, a, wide.splits);
        return tall.us < small.us ? gemm_launch<PARTS, GROUP, 2, 4, 3>(c, a, tall.splits) : gemm_launch<PARTS, GROUP, 2, 2, 3>(c, a, small.splits);
    }
}

template <int PARTS, int GROUP>
static int batch_sized(Ctx* c, const RowsArgs& a)
{
    if (a.blocks > 4) {
        if (a.bytes) return a.u.m.zeros ? gemm_sized<-1, GROUP>(c, a) : gemm_sized<0, GROUP>(c, a);
        return gemm_sized<PARTS, GROUP>(c, a);
    }
    // Up to 32 rows a strip a workgroup fills the card where there are few and the
    // matrix's rows are short (32 bf16 rows, 1024 x 4096: 5.4 us against 6.5 of two;
    // 4096 x 4096: 6.3 and 6.8).  Two of them read x's parts half as often and cut
    // long rows instead (4096 x 14336: 13.9 and 12.5; 64 rows of 2048 x 8192: 14.0 and
    // 10.2); four where there are still enough (14336 x 4096: 11.3 of two, 10.7 of
    // four; 64 rows 19.2 and 15.0; 8192 x 8192: 11.3 and 12.5).
    const int strips = q4_strips(a.u.m.out);
    if (a.blocks <= 2 && strips <= 256 && a.u.m.tiles < 64) return batch_blocks<PARTS, GROUP, 1, 16>(c, a);
    return strips < 800 ? batch_blocks<PARTS, GROUP, 2, 8>(c, a) : batch_blocks<PARTS, GROUP, 4, 8>(c, a);
}

template <int PARTS>
static int batch_grouped(Ctx* c, const RowsArgs& a)
{
    if (a.u.m.group == 32) return batch_sized<PARTS, 32>(c, a);
    if (a.u.m.group == 64) return batch_sized<PARTS, 64>(c, a);
    return batch_sized<PARTS, 128>(c, a);
}

// rows of a pass: what x takes as parts stays small beside the card's memory
// (2^29 values), and a launch has at most 2^30 threads (one for 32 products)
constexpr int kRowsSlice = 1 << 14;

int q4_mul_rows(Ctx* c, const MulArgs& all)
{
    const int parts = all.x_type == IAM_F32 ? 2 : 1;
    const int slice = (int)std::min({(int64_t)all.rows, (int64_t)kRowsSlice, ((int64_t)1 << 29) / (all.m.tiles * kTile),
                                     ((int64_t)1 << 35) / (q4_strips(all.m.out) * kStrip)});
    const size_t blocks = (size_t)(slice + 15) / 16, values = blocks * all.m.tiles * 2048;
    IAM_TRY(ensure_q4_scratch(c, values * 2 * parts + blocks * all.m.tiles * (64 + 1)));
    for (int r0 = 0; r0 < all.rows; r0 += slice) {
        MulArgs u = all;
        u.rows = std::min(slice, all.rows - r0);
        u.x = reinterpret_cast<const uint8_t*>(all.x) + (size_t)r0 * all.x_stride * row_type_bytes(all.x_type);
        u.y = reinterpret_cast<uint8_t*>(all.y) + (size_t)r0 * all.y_stride * type_bytes(all.y_type);
        if (u.x_scale) u.x_scale += (size_t)r0 * u.x_groups;
        RowsArgs a{};
        a.u = u;
        a.parts = reinterpret_cast<_Float16*>(c->q4_part);
        a.part_stride = values;
        a.blocks = (u.rows + 15) / 16;
        a.bytes = u.x_type == IAM_I8 && a.blocks > 4;
        float* factor = reinterpret_cast<float*>(c->q4_part + values * 2 * parts);
        uint8_t* scaled = reinterpret_cast<uint8_t*>(factor + blocks * all.m.tiles * 16);
        a.factor = factor;
        a.scaled = u.x_type == IAM_F32 || u.x_type == IAM_BF16 || u.x_groups > 1 ? scaled : nullptr;
        // a scale for each tile goes with the tiles; one of the whole row at the end
        const bool by_tile = u.x_groups > 1;
        a.row_scale = by_tile ? nullptr : u.x_scale;
        const PrepArgs p{u.x, u.x_type, u.x_stride, by_tile ? u.x_scale : nullptr, u.rows, u.m.in, u.m.tiles,
                         reinterpret_cast<_Float16*>(c->q4_part), values, factor, scaled, a.bytes ? 0 : parts};
        const dim3 grid((unsigned)((u.m.tiles + 3) / 4), (unsigned)a.blocks);
        IAM_TRY(launch(c, "q4_mul.prepare", k_q4_prep, grid, dim3(kPrepThreads), 0, p));
        IAM_TRY(parts == 2 ? batch_grouped<2>(c, a) : batch_grouped<1>(c, a));
    }
    return IAM_OK;
}

}  // namespace iam
