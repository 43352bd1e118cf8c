// Products of many rows (batches, prompts) with 4-bit weights, on the fp16 matrix
// instructions.
//
// A launch of its own brings x into the instructions' order as fp16: one part
// of values that fp16 holds (fp16 and 8-bit numbers; bf16 of a tile of 128 after
// a power of two where its largest value lies outside [2^-2, 2^15)), two, high
// and low, of fp32 (22 bits).  4-bit weights become fp16 under the exponents of
// 1024 and 64, n - zero exactly.  Products are then exact; a group's are added
// in fp32 by the instructions and go to the row's sum with the group's scale.
#include "q4_mul.h"

namespace iam {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// ---- x in the operands' order
// parts  fp16 [part][block of 16 rows][tile][j][lane 16 g + row][8]: inputs
//        32 j + 8 g and on of the tile
// factor fp32 [block][tile][16]: what the tile's values were divided by
struct PrepArgs {
    const void* x;
    int type;
    size_t stride;
    const float* x_scale;    // with a scale for each tile (else null)
    int rows, in, tiles;
    _Float16* parts;
    size_t part_stride;      // values of a part
    float* factor;
    int parts_n;
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
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const Raw8 r = load_raw8(a.x, a.type, (size_t)(there ? row : 0) * a.stride, tile * kTile + 32 * j + 8 * g, there ? a.in : 0);
        values8(r, a.type, v[j]);
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
    if (g == 0) a.factor[((size_t)block * a.tiles + tile) * 16 + c] = f;
}

// ---- the products
struct RowsArgs {
    MulArgs u;
    const _Float16* parts;
    size_t part_stride;
    const float* factor;
    const float* row_scale;   // of a whole row, or null
    bool factors;             // whether factor may hold anything but 1
    int blocks;               // of 16 rows
    int waves;
};

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

// A workgroup takes S strips of the matrix and NB blocks of 16 rows; its waves
// deal the tiles of 128 inputs among themselves and join their sums in LDS.
// Every operand comes straight from memory in the order in which it is used.
template <int PARTS, int GROUP, int S, int NB>
__global__ __launch_bounds__(1024) void k_q4_batch(RowsArgs a)
{
    extern __shared__ floatx4 join[];
    constexpr int GT = kTile / GROUP;      // groups of a tile
    const MulArgs& u = a.u;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int strips = q4_strips(u.m.out), s0 = xcd_remap(blockIdx.x, gridDim.x) * S, b0 = blockIdx.y * NB;
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
    uint4 next[S];
    if (wave < u.m.tiles) {
#pragma unroll
        for (int s = 0; s < S; s++) next[s] = words[s][(size_t)wave * 64];
    }
    for (int t = wave; t < u.m.tiles; t += a.waves) {
        half8 x[PARTS][NB][4];
        float f[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const size_t cell = (size_t)min(b0 + n, a.blocks - 1) * u.m.tiles + t;
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int j = 0; j < 4; j++) x[p][n][j] = *reinterpret_cast<const half8*>(a.parts + p * a.part_stride + (cell * 4 + j) * 512 + lane * 8);
            f[n] = a.factor[cell * 16 + c];
        }
        uint4 w[S];
        half4 sc[S][GT];
        uint32_t zero[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            w[s] = next[s];
            const size_t cell = (size_t)strip[s] * u.m.chunks + (t >> 2);
            const half4* q = reinterpret_cast<const half4*>(u.m.scales) + (cell * 4 + g) * (4 * GT) + (t & 3) * GT;
#pragma unroll
            for (int i = 0; i < GT; i++) sc[s][i] = q[i];
            zero[s] = 0x08080808u;
            if (u.m.zeros) {
                const uint8_t* z = u.m.zeros + (cell * kStrip + c) * (4 * GT) + (t & 3) * GT;
                if constexpr (GT == 1) zero[s] = *z;
                else if constexpr (GT == 2) zero[s] = *reinterpret_cast<const uint16_t*>(z);
                else zero[s] = *reinterpret_cast<const uint32_t*>(z);
            }
        }
        if (t + a.waves < u.m.tiles) {
#pragma unroll
            for (int s = 0; s < S; s++) next[s] = words[s][(size_t)(t + a.waves) * 64];
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
            const uint32_t wd[4] = {w[s].x, w[s].y, w[s].z, w[s].w};
            half8 wide[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const Minus m = minus_of(zero[s] >> (8 * (j * 32 / GROUP)) & 255u);
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
                        for (int p = 0; p < PARTS; p++) d = mfma_f16(wide[j], x[p][n][j], d);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[s][n][e] = __builtin_fmaf(d[e] * f[n], (float)sc[s][i][e], acc[s][n][e]);
                }
            }
        }
    }
    if (a.waves > 1) {
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int n = 0; n < NB; n++) join[(wave * S * NB + s * NB + n) * 64 + lane] = acc[s][n];
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const int i = s * NB + n;
            if (i % a.waves != wave) continue;
            floatx4 v = acc[s][n];
            if (a.waves > 1) {
                v = join[i * 64 + lane];
                for (int q = 1; q < a.waves; q++) v += join[(q * S * NB + i) * 64 + lane];
            }
            const int r = (b0 + n) * 16 + c;
            if (s0 + s >= strips || r >= u.rows) continue;
            if (a.row_scale) v *= a.row_scale[r];
            put_four(u, r, (s0 + s) * kStrip + 4 * g, v);
        }
}

// Many rows: a workgroup takes 64 WO rows of the matrix and 32 NB of x, its
// waves WO by two 64 x 16 NB of them.  What a tile of 128 inputs needs goes to
// LDS past the registers, STAGES - 1 tiles ahead: x's operands and the strips'
// words in runs of 1 KB, a share for each wave, then scales and zero points.
constexpr int kGemmStrips = 4;     // of a wave
constexpr int kGemmPanel = 8;      // workgroups side by side along x's rows that run together

template <int PARTS, int GROUP, int NB, int WO, int STAGES>
struct Gemm {
    static constexpr int GT = kTile / GROUP, S = kGemmStrips, WAVES = 2 * WO, STRIPS = S * WO;
    static constexpr int X = PARTS * 2 * NB * 4, RUNS = X + STRIPS, SHARE = RUNS / WAVES;
    static constexpr int SCALES = RUNS * 1024;                      // [group][strip][g] four halves
    static constexpr int ZEROS = SCALES + GT * STRIPS * 32;         // [strip][row] words
    static constexpr int BYTES = ZEROS + STRIPS * 64;
    static constexpr int PER_GROUP = STRIPS / 8, SMALL = GT * PER_GROUP + STRIPS / 4;   // loads of 256 bytes
    static_assert(RUNS % WAVES == 0, "every wave brings as many runs");
    uint4 at[STAGES][BYTES / 16];
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// LDS reads in one piece of assembly with their wait: the compiler, which
// cannot tell the stages apart, would wait for all loads in flight to LDS
// before any of them.
__device__ __forceinline__ void read_runs8(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:1024\n\tds_read_b128 %2, %8 offset:2048\n\tds_read_b128 %3, %8 offset:3072\n\t"
        "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %8 offset:5120\n\tds_read_b128 %6, %8 offset:6144\n\tds_read_b128 %7, %8 offset:7168\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(at)
        : "memory");
}
__device__ __forceinline__ void read_runs16(uint32_t at, u32x4* r)
{
    asm volatile(
        "ds_read_b128 %0, %16\n\tds_read_b128 %1, %16 offset:1024\n\tds_read_b128 %2, %16 offset:2048\n\tds_read_b128 %3, %16 offset:3072\n\t"
        "ds_read_b128 %4, %16 offset:4096\n\tds_read_b128 %5, %16 offset:5120\n\tds_read_b128 %6, %16 offset:6144\n\tds_read_b128 %7, %16 offset:7168\n\t"
        "ds_read_b128 %8, %16 offset:8192\n\tds_read_b128 %9, %16 offset:9216\n\tds_read_b128 %10, %16 offset:10240\n\tds_read_b128 %11, %16 offset:11264\n\t"
        "ds_read_b128 %12, %16 offset:12288\n\tds_read_b128 %13, %16 offset:13312\n\tds_read_b128 %14, %16 offset:14336\n\tds_read_b128 %15, %16 offset:15360\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]), "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]),
          "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
        : "v"(at)
        : "memory");
}
// four strips' words, zero points and scales of the first group
__device__ __forceinline__ void read_words(uint32_t words, uint32_t zeros, uint32_t scales, u32x4* w, uint32_t* z, u32x2* s)
{
    asm volatile(
        "ds_read_b128 %0, %12\n\tds_read_b128 %1, %12 offset:1024\n\tds_read_b128 %2, %12 offset:2048\n\tds_read_b128 %3, %12 offset:3072\n\t"
        "ds_read_b32 %4, %13\n\tds_read_b32 %5, %13 offset:64\n\tds_read_b32 %6, %13 offset:128\n\tds_read_b32 %7, %13 offset:192\n\t"
        "ds_read_b64 %8, %14\n\tds_read_b64 %9, %14 offset:32\n\tds_read_b64 %10, %14 offset:64\n\tds_read_b64 %11, %14 offset:96\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(z[0]), "=&v"(z[1]), "=&v"(z[2]), "=&v"(z[3]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(words), "v"(zeros), "v"(scales)
        : "memory");
}
// four strips' scales of a group
__device__ __forceinline__ void read_scales(uint32_t at, u32x2* s)
{
    asm volatile(
        "ds_read_b64 %0, %4\n\tds_read_b64 %1, %4 offset:32\n\tds_read_b64 %2, %4 offset:64\n\tds_read_b64 %3, %4 offset:96\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(at)
        : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }

// Tiles of a workgroup's products, with x's factors or (they are all 1) without.
// The two are loops of their own: no branch may lie between a matrix
// instruction and its results' first use, where the compiler leaves out the
// wait states of the edge that jumps.
template <int PARTS, int GROUP, int NB, int WO, int STAGES, bool FACTORS, bool SECOND>
__device__ __forceinline__ void gemm_tiles(const RowsArgs& a, Gemm<PARTS, GROUP, NB, WO, STAGES>& stage, int s0, int b0, floatx4 (&acc)[kGemmStrips][NB])
{
    typedef Gemm<PARTS, GROUP, NB, WO, STAGES> G;
    constexpr int GT = G::GT, S = G::S;
    const MulArgs& u = a.u;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
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
            const int b = min(b0 + (i >> 2) % (2 * NB), a.blocks - 1), p = (i >> 2) / (2 * NB);
            run[q] = reinterpret_cast<const uint8_t*>(a.parts + p * a.part_stride + ((size_t)b * u.m.tiles * 4 + (i & 3)) * 512);
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
            const uint8_t* src = run[q] + (uint32_t)t * ((q + 1) * G::WAVES <= G::X ? 4096u : 1024u);
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
    float f[NB];
    auto load_factors = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NB; n++) f[n] = a.factor[((size_t)min(b0 + wx * NB + n, a.blocks - 1) * u.m.tiles + t) * 16 + c];
    };
    if constexpr (FACTORS) load_factors(0);
#pragma unroll
    for (int t = 0; t < STAGES - 1; t++) fetch(min(t, u.m.tiles - 1), t);
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
    // matrix instructions idle: .)
    constexpr bool TURNS = G::WAVES == 8;
    arrived();
    meet();
    if constexpr (SECOND) meet();
#pragma unroll 1
    for (int t = 0; t < u.m.tiles; t++) {
        // Every wave's loads of this tile have arrived, and every wave has read
        // the tile before, whose place the newest tile takes.
        float fn[NB];
        if constexpr (FACTORS) {
#pragma unroll
            for (int n = 0; n < NB; n++) fn[n] = f[n];
            load_factors(min(t + 1, u.m.tiles - 1));
        }
        fetch(min(t + STAGES - 1, u.m.tiles - 1), free_buf);   // behind the last tile, the last one again
        const uint32_t at = base + buf * G::BYTES;
        free_buf = buf;
        buf = buf + 1 == STAGES ? 0 : buf + 1;
        u32x4 x[PARTS][NB * 4], w[S];
        u32x2 sc[GT][S];
        uint32_t zero[S];
        read_words(at + (G::X + wo * S) * 1024 + lane16, at + G::ZEROS + wo * S * 64 + c * 4, at + G::SCALES + wo * S * 32 + g * 8, w, zero, sc[0]);
#pragma unroll
        for (int i = 1; i < GT; i++) read_scales(at + G::SCALES + i * G::STRIPS * 32 + wo * S * 32 + g * 8, sc[i]);
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const uint32_t from = at + (p * 2 + wx) * NB * 4096 + lane16;
            if constexpr (NB == 4) read_runs16(from, x[p]);
            else read_runs8(from, x[p]);
        }
        // the next tile's loads, as late as the other group's turn allows
        if constexpr (SECOND) arrived();
        if constexpr (TURNS) meet();
#pragma unroll
        for (int s = 0; s < S; s++) {
            half8 wide[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t z = !u.m.zeros ? 8u
                                   : GT == 1  ? zero[s] >> (8 * (t & 3))
                                   : GT == 2  ? zero[s] >> (16 * (t & 1) + 8 * (j >> 1))
                                              : zero[s] >> (8 * j);
                const Minus m = minus_of(z & 255u);
                wide[j] = widen_half(w[s][j], m.k1024, m.k64);
            }
#pragma unroll
            for (int i = 0; i < GT; i++) {
                floatx4 d[NB];
                const half4 scale = __builtin_bit_cast(half4, sc[i][s]);
#pragma unroll
                for (int n = 0; n < NB; n++) d[n] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int j = i * 4 / GT; j < (i + 1) * 4 / GT; j++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int n = 0; n < NB; n++) d[n] = mfma_f16(wide[j], __builtin_bit_cast(half8, x[p][n * 4 + j]), d[n]);
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[s][n][e] = __builtin_fmaf(FACTORS ? d[n][e] * fn[n] : d[n][e], (float)scale[e], acc[s][n][e]);
            }
            if constexpr (GT > 1) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (GT == 1) {
            // the widening of the next strip and the sums of the last between
            // the matrix instructions (by strips, as below: ); smaller groups
            // would spill
            __builtin_amdgcn_sched_group_barrier(0x2, 40, 0);
#pragma unroll
            for (int i = 0; i < S * NB * 4 * PARTS; i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
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
    const MulArgs& u = a.u;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int strips = q4_strips(u.m.out);
    // panels of kGemmPanel along x's rows, the matrix's rows outermost in a panel
    const int along = (a.blocks + 2 * NB - 1) / (2 * NB), across = (strips + STRIPS - 1) / STRIPS;
    const int id = xcd_remap(blockIdx.x, gridDim.x), panel = id / (kGemmPanel * across), p0 = panel * kGemmPanel;
    const int width = min(kGemmPanel, along - p0), in_panel = id - panel * kGemmPanel * across;
    const int xt = p0 + in_panel % width, ot = in_panel / width;
    const int s0 = ot * STRIPS, b0 = xt * 2 * NB;
    bool factors = false;
    if (a.factors) {
        // whether any is not 1
        const int blocks = min(2 * NB, a.blocks - b0);
        const float4* q = reinterpret_cast<const float4*>(a.factor + (size_t)b0 * u.m.tiles * 16);
        bool mine = false;
        for (int i = threadIdx.x; i < blocks * u.m.tiles * 4; i += 128 * WO) {
            const float4 v = q[i];
            mine |= v.x != 1.0f || v.y != 1.0f || v.z != 1.0f || v.w != 1.0f;
        }
        uint32_t* any = reinterpret_cast<uint32_t*>(&stage);   // nothing else is there yet
        if (lane == 0) any[wave] = 0;
        if (mine) any[wave] = 1;
        __syncthreads();
        uint32_t all = 0;
        for (int i = 0; i < 2 * WO; i++) all |= any[i];
        factors = __builtin_amdgcn_readfirstlane(all) != 0;
        __syncthreads();
    }
    floatx4 acc[S][NB];
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int n = 0; n < NB; n++) acc[s][n] = floatx4{0, 0, 0, 0};
    auto tiles = [&](auto with_factors) __attribute__((always_inline)) {
        constexpr bool F = decltype(with_factors)::value;
        if (WO == 4 && wave >= 4) gemm_tiles<PARTS, GROUP, NB, WO, STAGES, F, WO == 4>(a, stage, s0, b0, acc);
        else gemm_tiles<PARTS, GROUP, NB, WO, STAGES, F, false>(a, stage, s0, b0, acc);
    };
    if (factors) tiles(std::true_type{});
    else tiles(std::false_type{});
#pragma unroll
    for (int n = 0; n < NB; n++) {
        const int r = (b0 + (wave & 1) * NB + n) * 16 + c;
        if (r >= u.rows) continue;
        const float rs = a.row_scale ? a.row_scale[r] : 1.0f;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int strip = s0 + (wave >> 1) * S + s;
            if (strip < strips) put_four(u, r, strip * kStrip + 4 * g, acc[s][n] * rs);
        }
    }
}

// ------------------------------------------------------------------ host ---
template <int PARTS, int GROUP, int S, int NB>
static int batch_launch(Ctx* c, RowsArgs a)
{
    // as many waves as there are tiles, up to 16 and what LDS holds of their sums
    const int most = std::min(16, 160 / (S * NB));
    const int rounds = (a.u.m.tiles + most - 1) / most;
    a.waves = (a.u.m.tiles + rounds - 1) / rounds;
    const dim3 grid((unsigned)((q4_strips(a.u.m.out) + S - 1) / S), (unsigned)((a.blocks + NB - 1) / NB));
    return launch(c, "q4_mul.batch", k_q4_batch<PARTS, GROUP, S, NB>, grid, dim3((unsigned)a.waves * 64), (size_t)a.waves * S * NB * 1024, a);
}

template <int PARTS, int GROUP, int NB, int WO, int STAGES>
static int gemm_launch(Ctx* c, const RowsArgs& a)
{
    const size_t along = (size_t)(a.blocks + 2 * NB - 1) / (2 * NB), across = (size_t)(q4_strips(a.u.m.out) + kGemmStrips * WO - 1) / (kGemmStrips * WO);
    return launch(c, "q4_mul.gemm", k_q4_gemm<PARTS, GROUP, NB, WO, STAGES>, dim3((unsigned)(along * across)), dim3(128 * WO), 0, a);
}

template <int PARTS, int GROUP>
static int batch_sized(Ctx* c, const RowsArgs& a)
{
    if (a.blocks > 4) {
        if constexpr (PARTS == 2) {
            return gemm_launch<PARTS, GROUP, 2, 4, 3>(c, a);
        } else {
            if (a.blocks > 32) return gemm_launch<PARTS, GROUP, 4, 4, 3>(c, a);
            return gemm_launch<PARTS, GROUP, 2, 2, 3>(c, a);
        }
    }
    if (a.blocks == 1) return batch_launch<PARTS, GROUP, 2, 1>(c, a);
    if (a.blocks == 2 || PARTS == 2) return batch_launch<PARTS, GROUP, 1, 2>(c, a);
    return batch_launch<PARTS, GROUP, 2, PARTS == 2 ? 2 : 4>(c, a);
}

template <int PARTS>
static int batch_grouped(Ctx* c, const RowsArgs& a)
{
    if (a.u.m.group == 32) return batch_sized<PARTS, 32>(c, a);
    if (a.u.m.group == 64) return batch_sized<PARTS, 64>(c, a);
    return batch_sized<PARTS, 128>(c, a);
}

// rows of a pass: what x takes as parts stays small beside the card's memory
constexpr int kRowsSlice = 1 << 14;

int q4_mul_rows(Ctx* c, const MulArgs& all)
{
    const int parts = all.x_type == IAM_F32 ? 2 : 1;
    const int slice = std::min(all.rows, kRowsSlice);
    const size_t blocks = (size_t)(slice + 15) / 16, values = blocks * all.m.tiles * 2048;
    IAM_TRY(ensure_q4_scratch(c, values * 2 * parts + blocks * all.m.tiles * 64));
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
        a.factors = u.x_type == IAM_F32 || u.x_type == IAM_BF16 || u.x_groups > 1;
        float* factor = reinterpret_cast<float*>(c->q4_part + values * 2 * parts);
        a.factor = factor;
        // a scale for each tile goes with the tiles; one of the whole row at the end
        const bool by_tile = u.x_groups > 1;
        a.row_scale = by_tile ? nullptr : u.x_scale;
        const PrepArgs p{u.x, u.x_type, u.x_stride, by_tile ? u.x_scale : nullptr, u.rows, u.m.in, u.m.tiles,
                         reinterpret_cast<_Float16*>(c->q4_part), values, factor, parts};
        const dim3 grid((unsigned)((u.m.tiles + 3) / 4), (unsigned)a.blocks);
        IAM_TRY(launch(c, "q4_mul.prepare", k_q4_prep, grid, dim3(kPrepThreads), 0, p));
        IAM_TRY(parts == 2 ? batch_grouped<2>(c, a) : batch_grouped<1>(c, a));
    }
    return IAM_OK;
}

}  // namespace iam
