// 4-bit weights: the order of their numbers, scales and zero points, and what
// the kernels that read them share.
#pragma once

#include "numbers.h"

namespace iam {

constexpr int kStrip = 16;            // rows of a strip
constexpr int kTile = 128;            // inputs of a tile: 1024 bytes of a strip
constexpr int kChunk = 512;           // inputs of a chunk, whose scales lie together

// A matrix as the kernels take it.
struct Q4 {
    const uint8_t* numbers;
    const uint16_t* scales;
    const uint8_t* zeros;     // null: 8 everywhere
    int out, in, group;
    int tiles, chunks;        // of a strip
};

__host__ __device__ inline int q4_tiles(int in) { return (in + kTile - 1) / kTile; }
__host__ __device__ inline int q4_chunks(int in) { return (in + kChunk - 1) / kChunk; }
__host__ __device__ inline int q4_strips(int out) { return (out + kStrip - 1) / kStrip; }

// Where the number of (row o, input k) lies: the 4-byte word, and its four bits
// there.  A word's numbers are in pairs 16 bits apart, (0, 1), (2, 3) ..: one
// mask takes two that lie next to each other, as the 16-bit operands want
// them.
__host__ __device__ inline size_t q4_word(const Q4& m, int o, int k)
{
    const int t = k / kTile, j = k % kTile / 32, g = k % 32 / 8;
    return (((size_t)(o / kStrip) * m.tiles + t) * 64 + g * 16 + o % kStrip) * 4 + j;
}
__host__ __device__ inline int q4_shift(int k) { return (k % 8 / 2 + (k & 1) * 4) * 4; }

// the scale's and the zero point's place
__host__ __device__ inline size_t q4_scale(const Q4& m, int o, int k)
{
    const int per = kChunk / m.group, r = o % kStrip;
    return (((size_t)(o / kStrip) * m.chunks + k / kChunk) * 4 + r / 4) * (per * 4) + k % kChunk / m.group * 4 + r % 4;
}
__host__ __device__ inline size_t q4_zero(const Q4& m, int o, int k)
{
    const int per = kChunk / m.group;
    return (((size_t)(o / kStrip) * m.chunks + k / kChunk) * kStrip + o % kStrip) * per + k % kChunk / m.group;
}

// checks a matrix's shape and memory
int q4_check(Ctx* c, const iam_q4_matrix* m, const char* what);
Q4 q4_of(const iam_q4_matrix* m);
struct Q4Bytes {
    size_t numbers, scales, zeros;
};
Q4Bytes q4_bytes(int out, int in, int group);
// whether [p, p + bytes) shares bytes with a part of the (checked) matrix
bool q4_overlaps(const iam_q4_matrix* m, const void* p, size_t bytes);

// rows of values of any type
__host__ __device__ inline bool is_float_type(int t) { return t == IAM_F32 || t == IAM_F16 || t == IAM_BF16; }
__host__ __device__ inline bool is_8bit_type(int t) { return t == IAM_I8 || t == IAM_E4M3; }
inline size_t row_type_bytes(int t) { return is_8bit_type(t) ? 1 : type_bytes(t); }

// the value of an e4m3 byte
__device__ __forceinline__ float e4m3_value(uint8_t b)
{
    typedef float float2v __attribute__((ext_vector_type(2)));
    const float2v v = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, false);
    return v[0];
}

}  // namespace iam
