// The 8-bit KV cache's order of values and conversions, shared by its writers
// and the attention over it.
#pragma once

#include "numbers.h"

namespace iam {

constexpr int kBlk = IAM_KV8_BLOCK;   // tokens that share a scale

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// A block's values of one KV head ("tile") in the order the attention's
// 16x16x32 matrix instructions take their first operand: lane l = 16 g + r of
// a wave holds 16 consecutive values of a group of 1024.
// K: group (16 tokens, 64 dimensions), r the token, 16 dimensions from 16 g on
// (the first 8 go into one instruction, the others into the next).
template <int HD>
__host__ __device__ __forceinline__ int k_place(int t, int d)
{
    return (((t >> 4) * (HD / 64) + (d >> 6)) * 64 + ((d & 63) >> 4) * 16 + (t & 15)) * 16 + (d & 15);
}
// V: group (16 dimensions, 64 tokens), r the dimension; per 32 tokens the 8
// that the lane's own probabilities belong to: 4 g .. 4 g + 3 and 16 more of each.
__host__ __device__ __forceinline__ int v_place(int t, int d)
{
    return ((d >> 4) * 64 + ((t >> 2) & 3) * 16 + (d & 15)) * 16 + (t >> 5) * 8 + ((t >> 4) & 1) * 4 + (t & 3);
}

// Four 8-bit numbers as fp16 (exact): two pairs, low bytes first.
// INT8: the byte (number + 128) under the exponent of 1024 is 1024 + byte,
// 1152 more than the number.
template <int FMT>
__device__ __forceinline__ void widen4(uint32_t w, half2v& lo, half2v& hi)
{
    if constexpr (FMT == IAM_KV8_INT8) {
        const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
    } else {
        lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
}

// The exact quotient x / s rounded to odd: one more rounding, to nearest even
// at 22 bits or fewer, then gives the correctly rounded result.  r: 1 / s,
// correctly rounded.  q is x r with its error taken out, within a step of
// the quotient; the sign of x - q s says on which side.
__device__ __forceinline__ float quotient_odd(float x, float s, float r)
{
    const float q0 = __fmul_rn(x, r);
    const float q = __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0);
    const float e = __builtin_fmaf(-q, s, x);
    int b = __float_as_int(q);
    if (e != 0.0f && !(b & 1)) b += ((e > 0.0f) == (x > 0.0f)) ? 1 : -1;
    return __int_as_float(b);
}

// x / s as an 8-bit number, in the low byte; s > 0
template <int FMT>
__device__ __forceinline__ uint32_t narrow(float x, float s, float r)
{
    const float q = x != 0.0f ? quotient_odd(x, s, r) : 0.0f;
    if constexpr (FMT == IAM_KV8_INT8) return (uint32_t)((int)rintf(q) + 128);
    else return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false) & 0xffu;
}
// the number 0
template <int FMT>
constexpr uint32_t kv8_zero() { return FMT == IAM_KV8_INT8 ? 128u : 0u; }

// the scale of a block whose largest magnitude is 1
template <int FMT>
constexpr float kv8_unit() { return FMT == IAM_KV8_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f; }

struct Kv8Geometry {
    int n_seq, max_ctx, n_kv, blocks;
};

// offsets in 64 bits: a long cache passes 2^31 bytes
__device__ __forceinline__ size_t kv8_cell(const Kv8Geometry& g, int seq, int block, int head)
{
    return ((size_t)seq * g.blocks + block) * g.n_kv + head;
}

inline int kv8_blocks(int max_ctx) { return max_ctx / kBlk + (max_ctx % kBlk != 0); }

// checks the cache's shape and memory
int kv8_check(Ctx* c, const iam_kv8_cache* k, const char* what);
// whether [p, p + bytes) shares bytes with a part of the (checked) cache
bool kv8_overlaps(const iam_kv8_cache* k, const void* p, size_t bytes);

}  // namespace iam
