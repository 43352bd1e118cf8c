// What the kernels of the 4-bit products share: arguments and results.
#pragma once

#include "q4.h"
#include "wave.h"

namespace iam {

struct MulArgs {
    Q4 m;
    const void* x;
    int x_type;
    size_t x_stride;
    const float* x_scale;   // 8-bit rows
    int x_groups;           // scales of a row
    int rows;
    void* y;
    int y_type;
    size_t y_stride;
};

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void put_value(void* y, int type, size_t at, float v)
{
    if (type == IAM_F32) reinterpret_cast<float*>(y)[at] = v;
    else if (type == IAM_F16) reinterpret_cast<_Float16*>(y)[at] = (_Float16)v;
    else reinterpret_cast<__bf16*>(y)[at] = (__bf16)v;
}

// Eight values of a row from place k on (zeros past its end), as they lie:
// f32 takes both words, 16 bits the first, 8 bits its first half.
struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw8(const void* x, int type, size_t row, int k, int in)
{
    Raw8 r{};
    const bool whole = k + 8 <= in;
    if (type == IAM_F32) {
        const float* p = reinterpret_cast<const float*>(x) + row + k;
        if (whole) {
            r.a = __builtin_bit_cast(uint4, *reinterpret_cast<const Pack<float, 4, 4>*>(p));
            r.b = __builtin_bit_cast(uint4, *reinterpret_cast<const Pack<float, 4, 4>*>(p + 4));
        } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = k + e < in ? __float_as_uint(p[e]) : 0u;
            r.a = {w[0], w[1], w[2], w[3]};
            r.b = {w[4], w[5], w[6], w[7]};
        }
    } else if (!is_8bit_type(type)) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + row + k;
        if (whole) {
            r.a = __builtin_bit_cast(uint4, *reinterpret_cast<const Pack<uint16_t, 8, 2>*>(p));
        } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = k + e < in ? p[e] : 0u;
            r.a = {w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
        }
    } else {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(x) + row + k;
        uint32_t w[2] = {0, 0};
        if (whole) {
            const uint2 v = __builtin_bit_cast(uint2, *reinterpret_cast<const Pack<uint8_t, 8, 1>*>(p));
            w[0] = v.x;
            w[1] = v.y;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e >> 2] |= (k + e < in ? (uint32_t)p[e] : 0u) << (8 * (e & 3));
        }
        r.a.x = w[0];
        r.a.y = w[1];
    }
    return r;
}

// their values (8 bits: the numbers, without their scale)
__device__ __forceinline__ void values8(const Raw8& r, int type, float* v)
{
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == IAM_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __uint_as_float(w[e]);
    } else if (type == IAM_F16) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e >> 1] >> (16 * (e & 1))));
    } else if (type == IAM_BF16) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    } else if (type == IAM_I8) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3)));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e4m3_value((uint8_t)(w[e >> 2] >> (8 * (e & 3))));
    }
}

// one launch for few rows: whether it takes these
bool q4_takes_few(const MulArgs& a);
int q4_mul_few(Ctx* c, const MulArgs& a);
// any number of them
int q4_mul_rows(Ctx* c, const MulArgs& a);

// A wave's LDS operations take place in order: this keeps them in the order they are written in.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace iam
