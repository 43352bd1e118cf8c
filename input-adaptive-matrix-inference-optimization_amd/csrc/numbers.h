// Activations in fp32, fp16 or bf16 (IAM_F32, IAM_F16, IAM_BF16) as the
// long-context operators read and write them, and small helpers they share.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"

namespace iam {

inline size_t type_bytes(int type) { return type == IAM_F32 ? 4 : 2; }

// one rounding to the type, to nearest even
template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// N consecutive values; the compiler loads and stores them with as few
// instructions as the alignment ALIGN (bytes) allows
template <typename T, int N, int ALIGN = N * (int)sizeof(T)>
struct alignas(ALIGN) Pack {
    T v[N];
};

// The call's device for as long as the call lasts: a context's launches go to
// its own device whichever one the thread has current.
struct DeviceGuard {
    int was = -1;
    bool moved = false;
    explicit DeviceGuard(const Ctx* c)
    {
        if (hipGetDevice(&was) == hipSuccess && was != c->device) moved = hipSetDevice(c->device) == hipSuccess;
    }
    ~DeviceGuard()
    {
        if (moved) (void)hipSetDevice(was);
    }
};

inline bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// whether [a, a + an) and [b, b + bn) share bytes
inline bool overlaps(const void* a, size_t an, const void* b, size_t bn)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + bn && y < x + an;
}

// bytes of `rows` rows of `width` values, `stride` values apart (2^62, which no
// allocation holds, where they would not fit 64 bits)
inline size_t rows_bytes(size_t rows, size_t width, size_t stride, size_t value)
{
    size_t n;
    if (!rows) return 0;
    if (__builtin_mul_overflow(rows - 1, stride, &n) || __builtin_add_overflow(n, width, &n) ||
        __builtin_mul_overflow(n, value, &n))
        return (size_t)1 << 62;
    return std::min(n, (size_t)1 << 62);
}

}  // namespace iam
