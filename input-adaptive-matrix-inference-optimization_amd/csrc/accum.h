// Global accumulators of the decode step: fp64 (or fp32) sums built with
// relaxed agent-scope atomics by many workgroups, read and cleared in one
// atomic exchange, and cleared in shares by the workgroups of a later
// launch.
#pragma once

#include <hip/hip_runtime.h>

namespace iam {

__device__ __forceinline__ void acc_add(double* p, double v) { unsafeAtomicAdd(p, v); }
__device__ __forceinline__ void acc_add(float* p, float v) { unsafeAtomicAdd(p, v); }

// the value, leaving zero behind
__device__ __forceinline__ double acc_take(double* p)
{
    const unsigned long long b = __hip_atomic_exchange(reinterpret_cast<unsigned long long*>(p), 0ull,
                                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __longlong_as_double((long long)b);
}
__device__ __forceinline__ float acc_take(float* p)
{
    const unsigned int b = __hip_atomic_exchange(reinterpret_cast<unsigned int*>(p), 0u, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
    return __uint_as_float(b);
}

// the value, read at the point of coherence of the atomics
__device__ __forceinline__ double acc_peek(double* p)
{
    const unsigned long long b = __hip_atomic_load(reinterpret_cast<unsigned long long*>(p), __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
    return __longlong_as_double((long long)b);
}
__device__ __forceinline__ float acc_peek(float* p)
{
    return __uint_as_float(__hip_atomic_load(reinterpret_cast<unsigned int*>(p), __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT));
}

// Results handed from one workgroup to the last one of a group to arrive:
// stores past the XCD's L2 (agent-scope atomics), the wait until they are
// performed, then the arrival; the last one reads with acc_peek.  An
// agent-scope fence instead writes back and invalidates the whole L2: with one
// in each of 1556 workgroups, 389 rows of 32000 logits took 198 us.
__device__ __forceinline__ void acc_put(double* p, double v)
{
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), (unsigned long long)__double_as_longlong(v),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void acc_put(float* p, float v)
{
    __hip_atomic_store(reinterpret_cast<unsigned int*>(p), __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void acc_put(unsigned long long* p, unsigned long long v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long acc_peek(unsigned long long* p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// every thread of the workgroup, after its acc_puts; whether this workgroup is
// the last of n (its counter, zero before the first, is then the caller's to
// clear with a plain store).  s: LDS
__device__ __forceinline__ bool acc_arrive(uint32_t* ctr, uint32_t n, int* s)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        *s = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
    __syncthreads();
    return *s != 0;
}

// zero n accumulator words, shared out over every workgroup of the grid (x
// and y): each one must call it, including those with no other work
template <typename Acc>
__device__ __forceinline__ void zero_share(void* p, int n, int nt)
{
    if (!p || n <= 0) return;
    const int nb = gridDim.x * gridDim.y;
    const int b = blockIdx.y * gridDim.x + blockIdx.x;
    const int per = (n + nb - 1) / nb;
    const int e = min(n, (b + 1) * per);
    Acc* q = reinterpret_cast<Acc*>(p);
    for (int i = b * per + (int)threadIdx.x; i < e; i += nt) q[i] = (Acc)0;
}

}  // namespace iam
