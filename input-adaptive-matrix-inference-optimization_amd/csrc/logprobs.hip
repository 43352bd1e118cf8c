// Log probabilities of given tokens, the entropy of their distribution and the
// likeliest alternatives, in one pass over the logits.
//
// With m the row's maximum, z = sum e^(x - m) and s = sum e^(x - m) (x - m):
//   log p(t) = x_t - m - log z,   entropy = log z - s / z.
#include "accum.h"
#include "numbers.h"
#include "wave.h"

namespace iam {

constexpr int kLpThreads = 256, kLpWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f;

struct LogprobArgs {
    const void* x;
    const int* targets;
    float* lp;
    float* entropy;       // may be null
    int* ids;             // [rows][k], may be null
    float* top;           // [rows][k], may be null
    int rows, vocab, k;
    size_t stride;
    int segs;             // workgroups per row
    int per;              // values of a segment (a multiple of a chunk)
    double* part;         // segs > 1: [rows][segs][3 + k]
    uint32_t* ctr;        // segs > 1: [rows] arrivals, zero on entry (left zero)
};

// Alternatives are ordered by whole numbers: the value's bits made monotone
// (NaN lowest, -0 as 0), then the lower token first.  0 is nothing.
__device__ __forceinline__ uint64_t key_of(float x, int id)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t o = x != x ? 0u : (b >> 31) ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k)
{
    const uint32_t o = (uint32_t)(k >> 32);
    return o == 0u ? NAN : __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

// ---- the best k of a row's (or segment's) values
// The k-th largest of the threads' maxima bounds the k-th largest value from
// below, and few threads reach it, most of them in one chunk alone: only those
// values are looked at again, so that the pass over the logits itself needs no
// exchange.
constexpr int kLpCap = 1024;    // keys held at a time

struct Top {
    uint64_t* keys;     // LDS [kLpCap]
    uint64_t* own;      // LDS [kLpThreads]: the threads' maxima
    int* n;             // LDS [3]: keys there (may pass kLpCap: then only the first are); threads looked at
};

// how many of the 256 keys of own[] are larger than y
__device__ __forceinline__ int larger(const uint64_t* own, uint64_t y)
{
    int r = 0;
#pragma unroll 16
    for (int i = 0; i < kLpThreads; i++) r += own[i] > y;
    return r;
}

// Orders the n <= kLpCap keys of t.keys (distinct, but for places that hold 0:
// nothing); the best min(k, n) end up in order in front.  Where there are many, the k-th best of the threads' best
// keys first thins them out.
__device__ __forceinline__ void lp_order(const Top& t, int n, int k)
{
    const int tid = threadIdx.x;
    constexpr int U = kLpCap / kLpThreads;
    uint64_t mine[U];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++) mine[u] = tid + u * kLpThreads < n ? t.keys[tid + u * kLpThreads] : 0;
    if (n > kLpThreads) {
        uint64_t b = 0;
#pragma unroll
        for (int u = 0; u < U; u++) b = mine[u] > b ? mine[u] : b;
        t.own[tid] = b;
        __syncthreads();
        const int r = larger(t.own, b);
        __syncthreads();
        // the keys of the k threads with the largest ones go on, a place each
        // (0: none)
        if (r < k) {
#pragma unroll
            for (int u = 0; u < U; u++) t.keys[r * U + u] = mine[u];
        }
        n = min(k, kLpThreads) * U;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++) mine[u] = tid + u * kLpThreads < n ? t.keys[tid + u * kLpThreads] : 0;
        __syncthreads();
    }
    int rank[U];
#pragma unroll
    for (int u = 0; u < U; u++) rank[u] = 0;
    if (n <= kLpThreads) {
#pragma unroll 8
        for (int i = 0; i < n; i++) rank[0] += t.keys[i] > mine[0];
    } else {
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const uint64_t y = t.keys[i];
#pragma unroll
            for (int u = 0; u < U; u++) rank[u] += y > mine[u];
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++)
        if (mine[u] != 0 && rank[u] < k) t.keys[rank[u]] = mine[u];
    __syncthreads();
}

// How far the maximum m lies below M, at most 200 (e^-200 is 0 in fp32): two
// finite ones can be farther apart than the largest number, and the factor 0
// times that infinity would be NaN.
__device__ __forceinline__ float lp_below(float m, float M)
{
    const float d = m - M;
    return d < -200.0f ? -200.0f : d;
}

// (m, z, s) of all threads from each one's, in every thread: a wave's first,
// then those of the four (sums to m0 become sums to M: e^(m0 - M) times z, and
// times s + (m0 - M) z)
struct Sums {
    float m;
    double z, s;

    __device__ __forceinline__ void raise(float M)
    {
        const float d = m == -INFINITY ? 0.0f : lp_below(m, M);
        const double f = m == -INFINITY ? (z != z ? NAN : 0.0) : (double)__builtin_amdgcn_exp2f(d * kLog2e);
        s = f * (s + (double)d * z);
        z = f * z;
        m = M;
    }
};
__device__ __forceinline__ void lp_join(float& m, double& z, double& s, Sums* red)
{
    Sums x{m, z, s};
    x.raise(wave_max(m));
    x.z = wave_sum(x.z);
    x.s = wave_sum(x.s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    m = red[0].m;
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) m = fmaxf(m, red[w].m);
    z = s = 0.0;
#pragma unroll
    for (int w = 0; w < kLpWaves; w++) {
        Sums y = red[w];
        y.raise(m);
        z += y.z;
        s += y.s;
    }
}

// VEC values from place i on; outside [v0, v1), -inf
template <typename T, int VEC>
__device__ __forceinline__ void lp_load(const T* x, int i, int v0, int v1, float* v)
{
    if (i >= v0 && i + VEC <= v1) {
        const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(x + i);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = to_f32(r.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = i + e >= v0 && i + e < v1 ? to_f32(x[i + e]) : -INFINITY;
    }
}

// The values of [v0, v1) that take(value) says, as keys behind the n there, of
// n1 threads in one chunk (from the front of `hot`: thread and chunk) and of n2
// threads in all of them (from its back); t.n counts them all.  The first load
// is at place o, a chunk has J for a thread.
template <typename T, int VEC, int J, typename Take>
__device__ __forceinline__ void lp_gather(const Top& t, const T* x, int o, int v0, int v1, const int* hot, int n1, int n2, Take take)
{
    constexpr int B = 4;   // loads in flight
    const int rounds = (v1 - o + kLpThreads * VEC - 1) / (kLpThreads * VEC), one = n1 * J, all = one + rounds * n2;
#pragma unroll 1
    for (int i0 = 0; i0 < all; i0 += B * kLpThreads) {
        float v[B][VEC];
        int at[B];
#pragma unroll
        for (int u = 0; u < B; u++) {
            const int q = i0 + u * kLpThreads + (int)threadIdx.x;
            int r, h;
            if (q < one) {
                h = hot[q / J];
                r = (h >> 8) * J + q % J;
                h &= 255;
            } else {
                r = (q - one) / max(n2, 1);
                h = q < all ? hot[kLpThreads - 1 - (q - one - r * n2)] : 0;
            }
            at[u] = q < all ? o + (r * kLpThreads + h) * VEC : v1;
            lp_load<T, VEC>(x, at[u], v0, v1, v[u]);
        }
        if (*(volatile int*)t.n > kLpCap) continue;   // too many already
#pragma unroll
        for (int u = 0; u < B; u++) {
            int c = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) c += at[u] + e >= v0 && at[u] + e < v1 && take(v[u][e]);
            if (!c) continue;
            int p = atomicAdd(t.n, c);
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (at[u] + e >= v0 && at[u] + e < v1 && take(v[u][e])) {
                    if (p < kLpCap) t.keys[p] = key_of(v[u][e], at[u] + e);
                    p++;
                }
        }
    }
    __syncthreads();
}

// The first `want` values of [v0, v1), by place, that take(value) says, as keys
// behind the n there; how many there were
template <typename T, int VEC, typename Take>
__device__ __forceinline__ int lp_first(const Top& t, const T* x, int o, int v0, int v1, int n, int want, Take take)
{
    __shared__ int wsum[kLpWaves];
    int got = 0;
    for (int c0 = o; c0 < v1 && got < want; c0 += kLpThreads * VEC) {
        const int i = c0 + (int)threadIdx.x * VEC;
        float v[VEC];
        lp_load<T, VEC>(x, i, v0, v1, v);
        int c = 0;
#pragma unroll
        for (int e = 0; e < VEC; e++) c += i + e >= v0 && i + e < v1 && take(v[e]);
        const int incl = wave_incl_sum(c), w = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 63) wsum[w] = incl;
        __syncthreads();
        int at = got + incl - c, all = 0;
#pragma unroll
        for (int u = 0; u < kLpWaves; u++) {
            at += u < w ? wsum[u] : 0;
            all += wsum[u];
        }
#pragma unroll
        for (int e = 0; e < VEC; e++)
            if (i + e >= v0 && i + e < v1 && take(v[e])) {
                if (at < want) t.keys[n + at] = key_of(v[e], i + e);
                at++;
            }
        got += all;
    }
    __syncthreads();
    return min(got, want);
}

// The thread's largest value of the segment, in which chunk that is, and the
// largest one of its other chunks.
struct Most {
    float m = -INFINITY, other = -INFINITY;
    int chunk = 0;

    __device__ __forceinline__ void add(float g, int c)
    {
        other = fmaxf(other, fminf(m, g));
        chunk = g > m ? c : chunk;
        m = fmaxf(m, g);
    }
};

// The best min(k, v1 - v0) keys of [v0, v1) in order in front of t.keys; most:
// of the thread's own loads (from place o on, its part of every 256 * VEC).
// kept: the thread's E values, where the segment is one chunk (`whole`):
// nothing is read again.
template <typename T, int VEC, int E, bool KEEP>
__device__ __forceinline__ int lp_top(const Top& t, int* hot, const T* x, int o, int v0, int v1, const Most& most, int k,
                                      bool whole, const float* kept)
{
    const int tid = threadIdx.x, have = min(k, v1 - v0);
    float* lane_max = reinterpret_cast<float*>(t.own);   // [kLpWaves][64]
    const float m = most.m;
    __syncthreads();
    lane_max[tid] = m;
    if (tid < 3) t.n[tid] = 0;
    __syncthreads();
    // In each wave bit by bit, the largest number that k of the maxima reach: of
    // 64 (each of four threads), or of all 256 where 64 would bound little (1024
    // x 128001 bf16 with 64 alternatives 70 us, else 126; with 20 64 and 63).
    uint32_t mine[kLpWaves];
#pragma unroll
    for (int w = 0; w < kLpWaves; w++) mine[w] = (uint32_t)(key_of(lane_max[w * 64 + (tid & 63)], 0) >> 32);
    uint32_t kth = 0;
    if (k <= 32) {
        uint32_t g = mine[0];
#pragma unroll
        for (int w = 1; w < kLpWaves; w++) g = max(g, mine[w]);
#pragma unroll
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t y = kth | 1u << bit;
            if (__popcll(__ballot(g >= y)) >= k) kth = y;
        }
    } else {
#pragma unroll 1
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t y = kth | 1u << bit;
            int c = 0;
#pragma unroll
            for (int w = 0; w < kLpWaves; w++) c += __popcll(__ballot(mine[w] >= y));
            if (c >= k) kth = y;
        }
    }
    const float b = key_value((uint64_t)kth << 32);
    if (most.other >= b) hot[kLpThreads - 1 - atomicAdd(t.n + 2, 1)] = tid;
    else if (m >= b) hot[atomicAdd(t.n + 1, 1)] = tid | most.chunk << 8;
    __syncthreads();
    const int n1 = t.n[1], n2 = t.n[2];
    if (KEEP && whole) {
        if (m >= b) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int i = o + (e / VEC * kLpThreads + tid) * VEC + e % VEC;
                if (kept[e] >= b && i >= v0 && i < v1) {
                    const int p = atomicAdd(t.n, 1);
                    if (p < kLpCap) t.keys[p] = key_of(kept[e], i);
                }
            }
        }
        __syncthreads();
    } else {
        lp_gather<T, VEC, E / VEC>(t, x, o, v0, v1, hot, n1, n2, [&](float v) { return v >= b; });
    }
    int n = t.n[0];
    const bool many = n > kLpCap;
    if (many) {
        // many equal values (a masked row's -inf): the larger ones, then the
        // first of the equal ones
        __syncthreads();
        if (tid == 0) t.n[0] = 0;
        __syncthreads();
        lp_gather<T, VEC, E / VEC>(t, x, o, v0, v1, hot, n1, n2, [&](float v) { return v > b; });
        n = t.n[0];
        __syncthreads();
        if (n > kLpCap) {
            // few threads hold very many of the largest (no order of a
            // vocabulary does that by itself): one at a time
            uint64_t last = ~0ull;
            for (n = 0; n < have; n++) {
                uint64_t best = 0;
#pragma unroll 1
                for (int i = v0 + tid; i < v1; i += kLpThreads) {
                    const uint64_t y = key_of(to_f32(x[i]), i);
                    best = y < last && y > best ? y : best;
                }
                __syncthreads();
                t.own[tid] = best;
                __syncthreads();
#pragma unroll 4
                for (int i = 0; i < kLpThreads; i++) best = t.own[i] > best ? t.own[i] : best;
                last = best;
                if (tid == 0) t.keys[n] = best;
            }
            __syncthreads();
            return have;
        }
    }
    // what is missing: the first that equal b, then the first NaN
#pragma unroll 1
    for (int nan = 0; nan < 2 && n < have; nan++)
        if (nan || many) n += lp_first<T, VEC>(t, x, o, v0, v1, n, have - n, [&](float v) { return nan ? v != v : v == b; });
    lp_order(t, n, k);
    return have;
}

// A workgroup takes one segment of a row, in chunks of 256 * E values that
// stay in registers: E of them a thread, by 16-byte loads issued together.
// Each wave has its own running maximum M (the factors of its sums change
// where a chunk raises it, seldom).  z's terms are added in fp32 within a
// chunk, without their whole part, which only values next to M have (it is
// counted apart), then in fp64: log z keeps its digits where one token has
// nearly all the probability, and no term costs fp64 instructions.  Bound by
// the reads in fp32; in 16 bits the arithmetic of a value (13 issue slots, 4
// of them its exponential) is about as long as its read.
template <typename T, int E, bool TOP>
__global__ __launch_bounds__(kLpThreads) void k_token_logprobs(LogprobArgs a)
{
    constexpr int VEC = 16 / (int)sizeof(T), J = E / VEC, CHUNK = kLpThreads * E;
    __shared__ uint64_t keys[TOP ? kLpCap : 1], own[TOP ? kLpThreads : 1];
    __shared__ int hot[TOP ? kLpThreads : 1], counts[3];
    __shared__ int s_last;
    __shared__ Sums red[kLpWaves];
    const int tid = threadIdx.x;
    const int row = a.segs == 1 ? blockIdx.x : blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.stride;
    // Chunks start at multiples of 16 bytes in memory, before the row's (or
    // segment's) first value if need be: rows at 2-byte boundaries, read as
    // they lie, took 9 us more (1024 x 128001 bf16, 54 us this way).
    const int off = (int)((uintptr_t)x / sizeof(T) % VEC);
    const int o = seg * a.per - off, v0 = max(o, 0), v1 = a.vocab - o > a.per ? o + a.per : a.vocab;
    float M = -INFINITY;            // the wave's
    Most most;                      // the thread's
    double z = 0.0, s = 0.0;        // the thread's, without the `ones` terms that are 1
    int ones = 0;
    float v[E];
    for (int c0 = o; c0 < v1; c0 += CHUNK) {
        if (c0 >= v0 && c0 + CHUNK <= v1) {
            typedef Pack<T, VEC> Run;
            Run r[J];
#pragma unroll
            for (int j = 0; j < J; j++) r[j] = *reinterpret_cast<const Run*>(x + c0 + (j * kLpThreads + tid) * VEC);
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < VEC; e++) v[j * VEC + e] = to_f32(r[j].v[e]);
        } else {
#pragma unroll
            for (int j = 0; j < J; j++) lp_load<T, VEC>(x, c0 + (j * kLpThreads + tid) * VEC, v0, v1, v + j * VEC);
        }
        float g = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e++) g = fmaxf(g, v[e]);
        if constexpr (TOP) most.add(g, (c0 - o) / CHUNK);
        const float gw = wave_max(g);
        if (gw > M) {
            const float d = M == -INFINITY ? 0.0f : lp_below(M, gw);
            const double f = (double)__builtin_amdgcn_exp2f(d * kLog2e);
            z += (double)ones;
            s = f * (s + (double)d * z);
            z = f * z;
            ones = 0;
            M = gw;
        }
        const float base = M == -INFINITY ? 0.0f : M;
        float zc = 0.0f, sc = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float d = v[e] - base;
            const float p = __builtin_amdgcn_exp2f(d * kLog2e);
            zc += __builtin_amdgcn_fractf(p);
            sc = __builtin_fmaf(p, __builtin_amdgcn_fmed3f(d, -200.0f, 0.0f), sc);   // p is 0 below
        }
        if (__builtin_amdgcn_exp2f((gw - base) * kLog2e) == 1.0f) {
#pragma unroll
            for (int e = 0; e < E; e++) ones += __builtin_amdgcn_exp2f((v[e] - base) * kLog2e) == 1.0f;
        }
        z += (double)zc;
        s += (double)sc;
    }
    float m = M;
    z += (double)ones;
    int have = 0;
    const Top top{keys, own, counts};
    if constexpr (TOP) have = lp_top<T, VEC, E, E == 8>(top, hot, x, o, v0, v1, most, a.k, v1 - o <= CHUNK, v);
    lp_join(m, z, s, red);
    if (a.segs > 1) {
        const int words = 3 + a.k;
        double* mine = a.part + ((size_t)row * a.segs + seg) * words;
        if (tid == 0) {
            acc_put(mine, (double)m);
            acc_put(mine + 1, z);
            acc_put(mine + 2, s);
        }
        if constexpr (TOP)
            for (int i = tid; i < a.k; i += kLpThreads)
                acc_put(reinterpret_cast<unsigned long long*>(mine) + 3 + i, i < have ? keys[i] : 0);
        if (!acc_arrive(a.ctr + row, (uint32_t)a.segs, &s_last)) return;
        double* parts = a.part + (size_t)row * a.segs * words;
        m = -INFINITY;
        z = s = 0.0;
        if (tid < a.segs) {
            m = (float)acc_peek(parts + tid * words);
            z = acc_peek(parts + tid * words + 1);
            s = acc_peek(parts + tid * words + 2);
        }
        if constexpr (TOP) {
            // segs * k <= kLpCap; missing keys (of short segments) are 0
            uint64_t y[kLpCap / kLpThreads];
#pragma unroll
            for (int u = 0; u < kLpCap / kLpThreads; u++) {
                const int i = u * kLpThreads + tid;
                y[u] = i < a.segs * a.k
                           ? acc_peek(reinterpret_cast<unsigned long long*>(parts) + (size_t)(i / a.k) * words + 3 + i % a.k)
                           : 0;
            }
#pragma unroll
            for (int u = 0; u < kLpCap / kLpThreads; u++)
                if (u * kLpThreads + tid < a.segs * a.k) keys[u * kLpThreads + tid] = y[u];
            lp_order(top, a.segs * a.k, a.k);
        }
        lp_join(m, z, s, red);
        if (tid == 0) a.ctr[row] = 0u;
    }
    const bool none = m == -INFINITY && z == 0.0;   // nothing but -inf
    const double lz = log(z);
    if (tid == 0) {
        const int t = a.targets[row];
        float r = 0.0f;
        if (t >= 0 && t < a.vocab) {
            const float xt = to_f32(x[t]);
            r = none ? -INFINITY : (float)((double)xt - (double)m - lz);
        }
        a.lp[row] = r;
        if (a.entropy) {
            const double h = none ? 0.0 : lz - s / z;
            a.entropy[row] = h < 0.0 ? 0.0f : (float)h;
        }
    }
    if constexpr (TOP)
        for (int i = tid; i < a.k; i += kLpThreads) {
            const uint64_t y = keys[i];
            const float v = key_value(y);
            if (a.ids) a.ids[(size_t)row * a.k + i] = key_id(y);
            if (a.top) a.top[(size_t)row * a.k + i] = none ? -INFINITY : (float)((double)v - (double)m - lz);
        }
}

// ------------------------------------------------------------------ host ---
// workgroups that the rows are cut into segments for: 4 on each of 256 CUs (389
// x 32000 fp32 15 us, 1024 x 128001 bf16 54; with 8 on each 16 and 62: a row's
// join costs about as much as a segment)
constexpr int kLpTarget = 1024;
constexpr int kLpMaxSegs = 64;
constexpr int kLpSlice = 1 << 22;  // rows of a launch (of 2^32 threads at most)

template <typename T, int E>
static int logprobs_launch(Ctx* c, LogprobArgs a)
{
    constexpr int CHUNK = kLpThreads * E;
    // values before a row's first that its first chunk holds, at most
    constexpr int VEC = 16 / (int)sizeof(T);
    const int off = a.rows == 1 || a.stride % VEC == 0 ? (int)((uintptr_t)a.x / sizeof(T) % VEC) : VEC - 1;
    const int chunks = (int)(((int64_t)a.vocab + off + CHUNK - 1) / CHUNK);
    // A row's segments' keys are ordered together, quickest up to 256 of them
    // (64 x 32000 with 20 alternatives 15.7 us, with 320 keys 20.4), unless
    // segments would be long (1 x 1000000 with 20: 31 us, with 1020 keys 19).
    const int keys = (int64_t)chunks * a.k <= 8 * kLpThreads ? kLpThreads : kLpCap;
    const int most = a.k ? std::min(kLpMaxSegs, keys / a.k) : kLpMaxSegs;
    const int want = std::max(1, std::min({chunks, most, kLpTarget / std::max(a.rows, 1)}));
    const int each = (chunks + want - 1) / want;
    a.segs = (chunks + each - 1) / each;
    a.per = (int)std::min<int64_t>((int64_t)each * CHUNK, 0x7fffffff);
    if (a.segs > 1) {
        IAM_TRY(ensure_lp_scratch(c, (size_t)a.rows * a.segs * (3 + a.k), (size_t)a.rows));
        a.part = c->lp_part;
        a.ctr = c->lp_ctr;
    }
    const dim3 grid((unsigned)(a.rows * a.segs));
    return a.k ? launch(c, "token_logprobs", k_token_logprobs<T, E, true>, grid, dim3(kLpThreads), 0, a)
               : launch(c, "token_logprobs", k_token_logprobs<T, E, false>, grid, dim3(kLpThreads), 0, a);
}

template <typename T>
static int logprobs_typed(Ctx* c, LogprobArgs a)
{
    for (int left = a.rows; left > 0; left -= kLpSlice) {
        a.rows = std::min(left, kLpSlice);
        // Smaller chunks for few values in all, so that more workgroups share
        // them, and where large ones would be empty by a quarter of a row or
        // more (1500 rows of 2425 bf16 with 1 alternative 16 us, with large
        // chunks 21; of 12000 21 and 24; of 24000 29 and 28).
        const int64_t large = (int64_t)kLpThreads * 32, empty = (a.vocab + large - 1) / large * large - a.vocab;
        if (a.rows * (int64_t)a.vocab <= 256 * large || 4 * empty > a.vocab) IAM_TRY((logprobs_launch<T, 8>(c, a)));
        else IAM_TRY((logprobs_launch<T, 32>(c, a)));
        a.x = reinterpret_cast<const T*>(a.x) + a.rows * a.stride;
        a.targets += a.rows;
        a.lp += a.rows;
        if (a.entropy) a.entropy += a.rows;
        if (a.ids) a.ids += (size_t)a.rows * a.k;
        if (a.top) a.top += (size_t)a.rows * a.k;
    }
    return IAM_OK;
}

}  // namespace iam

using namespace iam;

extern "C" int iam_token_logprobs(iam_ctx* c, const void* x, int type, int rows, int vocab, size_t stride,
                                  const int* targets, float* lp, float* entropy, int k, int* ids, float* top)
{
    if (!c || !x || !targets || !lp) return fail(IAM_E_INVALID, "token_logprobs: null argument");
    IAM_REQUIRE(type == IAM_F32 || type == IAM_F16 || type == IAM_BF16, "token_logprobs: unknown type");
    IAM_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= (1 << 30), "token_logprobs: n_rows must not be negative, vocab 1 to 2^30");
    IAM_REQUIRE(k >= 0 && k <= IAM_LOGPROBS_MAX_TOP && k <= vocab, "token_logprobs: top_k must be 0 to min(vocab, 64)");
    if (!ids && !top) k = 0;
    const size_t B = type_bytes(type);
    if (!stride) stride = (size_t)vocab;
    IAM_REQUIRE(stride >= (size_t)vocab && stride < ((size_t)1 << 40), "token_logprobs: the stride is smaller than a row");
    IAM_REQUIRE(aligned(x, B) && aligned(targets, 4) && aligned(lp, 4) && aligned(entropy, 4) && aligned(ids, 4) && aligned(top, 4),
                "token_logprobs: pointers must be aligned to their type");
    if (rows == 0) return IAM_OK;
    const size_t n = (size_t)rows, xb = rows_bytes(n, (size_t)vocab, stride, B);
    struct {
        const void* p;
        size_t bytes;
        const char* what;
    } const part[] = {{lp, n * 4, "token_logprobs logprob"},          {entropy, n * 4, "token_logprobs entropy"},
                      {k ? ids : nullptr, n * k * 4, "token_logprobs ids"}, {k ? top : nullptr, n * k * 4, "token_logprobs top"},
                      {targets, n * 4, "token_logprobs targets"},     {x, xb, "token_logprobs logits"}};
    for (int i = 0; i < 6; i++) {
        if (!part[i].p) continue;
        IAM_TRY(check_dev_range(c, part[i].p, part[i].bytes, part[i].what));
        for (int j = 0; j < i && j < 4; j++)
            IAM_REQUIRE(!part[j].p || !overlaps(part[i].p, part[i].bytes, part[j].p, part[j].bytes),
                        "token_logprobs: an output overlaps another array");
    }
    DeviceGuard on(c);
    LogprobArgs a{};
    a.x = x;
    a.targets = targets;
    a.lp = lp;
    a.entropy = entropy;
    a.ids = ids;
    a.top = top;
    a.rows = rows;
    a.vocab = vocab;
    a.k = k;
    a.stride = stride;
    if (type == IAM_F32) return logprobs_typed<float>(c, a);
    if (type == IAM_F16) return logprobs_typed<_Float16>(c, a);
    return logprobs_typed<__bf16>(c, a);
}
