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

// The best k keys offered so far by the workgroup's threads.  `keys` holds at
// most cap = 33 k of them; `floor` is a key that k others are known to reach:
// lower ones are not taken.  A thread offers N keys at a time.  Too many at
// once (as in a row's first chunk): the k-th best of the threads' own best
// keys becomes the floor, which leaves at most k threads with N <= 32 keys each.
struct Best {
    uint64_t* keys;       // LDS [cap]
    uint64_t* own;        // LDS [kLpThreads]
    uint64_t* floor_p;    // LDS
    int* count;           // LDS
    int k, cap;
    int have = 0;         // uniform
    uint64_t floor = 0;   // uniform: keys above it are taken

    __device__ __forceinline__ void start()
    {
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
    }
    // keeps the best k, in order
    __device__ void prune()
    {
        uint64_t mine[9];
        int rank[9];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 9; u++) {
            const int i = (int)threadIdx.x + u * kLpThreads;
            mine[u] = i < have ? keys[i] : 0;
            rank[u] = 0;
        }
        for (int j = 0; j < have; j++) {
            const uint64_t y = keys[j];
#pragma unroll
            for (int u = 0; u < 9; u++) rank[u] += y > mine[u];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 9; u++)
            if (mine[u] != 0 && rank[u] < k) keys[rank[u]] = mine[u];
        have = min(have, k);
        if (threadIdx.x == 0) *count = have;
        __syncthreads();
        if (have == k && keys[k - 1] > floor) floor = keys[k - 1];
    }
    template <int N, typename Key>
    __device__ void offer(Key key, bool hot)
    {
        if (!__syncthreads_or(hot)) return;
        int c = 0;
#pragma unroll
        for (int e = 0; e < N; e++) c += hot && key(e) > floor;
        int at = c ? atomicAdd(count, c) : 0;
        __syncthreads();
        int total = *count;
        if (total > cap) {
            __syncthreads();
            prune();      // also takes back the count
            uint64_t b = 0;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const uint64_t y = hot ? key(e) : 0;
                b = y > b ? y : b;
            }
            own[threadIdx.x] = b;
            if (threadIdx.x == 0) *floor_p = 0;
            __syncthreads();
            int rank = 0;
            for (int j = 0; j < kLpThreads; j++) rank += own[j] > b;
            if (b != 0 && rank == k - 1) *floor_p = b - 1;
            __syncthreads();
            if (*floor_p > floor) floor = *floor_p;
            c = 0;
#pragma unroll
            for (int e = 0; e < N; e++) c += hot && key(e) > floor;
            at = c ? atomicAdd(count, c) : 0;
            __syncthreads();
            total = *count;
        }
        if (c) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const uint64_t y = key(e);
                if (y > floor && at < cap) keys[at++] = y;
            }
        }
        have = min(total, cap);
        __syncthreads();
        if (have > 3 * k + 32) prune();
    }
};

__device__ __forceinline__ double lp_sum(double v, double* red)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = red[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) t += red[w];
    return t;
}

__device__ __forceinline__ float lp_max(float v, float* red)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) t = fmaxf(t, red[w]);
    return t;
}

// (m, z, s) of all threads from each one's, in every thread
__device__ __forceinline__ void lp_join(float& m, double& z, double& s, float* redf, double* redd)
{
    const float M = lp_max(m, redf);
    const float d = m == -INFINITY ? 0.0f : m - M;
    const double f = m == -INFINITY ? (z != z ? NAN : 0.0) : (double)__builtin_amdgcn_exp2f(d * kLog2e);
    s = lp_sum(f * (s + (double)d * z), redd);
    z = lp_sum(f * z, redd);
    m = M;
}

// A workgroup takes one segment of a row, in chunks of 256 * E values that
// stay in registers: E of them a thread, by 16-byte loads issued together.
// Each thread keeps its own running maximum (the factors of its sums change
// at most once a chunk), terms of z are added in fp64 (so that log z keeps
// its digits where one token has nearly all the probability), those of s in
// fp32 within a chunk; the threads' sums meet at the row's end.  Bound by the
// reads where rows are many.
template <typename T, int E, bool TOP>
__global__ __launch_bounds__(kLpThreads) void k_token_logprobs(LogprobArgs a)
{
    constexpr int VEC = 16 / (int)sizeof(T), J = E / VEC, CHUNK = kLpThreads * E;
    extern __shared__ uint64_t cand[];
    __shared__ uint64_t own[TOP ? kLpThreads : 1];
    __shared__ uint64_t floor_s;
    __shared__ int count_s, s_last;
    __shared__ double redd[kLpWaves];
    __shared__ float redf[kLpWaves];
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.stride;
    const int v0 = seg * a.per, v1 = a.vocab - v0 > a.per ? v0 + a.per : a.vocab;
    float m = -INFINITY;
    double z = 0.0, s = 0.0;
    Best best{cand, own, &floor_s, &count_s, a.k, 33 * a.k};
    if constexpr (TOP) best.start();
    for (int c0 = v0; c0 < v1; c0 += CHUNK) {
        float v[E];
        const bool inside = c0 + CHUNK <= v1;
        if (inside) {
            typedef Pack<T, VEC, (int)sizeof(T)> Run;
            Run r[J];
#pragma unroll
            for (int j = 0; j < J; j++) r[j] = *reinterpret_cast<const Run*>(x + c0 + (j * kLpThreads + tid) * VEC);
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < VEC; e++) v[j * VEC + e] = to_f32(r[j].v[e]);
        } else {
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int i = (j * kLpThreads + tid) * VEC + e;
                    v[j * VEC + e] = i < v1 - c0 ? to_f32(x[c0 + i]) : -INFINITY;
                }
        }
        float g = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e++) g = fmaxf(g, v[e]);
        if (g > m) {
            const float d = m == -INFINITY ? 0.0f : m - g;
            const double f = (double)__builtin_amdgcn_exp2f(d * kLog2e);
            s = f * (s + (double)d * z);
            z = f * z;
            m = g;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sc = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float d = v[e] - base;
            const float p = __builtin_amdgcn_exp2f(d * kLog2e);
            z += (double)p;
            sc = __builtin_fmaf(p, fmaxf(d, -200.0f), sc);   // p is 0 below
        }
        s += (double)sc;
        if constexpr (TOP) {
            auto key = [&](int e) __attribute__((always_inline)) {
                const int i = ((e / VEC) * kLpThreads + tid) * VEC + e % VEC;
                return inside || i < v1 - c0 ? key_of(v[e], c0 + i) : 0ull;
            };
            // below the floor's value none of the thread's keys is taken
            best.template offer<E>(key, best.floor < (1ull << 32) || g >= key_value(best.floor));
        }
    }
    if constexpr (TOP) best.prune();
    lp_join(m, z, s, redf, redd);
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
                acc_put(reinterpret_cast<unsigned long long*>(mine) + 3 + i, i < best.have ? best.keys[i] : 0);
        if (!acc_arrive(a.ctr + row, (uint32_t)a.segs, &s_last)) return;
        double* parts = a.part + (size_t)row * a.segs * words;
        m = -INFINITY;
        z = s = 0.0;
        if (tid < a.segs) {
            m = (float)acc_peek(parts + tid * words);
            z = acc_peek(parts + tid * words + 1);
            s = acc_peek(parts + tid * words + 2);
        }
        lp_join(m, z, s, redf, redd);
        if constexpr (TOP) {
            best.have = 0;
            best.floor = 0;
            best.start();
            constexpr int N = 8;
            for (int i0 = 0; i0 < a.segs * a.k; i0 += N * kLpThreads) {
                uint64_t y[N];
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int i = i0 + e * kLpThreads + tid;
                    y[e] = i < a.segs * a.k
                               ? acc_peek(reinterpret_cast<unsigned long long*>(parts) + (size_t)(i / a.k) * words + 3 + i % a.k)
                               : 0;
                }
                best.template offer<N>([&](int e) __attribute__((always_inline)) { return y[e]; }, true);
            }
            best.prune();
        }
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
            const uint64_t y = best.keys[i];
            const float v = key_value(y);
            if (a.ids) a.ids[(size_t)row * a.k + i] = key_id(y);
            if (a.top) a.top[(size_t)row * a.k + i] = none ? -INFINITY : (float)((double)v - (double)m - lz);
        }
}

// ------------------------------------------------------------------ host ---
constexpr int kLpTarget = 2048;    // workgroups that fill the card: 8 on each of 256 CUs
constexpr int kLpMaxSegs = 64;

template <typename T, int E>
static int logprobs_launch(Ctx* c, LogprobArgs a)
{
    constexpr int CHUNK = kLpThreads * E;
    const int chunks = (int)(((int64_t)a.vocab + CHUNK - 1) / CHUNK);
    const int want = std::max(1, std::min({chunks, kLpMaxSegs, kLpTarget / std::max(a.rows, 1)}));
    const int each = (chunks + want - 1) / want;
    a.segs = (chunks + each - 1) / each;
    a.per = (int)std::min<int64_t>((int64_t)each * CHUNK, 0x7fffffff);
    if (a.segs > 1) {
        IAM_TRY(ensure_lp_scratch(c, (size_t)a.rows * a.segs * (3 + a.k), (size_t)a.rows));
        a.part = c->lp_part;
        a.ctr = c->lp_ctr;
    }
    IAM_REQUIRE((int64_t)a.rows * a.segs < ((int64_t)1 << 31), "token_logprobs: too many rows");
    const dim3 grid((unsigned)(a.rows * a.segs));
    return a.k ? launch(c, "token_logprobs", k_token_logprobs<T, E, true>, grid, dim3(kLpThreads), (size_t)33 * a.k * 8, a)
               : launch(c, "token_logprobs", k_token_logprobs<T, E, false>, grid, dim3(kLpThreads), 0, a);
}

template <typename T>
static int logprobs_typed(Ctx* c, const LogprobArgs& a)
{
    // few values in all: smaller chunks, so that more workgroups share them
    if ((int64_t)a.rows * a.vocab <= (int64_t)256 * kLpThreads * 32) return logprobs_launch<T, 8>(c, a);
    return logprobs_launch<T, 32>(c, a);
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
