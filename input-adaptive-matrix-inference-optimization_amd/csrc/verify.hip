// Verification of drafted tokens by the target's probabilities from given random
// numbers.
//
// With p and q the target's and the draft's probabilities of a place and u its
// random number, the token t drafted from q is kept if u q(t) < p(t); the first
// one that is not is replaced by one drawn from max(p - q, 0), so that what
// comes out is distributed as p.  Both are decided in fp64 from the logits on:
// at a vocabulary of 10^5 tokens, 10^-7 of the sum is a tenth of a token's
// share, and errors of that size would pick neighbours.
#include "accum.h"
#include "numbers.h"
#include "wave.h"

namespace iam {

constexpr int kVerThreads = 256, kVerWaves = 4;
constexpr int kVerMaxSegs = 64;

// One kind of rows of logits (the target's, or the draft's)
struct Rows {
    const void* x;
    size_t stride;
    int type;
    double unit;             // 1 / temperature in the exponential's units
};

struct VerifyArgs {
    Rows target, draft;      // draft.x may be null
    int seqs, n, vocab;
    int segs, per;           // segments of a row, and their values (a multiple of a chunk)
    const int* tokens;
    const int* count;        // may be null
    const float* uniform;
    int* out;
    int* accepted;
    double* stat;            // [seqs (n + 1) + seqs n][segs][2]: largest logit, sum of exponentials; the best key (greedy)
    double* part;            // [seqs][segs]: weights of the segment the last token is drawn from
    uint32_t* ctr;           // [seqs], zero on entry (left zero)
};

// ---- exponentials
// 2^(t / 64) in fp64 for t <= 0: the table's 2^(j / 64) times a polynomial of the
// rest f, |f| <= 1/2 (the series of e^(f ln 2 / 64) up to the fifth power: 4e-17).
constexpr double kUnit = 64.0 * 1.44269504088896340736;   // t of e^1
struct ExpTable {
    double t[64];
};
__device__ __forceinline__ void fill_table(ExpTable* e)
{
    if (threadIdx.x < 64) e->t[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
}
__device__ __forceinline__ double exp_of(const ExpTable* e, double t)
{
    constexpr double u = 1.0 / kUnit;
    const double n = rint(t), f = t - n;
    double p = u * u * u * u * u / 120.0;
    p = __builtin_fma(p, f, u * u * u * u / 24.0);
    p = __builtin_fma(p, f, u * u * u / 6.0);
    p = __builtin_fma(p, f, u * u / 2.0);
    p = __builtin_fma(p, f, u);
    p = __builtin_fma(p, f, 1.0);
    const int i = (int)n;
    return ldexp(p * e->t[i & 63], i >> 6);
}

// What a row's exponentials are taken relative to: its largest logit.
struct Base {
    double unit, m;
    // e^((x - m) / temperature); 0 below 2^-1074, -inf too
    __device__ __forceinline__ double weight(const ExpTable* e, float x) const
    {
        return exp_of(e, fmax(((double)x - m) * unit, -64.0 * 1100.0));
    }
};

// ---- reading a row
// E values a thread of a chunk of 256 E, from place c0 on, runs of 16 bytes:
// value e of the thread is at place_of(c0, e).  Outside [v0, v1), -inf.
template <typename T, int E>
__device__ __forceinline__ void load_chunk(const T* x, int c0, int v0, int v1, float* v)
{
    // the runs of 8 values (of fp32 two loads)
    typedef Pack<T, 8, (int)sizeof(T)> Run;
    Run r[E / 8];
    if (c0 >= v0 && c0 + kVerThreads * E <= v1) {
#pragma unroll
        for (int j = 0; j < E / 8; j++) r[j] = *reinterpret_cast<const Run*>(x + c0 + (j * kVerThreads + (int)threadIdx.x) * 8);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = to_f32(r[e / 8].v[e % 8]);
        return;
    }
#pragma unroll
    for (int j = 0; j < E / 8; j++) {
        const int i = c0 + (j * kVerThreads + (int)threadIdx.x) * 8;
        if (i >= v0 && i + 8 <= v1) {
            const Run q = *reinterpret_cast<const Run*>(x + i);
#pragma unroll
            for (int e = 0; e < 8; e++) v[j * 8 + e] = to_f32(q.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[j * 8 + e] = i + e >= v0 && i + e < v1 ? to_f32(x[i + e]) : -INFINITY;
        }
    }
}
__device__ __forceinline__ int place_of(int c0, int e) { return c0 + (e / 8 * kVerThreads + (int)threadIdx.x) * 8 + e % 8; }

__device__ __forceinline__ size_t value_bytes(int type) { return type == IAM_F32 ? 4 : 2; }
template <int E>
__device__ __forceinline__ void load_chunk(const Rows& r, size_t row, int c0, int v0, int v1, float* v)
{
    if (r.type == IAM_F32) load_chunk<float, E>(reinterpret_cast<const float*>(r.x) + row * r.stride, c0, v0, v1, v);
    else if (r.type == IAM_F16) load_chunk<_Float16, E>(reinterpret_cast<const _Float16*>(r.x) + row * r.stride, c0, v0, v1, v);
    else load_chunk<__bf16, E>(reinterpret_cast<const __bf16*>(r.x) + row * r.stride, c0, v0, v1, v);
}
__device__ __forceinline__ float logit_of(const Rows& r, size_t row, int t)
{
    const size_t at = row * r.stride + t;
    if (r.type == IAM_F32) return reinterpret_cast<const float*>(r.x)[at];
    if (r.type == IAM_F16) return (float)reinterpret_cast<const _Float16*>(r.x)[at];
    return (float)reinterpret_cast<const __bf16*>(r.x)[at];
}

// A segment's values.  Chunks start at multiples of 16 bytes of the row, before
// its first value if need be.
struct Segment {
    int o, v0, v1;
};
__device__ __forceinline__ Segment segment_of(const VerifyArgs& a, const Rows& r, size_t row, int seg)
{
    const size_t bytes = value_bytes(r.type);
    const int off = (int)(((uintptr_t)r.x + row * r.stride * bytes) / bytes % (16 / bytes));
    Segment s;
    s.o = seg * a.per - off;
    s.v0 = max(s.o, 0);
    s.v1 = a.vocab - s.o > a.per ? s.o + a.per : a.vocab;
    return s;
}

// drafted tokens of a sequence
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int s) { return a.count ? min(max(a.count[s], 0), a.n) : a.n; }

// which row a workgroup of the first launch takes; false: one that is not needed
struct Which {
    bool draft;
    size_t row;      // of its kind
    size_t stat;     // its results
    int seg;
};
__device__ __forceinline__ bool which_of(const VerifyArgs& a, int first, Which& w)
{
    const int r = first + blockIdx.x / a.segs, targets = a.seqs * (a.n + 1);
    w.seg = blockIdx.x % a.segs;
    w.stat = ((size_t)r * a.segs + w.seg) * 2;
    w.draft = r >= targets;
    w.row = w.draft ? r - targets : r;
    const int each = w.draft ? a.n : a.n + 1, s = (int)w.row / each, i = (int)w.row - s * each;
    return i < drafts_of(a, s) + (w.draft ? 0 : 1);
}

// The largest logit m of a segment and the sum of e^((x - m) / temperature); NaN
// where there is a NaN or +inf, 0 where there is nothing but -inf.  Each wave
// has its own m.  Bound by the fp64 arithmetic (17 instructions a value).
template <int E>
__global__ __launch_bounds__(kVerThreads) void k_verify_rows(VerifyArgs a, int first)
{
    __shared__ ExpTable table;
    __shared__ float wave_m[kVerWaves];
    __shared__ double wave_z[kVerWaves];
    Which w;
    if (!which_of(a, first, w)) return;
    fill_table(&table);
    __syncthreads();
    const Rows& r = w.draft ? a.draft : a.target;
    const Segment g = segment_of(a, r, w.row, w.seg);
    float m = -INFINITY;
    double z = 0.0;
    bool bad = false;
    for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * E) {
        float v[E];
        load_chunk<E>(r, w.row, c0, g.v0, g.v1, v);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < E; e++) top = __builtin_elementwise_maximum(top, v[e]);
        top = wave_reduce(top, [](float x, float y) { return __builtin_elementwise_maximum(x, y); });
        bad |= !(top < INFINITY);
        if (top == -INFINITY || bad) continue;
        if (top > m) {
            if (m != -INFINITY) z *= exp(((double)m - (double)top) * (r.unit / kUnit));
            m = top;
        }
        const Base b{r.unit, (double)m};
#pragma unroll
        for (int e = 0; e < E; e++) z += b.weight(&table, v[e]);
    }
    z = wave_sum(z);
    if (bad) z = NAN;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        wave_m[wave] = m;
        wave_z[wave] = z;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float top = wave_m[0];
        for (int i = 1; i < kVerWaves; i++) top = fmaxf(top, wave_m[i]);
        double sum = 0.0;
        for (int i = 0; i < kVerWaves; i++)
            if (wave_m[i] != -INFINITY || wave_z[i] != wave_z[i]) sum += wave_m[i] == top ? wave_z[i] : wave_z[i] * exp(((double)wave_m[i] - (double)top) * (r.unit / kUnit));
        a.stat[w.stat] = (double)top;
        a.stat[w.stat + 1] = sum;
    }
}

// A row's largest logit and sum from its segments', in every lane; z is NaN where
// the row has no distribution
struct Joined {
    float m;
    double z;
};
__device__ __forceinline__ Joined join_row(const VerifyArgs& a, size_t r, double unit)
{
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    double z = 0.0;
    if (lane < a.segs) {
        m = (float)a.stat[(r * a.segs + lane) * 2];
        z = a.stat[(r * a.segs + lane) * 2 + 1];
    }
    const float top = wave_max(m);
    const double f = m == -INFINITY ? 0.0 : m == top ? 1.0 : exp(((double)m - (double)top) * (unit / kUnit));
    const double sum = wave_sum(z != z ? z : z * f);
    return {top, top == -INFINITY ? NAN : sum};
}

__device__ __forceinline__ double wave_scan(double v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double u = __shfl_up(v, d);
        v += lane >= d ? u : 0.0;
    }
    return v;
}

// what a token of a sequence is drawn by: p, less q (or the drafted token) where it was rejected
struct Draw {
    bool less;
    size_t row, qrow;
    int gone;                // the drafted token, where q is 1 there
    float pm, qm;
    double pz, qz;           // 1 / sums
};

// the weights of a chunk's values in a thread's registers
template <int E>
__device__ __forceinline__ void weights_of(const VerifyArgs& a, const Draw& d, const ExpTable* table, const Segment& g, int c0, double* w)
{
    float v[E];
    load_chunk<E>(a.target, d.row, c0, g.v0, g.v1, v);
    const Base b{a.target.unit, (double)d.pm};
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = b.weight(table, v[e]) * d.pz;
    if (!d.less) return;
    if (!a.draft.x) {
#pragma unroll
        for (int e = 0; e < E; e++) w[e] = place_of(c0, e) == d.gone ? 0.0 : w[e];
        return;
    }
    load_chunk<E>(a.draft, d.qrow, c0, g.v0, g.v1, v);
    const Base q{a.draft.unit, (double)d.qm};
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = fmax(__builtin_fma(q.weight(table, v[e]), -d.qz, w[e]), 0.0);
}

// Workgroup (sequence, segment): which drafted tokens are kept (every workgroup
// of the sequence finds out by itself), the weights of its segment of the row
// that the next token is drawn from; the sequence's last workgroup finds the
// segment in which their sum passes the random share, and the token in it.
template <int E>
__global__ __launch_bounds__(kVerThreads) void k_verify_pick(VerifyArgs a)
{
    constexpr int J = E / 8;
    __shared__ ExpTable table;
    __shared__ Joined p[IAM_VERIFY_MAX_DRAFT + 1], q[IAM_VERIFY_MAX_DRAFT];
    __shared__ int ok[IAM_VERIFY_MAX_DRAFT];
    __shared__ double sums[J][kVerWaves], part[kVerMaxSegs];
    __shared__ int last, picked;
    const int s = blockIdx.x / a.segs, seg = blockIdx.x - s * a.segs, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int n = drafts_of(a, s);
    const int* tokens = a.tokens + (size_t)s * a.n;
    const float* uniform = a.uniform + (size_t)s * (a.n + 1);
    fill_table(&table);
    for (int i = wave; i <= n; i += kVerWaves) {
        const size_t row = (size_t)s * (a.n + 1) + i, qrow = (size_t)s * a.n + i;
        const Joined x = join_row(a, row, a.target.unit);
        Joined y{0.0f, 1.0};
        if (i < n && a.draft.x) y = join_row(a, (size_t)a.seqs * (a.n + 1) + qrow, a.draft.unit);
        if (lane == 0) {
            p[i] = x;
            if (i < n) {
                q[i] = y;
                const int t = tokens[i];
                bool keep = false;
                if (t >= 0 && t < a.vocab) {
                    const double pt = exp(((double)logit_of(a.target, row, t) - (double)x.m) * (a.target.unit / kUnit)) / x.z;
                    const double qt = a.draft.x ? exp(((double)logit_of(a.draft, qrow, t) - (double)y.m) * (a.draft.unit / kUnit)) / y.z : 1.0;
                    keep = (double)uniform[i] * qt < pt;
                }
                ok[i] = keep;
            }
        }
    }
    __syncthreads();
    int kept = 0;
    while (kept < n && ok[kept]) kept++;
    const Joined pk = p[kept];
    int follow = -1;
    if (pk.z == pk.z) {
        Draw d;
        d.row = (size_t)s * (a.n + 1) + kept;
        d.qrow = (size_t)s * a.n + kept;
        d.gone = kept < n ? tokens[kept] : -1;
        d.less = kept < n && d.gone >= 0 && d.gone < a.vocab;
        d.pm = pk.m;
        d.pz = 1.0 / pk.z;
        d.qm = 0.0f;
        d.qz = 0.0;
        if (d.less && a.draft.x) {
            d.qm = q[kept].m;
            d.qz = 1.0 / q[kept].z;
            d.less = d.qz == d.qz;
        }
        Segment g = segment_of(a, a.target, d.row, seg);
        double sum = 0.0;
        for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * E) {
            double w[E];
            weights_of<E>(a, d, &table, g, c0, w);
#pragma unroll
            for (int e = 0; e < E; e++) sum += w[e];
        }
        sum = wave_sum(sum);
        if (lane == 0) sums[0][wave] = sum;
        __syncthreads();
        sum = 0.0;
        for (int i = 0; i < kVerWaves; i++) sum += sums[0][i];
        if (a.segs > 1) {
            if (tid == 0) acc_put(a.part + (size_t)s * a.segs + seg, sum);
            if (!acc_arrive(a.ctr + s, (uint32_t)a.segs, &last)) return;
            if (tid < a.segs) part[tid] = acc_peek(a.part + (size_t)s * a.segs + tid);
            if (tid == 0) a.ctr[s] = 0u;
        } else if (tid == 0) {
            part[0] = sum;
        }
        __syncthreads();
        double all = 0.0;
        for (int i = 0; i < a.segs; i++) all += part[i];
        if (d.less && !(all > 0.0)) {
            // nowhere positive: p alone, whose segments' sums are at hand
            d.less = false;
            __syncthreads();
            if (tid < a.segs) {
                const double* st = a.stat + (d.row * a.segs + tid) * 2;
                part[tid] = (float)st[0] == -INFINITY ? 0.0 : st[1] * exp((st[0] - (double)pk.m) * (a.target.unit / kUnit)) * d.pz;
            }
            __syncthreads();
            all = 0.0;
            for (int i = 0; i < a.segs; i++) all += part[i];
        }
        const double want = (double)uniform[a.n] * all;
        // the segment in which the sum passes it (by rounding none: the last of any weight)
        double before = 0.0;
        int at = -1;
        for (int i = 0; i < a.segs; i++) {
            if (before + part[i] > want) {
                at = i;
                break;
            }
            before += part[i];
        }
        if (at < 0)
            for (at = a.segs - 1; at > 0 && !(part[at] > 0.0); at--) before -= part[at];
        if (tid == 0) picked = -1;
        g = segment_of(a, a.target, d.row, at);
        int mine = -1;           // the last place of any weight
        for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * E) {
            double w[E], run[J];
            weights_of<E>(a, d, &table, g, c0, w);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < J; j++) {
                run[j] = 0.0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    run[j] += w[j * 8 + e];
                    if (w[j * 8 + e] > 0.0) mine = place_of(c0, j * 8 + e);
                }
                const double t = wave_sum(run[j]);
                if (lane == 0) sums[j][wave] = t;
            }
            __syncthreads();
            // the places are in the order of (run, wave, lane, value)
            int hit = -1;
            for (int i = 0; i < J * kVerWaves && hit < 0; i++) {
                const double t = sums[i / kVerWaves][i % kVerWaves];
                if (before + t > want) hit = i;
                else before += t;
            }
            if (hit < 0) continue;
            if (wave == hit % kVerWaves) {
#pragma unroll
                for (int j = 0; j < J; j++) {
                    if (j != hit / kVerWaves) continue;
                    const double incl = wave_scan(run[j]);
                    const uint64_t over = __ballot(before + incl > want), some = __ballot(run[j] > 0.0);
                    const int who = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
                    if (lane == who) {
                        double c = before + (incl - run[j]);
                        int place = -1;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const bool open = place < 0 || !(c > want);
                            c += w[j * 8 + e];
                            if (open && w[j * 8 + e] > 0.0) place = place_of(c0, j * 8 + e);
                        }
                        picked = place;
                    }
                }
            }
            break;
        }
        __syncthreads();
        if (picked < 0) {
            const uint32_t most = wave_max_u32((uint32_t)(mine + 1));
            __syncthreads();
            if (lane == 0) sums[0][wave] = (double)most;
            __syncthreads();
            double best = 0.0;
            for (int i = 0; i < kVerWaves; i++) best = fmax(best, sums[0][i]);
            follow = (int)best - 1;
        } else {
            follow = picked;
        }
    } else if (seg != 0) {
        return;
    }
    int* out = a.out + (size_t)s * (a.n + 1);
    for (int i = tid; i <= a.n; i += kVerThreads) out[i] = i < kept ? tokens[i] : i == kept ? follow : -1;
    if (tid == 0) a.accepted[s] = kept;
}

// ---- greedy
// Larger logits, then lower tokens, as whole numbers (0: nothing; a NaN or +inf
// is more than any)
__device__ __forceinline__ unsigned long long best_key(float x, int id)
{
    const uint32_t b = __float_as_uint(x + 0.0f), o = (b >> 31) ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (uint32_t)~id;
}

template <int E>
__global__ __launch_bounds__(kVerThreads) void k_verify_best(VerifyArgs a, int first)
{
    __shared__ unsigned long long best[kVerWaves];
    Which w;
    if (!which_of(a, first, w)) return;
    const Segment g = segment_of(a, a.target, w.row, w.seg);
    float m = -INFINITY;
    int at = -1;
    bool bad = false;
    for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * E) {
        float v[E];
        load_chunk<E>(a.target, w.row, c0, g.v0, g.v1, v);
#pragma unroll
        for (int e = 0; e < E; e++) {
            bad |= !(v[e] < INFINITY);
            at = v[e] > m ? place_of(c0, e) : at;
            m = fmaxf(m, v[e]);
        }
    }
    unsigned long long key = bad ? ~0ull : at >= 0 ? best_key(m, at) : 0ull;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long o = __shfl_xor(key, d);
        key = o > key ? o : key;
    }
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = key;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kVerWaves; i++) key = best[i] > key ? best[i] : key;
        reinterpret_cast<unsigned long long*>(a.stat)[w.stat] = key;
    }
}

// A wave takes a sequence.
__global__ __launch_bounds__(64) void k_verify_greedy(VerifyArgs a)
{
    const int s = blockIdx.x, lane = threadIdx.x, n = drafts_of(a, s);
    const int* tokens = a.tokens + (size_t)s * a.n;
    int* out = a.out + (size_t)s * (a.n + 1);
    const unsigned long long* stat = reinterpret_cast<const unsigned long long*>(a.stat);
    // lane i: row i (and row 64, of 65 at most)
    auto best_of = [&](int i) {
        unsigned long long key = 0;
        const size_t at = ((size_t)s * (a.n + 1) + i) * a.segs;
        for (int g = 0; g < a.segs; g++) {
            const unsigned long long o = stat[(at + g) * 2];
            key = o > key ? o : key;
        }
        return key == 0 || key == ~0ull ? -1 : (int)~(uint32_t)key;
    };
    const int mine = lane <= n ? best_of(lane) : -1, t = lane < n ? tokens[lane] : -1;
    const uint64_t wrong = __ballot(lane >= n || mine < 0 || mine != t);
    const int kept = min(n, wrong ? __ffsll((unsigned long long)wrong) - 1 : 64);
    const int follow = kept < 64 ? __shfl(mine, kept & 63) : best_of(64);
    for (int i = lane; i <= a.n; i += 64) out[i] = i < kept ? tokens[i] : i == kept ? follow : -1;
    if (lane == 0) a.accepted[s] = kept;
}

// ------------------------------------------------------------------ host ---
// workgroups that rows are cut into segments for
constexpr int kVerTarget = 2048;

template <int E>
static int verify_launch(Ctx* c, VerifyArgs a, bool greedy)
{
    constexpr int chunk = kVerThreads * E;
    const int targets = a.seqs * (a.n + 1), rows = targets + (a.draft.x ? a.seqs * a.n : 0);
    const int chunks = (int)(((int64_t)a.vocab + 7 + chunk - 1) / chunk);   // 7: values before the first that its chunk may hold
    const int want = std::max(1, std::min({chunks, kVerMaxSegs, (kVerTarget + rows - 1) / rows}));
    const int each = (chunks + want - 1) / want;
    a.segs = (chunks + each - 1) / each;
    a.per = (int)std::min<int64_t>((int64_t)each * chunk, 0x7fffffff);
    const size_t stats = (size_t)rows * a.segs * 2;
    IAM_TRY(ensure_verify_scratch(c, stats + (size_t)a.seqs * a.segs, (size_t)a.seqs));
    a.stat = c->ver_part;
    a.part = c->ver_part + stats;
    a.ctr = c->ver_ctr;
    // at most 2^22 workgroups a launch
    const int most = (1 << 22) / a.segs;
    for (int r0 = 0; r0 < rows; r0 += most) {
        const dim3 grid((unsigned)(std::min(most, rows - r0) * a.segs));
        IAM_TRY(greedy ? launch(c, "verify_best", k_verify_best<E>, grid, dim3(kVerThreads), 0, a, r0)
                       : launch(c, "verify_rows", k_verify_rows<E>, grid, dim3(kVerThreads), 0, a, r0));
    }
    if (greedy) return launch(c, "verify_greedy", k_verify_greedy, dim3((unsigned)a.seqs), dim3(64), 0, a);
    return launch(c, "verify_pick", k_verify_pick<E>, dim3((unsigned)(a.seqs * a.segs)), dim3(kVerThreads), 0, a);
}

}  // namespace iam

using namespace iam;

extern "C" int iam_verify_drafts(iam_ctx* c, const void* target, int t_type, size_t t_stride, const void* draft, int d_type,
                                 size_t d_stride, int seqs, int n, int vocab, double temperature, double draft_temperature,
                                 const int* tokens, const int* count, const float* uniform, int* out, int* accepted)
{
    if (!c || !target || !out || !accepted) return fail(IAM_E_INVALID, "verify_drafts: null argument");
    auto float_type = [](int t) { return t == IAM_F32 || t == IAM_F16 || t == IAM_BF16; };
    IAM_REQUIRE(float_type(t_type) && (!draft || float_type(d_type)), "verify_drafts: unknown type");
    IAM_REQUIRE(seqs >= 0 && seqs <= (1 << 16) && n >= 0 && n <= IAM_VERIFY_MAX_DRAFT, "verify_drafts: n_seq must be 0 to 2^16, n_draft 0 to 64");
    IAM_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "verify_drafts: vocab must be 1 to 2^30");
    const double least = 0x1p-64, most = 0x1p64;
    const bool greedy = temperature == 0.0;
    IAM_REQUIRE(greedy || (temperature >= least && temperature <= most), "verify_drafts: temperature must be 0, or 2^-64 to 2^64");
    if (greedy || n == 0) draft = nullptr;
    IAM_REQUIRE(!draft || (draft_temperature >= least && draft_temperature <= most), "verify_drafts: draft_temperature must be 2^-64 to 2^64");
    IAM_REQUIRE(greedy || uniform, "verify_drafts: random numbers are missing");
    IAM_REQUIRE(n == 0 || tokens, "verify_drafts: drafted tokens are missing");
    const size_t S = (size_t)seqs, V = (size_t)vocab, tb = type_bytes(t_type), db = draft ? type_bytes(d_type) : 4;
    if (!t_stride) t_stride = V;
    if (!d_stride) d_stride = V;
    const size_t far = (size_t)1 << 40;
    IAM_REQUIRE(t_stride >= V && d_stride >= V && t_stride < far && d_stride < far, "verify_drafts: a stride is smaller than a row");
    IAM_REQUIRE(aligned(target, tb) && aligned(draft, db) && aligned(tokens, 4) && aligned(count, 4) && aligned(uniform, 4) && aligned(out, 4) && aligned(accepted, 4),
                "verify_drafts: pointers must be aligned to their type");
    if (seqs == 0) return IAM_OK;
    struct {
        const void* p;
        size_t bytes;
        const char* what;
    } const part[] = {{out, S * (n + 1) * 4, "verify_drafts out"},
                      {accepted, S * 4, "verify_drafts accepted"},
                      {target, rows_bytes(S * (n + 1), V, t_stride, tb), "verify_drafts target"},
                      {draft, rows_bytes(S * n, V, d_stride, db), "verify_drafts draft"},
                      {n ? tokens : nullptr, S * n * 4, "verify_drafts tokens"},
                      {count, S * 4, "verify_drafts count"},
                      {greedy ? nullptr : uniform, S * (n + 1) * 4, "verify_drafts uniform"}};
    for (int i = 0; i < 7; i++) {
        if (!part[i].p) continue;
        IAM_TRY(check_dev_range(c, part[i].p, part[i].bytes, part[i].what));
        for (int j = 0; j < i && j < 2; j++)
            IAM_REQUIRE(!overlaps(part[i].p, part[i].bytes, part[j].p, part[j].bytes), "verify_drafts: an output overlaps another array");
    }
    DeviceGuard on(c);
    VerifyArgs a{};
    a.target = {target, t_stride, t_type, greedy ? 0.0 : kUnit / temperature};
    a.draft = {draft, d_stride, d_type, draft ? kUnit / draft_temperature : 0.0};
    a.seqs = seqs;
    a.n = n;
    a.vocab = vocab;
    a.tokens = tokens;
    a.count = count;
    a.uniform = uniform;
    a.out = out;
    a.accepted = accepted;
    // Smaller chunks where there are few values in all.
    const int64_t values = (int64_t)S * (n + 1) * vocab;
    return values <= ((int64_t)1 << 21) ? verify_launch<8>(c, a, greedy) : verify_launch<32>(c, a, greedy);
}
