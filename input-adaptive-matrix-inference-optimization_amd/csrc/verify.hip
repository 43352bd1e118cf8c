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
// p - q counts as nowhere positive where its positive parts add up to less: each
// of p and q is off by about 1e-13 of itself (the exponentials' 4e-14, and fp64
// sums in an order that depends on where a row lies)
constexpr double kNowhere = 1e-12;

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
    int draw_segs, draw_per; // the same of the row that the last token is drawn from
    const int* tokens;
    const int* count;        // may be null
    const float* uniform;
    int* out;
    int* accepted;
    double* stat;            // [seqs (n + 1) + seqs n][segs][2]: largest logit, sum of exponentials; the best key (greedy)
    double* part;            // [seqs][draw_segs][waves]: weights of the row's parts that the last token is drawn from
    uint32_t* ctr;           // [seqs], zero on entry (left zero)
};

// ---- exponentials
// 2^(t / 64) in fp64 for t <= 0: the table's 2^(j / 64) times a polynomial of the
// rest f, |f| <= 1/2 (the series of e^(f ln 2 / 64) up to the fourth power: 4e-14).
constexpr double kUnit = 64.0 * 1.44269504088896340736;   // t of e^1
// 2^(j / 64)
__constant__ const double kRoots[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};
// The table is held 32 times, side by side: each lane reads its own banks, so
// that 64 lanes' places do not meet.
constexpr int kCopies = 32;
struct ExpTable {
    double t[64 * kCopies];
};
__device__ __forceinline__ void fill_table(ExpTable* e)
{
    constexpr int each = kCopies / kVerWaves;
    const double v = kRoots[threadIdx.x & 63];
#pragma unroll
    for (int i = 0; i < each; i++) e->t[(threadIdx.x & 63) * kCopies + (threadIdx.x >> 6) * each + (threadIdx.x + i) % each] = v;
}
// e^(d unit / kUnit) as p e, e a power of two times a table's entry
struct ExpParts {
    double p, e;
};
__device__ __forceinline__ ExpParts exp_of(const ExpTable* table, double d, double unit)
{
    constexpr double u = 1.0 / kUnit;
    constexpr double whole = 6755399441055744.0;   // 1.5 2^52: what is added to it is rounded to whole numbers
    const double tn = __builtin_fma(d, unit, whole), f = __builtin_fma(d, unit, whole - tn);
    // (an operand of an instruction from the scalar registers or constants at
    // most: a copy for each value otherwise)
    double p = u * u * u * u / 24.0;
    asm("" : "+v"(p));
    p = __builtin_fma(p, f, u * u * u / 6.0);
    p = __builtin_fma(p, f, u * u / 2.0);
    p = __builtin_fma(p, f, u);
    p = __builtin_fma(p, f, 1.0);
    const int i = (int)(uint32_t)__double_as_longlong(tn);
    return {p, ldexp(table->t[(i & 63) * kCopies + (threadIdx.x & (kCopies - 1))], i >> 6)};
}

// What a row's exponentials are taken relative to: its largest logit.
struct Base {
    double unit, m, lowest;
    __device__ __forceinline__ Base(double unit, float m) : unit(unit), m((double)m), lowest(-64.0 * 1100.0 / unit) {}
    // e^((x - m) / temperature); 0 below 2^-1074, -inf too
    __device__ __forceinline__ ExpParts weight(const ExpTable* e, float x) const { return exp_of(e, fmax((double)x - m, lowest), unit); }
};

// ---- reading a row
// E values a thread of a chunk of 256 E, from place c0 on, in runs of 8 that lie
// 2048 values apart: value e of the thread is at place_of(c0, e).  Outside
// [v0, v1), -inf.
__device__ __forceinline__ int place_of(int c0, int e) { return c0 + (e / 8 * kVerThreads + (int)threadIdx.x) * 8 + e % 8; }
// RUN values from place i on
template <typename T, int RUN>
__device__ __forceinline__ Pack<T, RUN, (int)sizeof(T)> run_at(const T* x, int i, int v0, int v1)
{
    typedef Pack<T, RUN, (int)sizeof(T)> Run;
    if (i >= v0 && i + RUN <= v1) return *reinterpret_cast<const Run*>(x + i);
    Run r;
#pragma unroll
    for (int e = 0; e < RUN; e++) r.v[e] = i + e >= v0 && i + e < v1 ? x[i + e] : (T)-INFINITY;
    return r;
}
template <typename T, int E>
struct Runs {
    typedef Pack<T, 8, (int)sizeof(T)> Run;
    Run r[E / 8];

    __device__ __forceinline__ void load(const T* x, int c0, int v0, int v1)
    {
        if (c0 >= v0 && c0 + kVerThreads * E <= v1) {
#pragma unroll
            for (int j = 0; j < E / 8; j++) r[j] = *reinterpret_cast<const Run*>(x + place_of(c0, j * 8));
            return;
        }
#pragma unroll
        for (int j = 0; j < E / 8; j++) r[j] = run_at<T, 8>(x, place_of(c0, j * 8), v0, v1);
    }
    __device__ __forceinline__ float operator[](int e) const { return to_f32(r[e / 8].v[e % 8]); }
};

__device__ __forceinline__ size_t value_bytes(int type) { return type == IAM_F32 ? 4 : 2; }
// f(the row's values in their type)
template <typename F>
__device__ __forceinline__ void with_row(const Rows& r, size_t row, F f)
{
    if (r.type == IAM_F32) f(reinterpret_cast<const float*>(r.x) + row * r.stride);
    else if (r.type == IAM_F16) f(reinterpret_cast<const _Float16*>(r.x) + row * r.stride);
    else f(reinterpret_cast<const __bf16*>(r.x) + row * r.stride);
}
template <int E>
__device__ __forceinline__ void load_chunk(const Rows& r, size_t row, int c0, int v0, int v1, float* v)
{
    with_row(r, row, [&](auto* x) __attribute__((always_inline)) {
        Runs<std::remove_const_t<std::remove_pointer_t<decltype(x)>>, E> q;
        q.load(x, c0, v0, v1);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = q[e];
    });
}
// E values in a row, from place i on
template <int E>
__device__ __forceinline__ void load_place(const Rows& r, size_t row, int i, int v0, int v1, float* v)
{
    constexpr int RUN = E < 8 ? E : 8;
    with_row(r, row, [&](auto* x) __attribute__((always_inline)) {
        typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
        Pack<T, RUN, (int)sizeof(T)> q[E / RUN];
#pragma unroll
        for (int j = 0; j < E / RUN; j++) q[j] = run_at<T, RUN>(x, i + j * RUN, v0, v1);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = to_f32(q[e / RUN].v[e % RUN]);
    });
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
__device__ __forceinline__ Segment segment_of(const VerifyArgs& a, const Rows& r, size_t row, int seg, int per)
{
    const size_t bytes = value_bytes(r.type);
    const int off = (int)(((uintptr_t)r.x + row * r.stride * bytes) / bytes % (16 / bytes));
    Segment s;
    s.o = seg * per - off;
    s.v0 = max(s.o, 0);
    s.v1 = a.vocab - s.o > per ? s.o + per : a.vocab;
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
// has its own m.  Bound by the fp64 arithmetic: 17 instructions a value, 12 of
// them fp64, 0.70 us per million values (128 rows of 128001 bf16 logits 24 us, 256 41).
template <typename T, int E>
__global__ __launch_bounds__(kVerThreads) void k_verify_rows(VerifyArgs a, int first)
{
    __shared__ ExpTable table;
    __shared__ float wave_m[kVerWaves];
    __shared__ double wave_z[kVerWaves];
    Which w;
    if (!which_of(a, first, w)) return;
    const Rows& r = w.draft ? a.draft : a.target;
    const T* x = reinterpret_cast<const T*>(r.x) + w.row * r.stride;
    const Segment g = segment_of(a, r, w.row, w.seg, a.per);
    Runs<T, E> next;
    if (g.o < g.v1) next.load(x, g.o, g.v0, g.v1);
    fill_table(&table);
    __syncthreads();
    float m = -INFINITY;
    double z = 0.0;
    bool bad = false;
    for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * E) {
        const Runs<T, E> v = next;
        if (c0 + kVerThreads * E < g.v1) next.load(x, c0 + kVerThreads * E, g.v0, g.v1);
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
        const Base b(r.unit, m);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const ExpParts w = b.weight(&table, v[e]);
            z = __builtin_fma(w.p, w.e, z);
        }
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

// A row's largest logit and sum; the sum is NaN where the row has no distribution
struct Joined {
    float m;
    double z;
};

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

// the weights of the E values from place i on
template <int E>
__device__ __forceinline__ void weights_of(const VerifyArgs& a, const Draw& d, const ExpTable* table, const Segment& g, int i, double* w)
{
    const bool two = d.less && a.draft.x;
    float v[E], u[E];
    load_place<E>(a.target, d.row, i, g.v0, g.v1, v);
    if (two) load_place<E>(a.draft, d.qrow, i, g.v0, g.v1, u);
    const Base b(a.target.unit, d.pm);
#pragma unroll
    for (int e = 0; e < E; e++) {
        const ExpParts t = b.weight(table, v[e]);
        w[e] = t.p * t.e * d.pz;
    }
    if (two) {
        const Base q(a.draft.unit, d.qm);
#pragma unroll
        for (int e = 0; e < E; e++) {
            // rounded like p (no fma): equal rows leave 0, not p's rounding error
            const ExpParts t = q.weight(table, u[e]);
            w[e] = fmax(w[e] - t.p * t.e * d.qz, 0.0);
        }
    } else if (d.less) {
#pragma unroll
        for (int e = 0; e < E; e++) w[e] = i + e == d.gone ? 0.0 : w[e];
    }
}

// Which drafted tokens of a sequence are kept, by every workgroup of it: the rows'
// segments joined by `width` lanes a row, all rows at once where they
// are few, then lane i judges token i.  p, q: LDS
__device__ __forceinline__ int kept_of(const VerifyArgs& a, int s, int n, Joined* p, Joined* q)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const int* tokens = a.tokens + (size_t)s * a.n;
    // what lane i needs of token i, on its way while the rows are joined
    const int t = lane < n ? tokens[lane] : -1;
    const bool there = t >= 0 && t < a.vocab;
    const size_t row = (size_t)s * (a.n + 1) + lane, qrow = (size_t)s * a.n + lane;
    float u = 0.0f, x = 0.0f, y = 0.0f;
    if (there) {
        u = a.uniform[(size_t)s * (a.n + 1) + lane];
        x = logit_of(a.target, row, t);
        if (a.draft.x) y = logit_of(a.draft, qrow, t);
    }
    int width = 1;
    while (width < a.segs) width *= 2;
    const int rows = n + 1 + (a.draft.x ? n : 0), g = tid & (width - 1);
    for (int r0 = 0; r0 < rows; r0 += kVerThreads / width) {
        const int r = r0 + tid / width, i = r <= n ? r : r - n - 1;
        const size_t at = ((r <= n ? (size_t)s * (a.n + 1) : (size_t)a.seqs * (a.n + 1) + (size_t)s * a.n) + i) * a.segs + g;
        const double unit = r <= n ? a.target.unit : a.draft.unit;
        float m = -INFINITY;
        double z = 0.0;
        if (r < rows && g < a.segs) {
            m = (float)a.stat[at * 2];
            z = a.stat[at * 2 + 1];
        }
        float top = m;
        for (int d = 1; d < width; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        const double f = m == top ? 1.0 : m == -INFINITY ? 0.0 : exp(((double)m - (double)top) * (unit / kUnit));
        z = z != z ? z : z * f;
        for (int d = 1; d < width; d *= 2) z += __shfl_xor(z, d);
        if (r < rows && g == 0) (r <= n ? p : q)[i] = {top, top == -INFINITY ? NAN : z};
    }
    __syncthreads();
    bool keep = false;
    if (there) {
        const Joined pi = p[lane];
        const double pt = exp(((double)x - (double)pi.m) * (a.target.unit / kUnit)) / pi.z;
        double qt = 1.0;
        if (a.draft.x) {
            const Joined qi = q[lane];
            qt = exp(((double)y - (double)qi.m) * (a.draft.unit / kUnit)) / qi.z;
        }
        keep = (double)u * qt < pt;
    }
    const uint64_t wrong = __ballot(!keep);
    return wrong ? __ffsll((unsigned long long)wrong) - 1 : 64;   // lanes from n on keep nothing
}

// the sum of the weights of a wave's part of segment seg, in every lane; E values in a row a lane
template <int E>
__device__ __forceinline__ double part_sum(const VerifyArgs& a, const Draw& d, const ExpTable* table, int seg)
{
    const Segment g = segment_of(a, a.target, d.row, seg * kVerWaves + (int)(threadIdx.x >> 6), a.draw_per / kVerWaves);
    double sum = 0.0;
    for (int c0 = g.o; c0 < g.v1; c0 += 64 * E) {
        double w[E];
        weights_of<E>(a, d, table, g, c0 + (int)(threadIdx.x & 63) * E, w);
#pragma unroll
        for (int e = 0; e < E; e++) sum += w[e];
    }
    return wave_sum(sum);
}

// Workgroup (sequence, segment): which drafted tokens are kept, the weights of
// its segment of the row that the next token is drawn from, a sum for each
// wave's part of it; the sequence's last workgroup finds the part in which their
// sum passes the random share, and the token in it.  Of 19.3 us for 32 sequences of
// 128001 bf16 logits 4 are the launch, 3.5 the judging, 6 the weights (fp64
// arithmetic) and the rest the last workgroups' chain of loads.
template <int E>
__global__ __launch_bounds__(kVerThreads, 4) void k_verify_pick(VerifyArgs a)
{
    constexpr int kLast = 4;     // values of a thread in the last workgroup's search
    __shared__ ExpTable table;
    __shared__ Joined p[IAM_VERIFY_MAX_DRAFT + 1], q[IAM_VERIFY_MAX_DRAFT];
    __shared__ double sums[kVerWaves], part[kVerMaxSegs * kVerWaves];
    __shared__ int last, found[kVerWaves];
    const int s = blockIdx.x / a.draw_segs, seg = blockIdx.x - s * a.draw_segs, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int n = drafts_of(a, s), parts = a.draw_segs * kVerWaves;
    const double share = (double)a.uniform[(size_t)s * (a.n + 1) + a.n];
    fill_table(&table);
    const int kept = kept_of(a, s, n, p, q);
    const Joined pk = p[kept];
    const int* tokens = a.tokens + (size_t)s * a.n;
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
        const double sum = part_sum<E>(a, d, &table, seg);
        if (a.draw_segs > 1) {
            double* all = a.part + (size_t)s * parts;
            if (lane == 0) acc_put(all + seg * kVerWaves + wave, sum);
            if (!acc_arrive(a.ctr + s, (uint32_t)a.draw_segs, &last)) return;
            if (tid < parts) part[tid] = acc_peek(all + tid);
            if (tid == 0) a.ctr[s] = 0u;
        } else if (lane == 0) {
            part[wave] = sum;
        }
        __syncthreads();
        // lane i: segment i
        double own[kVerWaves];
        auto take = [&] {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < kVerWaves; i++) sum += own[i] = lane < a.draw_segs ? part[lane * kVerWaves + i] : 0.0;
            return sum;
        };
        double whole = take(), upto = wave_scan(whole);
        if (d.less && !(__shfl(upto, 63) > kNowhere)) {
            // nowhere positive: p alone (a token that neither row gives any probability)
            d.less = false;
            __syncthreads();
            for (int i = 0; i < a.draw_segs; i++) {
                const double t = part_sum<E>(a, d, &table, i);
                if (lane == 0) part[i * kVerWaves + wave] = t;
            }
            __syncthreads();
            whole = take();
            upto = wave_scan(whole);
        }
        const double want = share * __shfl(upto, 63);
        // the segment, then the part, in which the sum passes it (by rounding none:
        // the last of any weight).  Of those with any weight: the scan adds in a tree,
        // and behind the border a weightless one's sum may differ from the one before
        // by rounding.
        const uint64_t past = __ballot(whole > 0.0 && upto > want), some = __ballot(whole > 0.0);
        const int at = past ? __ffsll((unsigned long long)past) - 1 : some ? 63 - __clzll((long long)some) : 0;
        const double left = __shfl(upto, max(at - 1, 0));
        double before = at ? left : 0.0, sofar = before;
        int in = -1;
#pragma unroll
        for (int i = 0; i < kVerWaves; i++) {
            const double w = __shfl(own[i], at);
            if (w > 0.0 && (in < 0 || !(sofar > want))) {
                in = i;
                before = sofar;
            }
            sofar += w;
        }
        const Segment g = segment_of(a, a.target, d.row, at * kVerWaves + max(in, 0), a.draw_per / kVerWaves);
        int mine = -1;           // the thread's last place of any weight
        for (int c0 = g.o; c0 < g.v1; c0 += kVerThreads * kLast) {
            double w[kLast], run = 0.0;
            const int i0 = c0 + tid * kLast;
            weights_of<kLast>(a, d, &table, g, i0, w);
#pragma unroll
            for (int e = 0; e < kLast; e++) {
                run += w[e];
                if (w[e] > 0.0) mine = i0 + e;
            }
            const double incl = wave_scan(run);
            __syncthreads();
            if (lane == 63) sums[wave] = incl;
            __syncthreads();
            // each wave's first lane of any weight whose sum passes it, then the first wave's
            double start = before;
            for (int i = 0; i < wave; i++) start += sums[i];
            const uint64_t over = __ballot(run > 0.0 && start + incl > want);
            const double left = __shfl_up(incl, 1);
            if (lane == (over ? __ffsll((unsigned long long)over) - 1 : 0)) {
                double c = start + (lane ? left : 0.0);
                int place = -1;
#pragma unroll
                for (int e = 0; e < kLast; e++) {
                    if (w[e] > 0.0 && (place < 0 || !(c > want))) place = i0 + e;
                    c += w[e];
                }
                found[wave] = over ? place : -1;
            }
            __syncthreads();
            for (int i = 0; i < kVerWaves; i++) {
                if (follow < 0) follow = found[i];
                before += sums[i];
            }
            if (follow >= 0) break;
        }
        if (follow < 0) {
            const uint32_t most = wave_max_u32((uint32_t)(mine + 1));
            __syncthreads();
            if (lane == 0) sums[wave] = (double)most;
            __syncthreads();
            double best = 0.0;
            for (int i = 0; i < kVerWaves; i++) best = fmax(best, sums[i]);
            follow = (int)best - 1;
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
    const Segment g = segment_of(a, a.target, w.row, w.seg, a.per);
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
constexpr int kVerTarget = 4096;

// segments of a row for about `want` of them, in whole chunks
static void cut_row(int vocab, int chunk, int want, int* segs, int* per)
{
    const int chunks = (int)(((int64_t)vocab + 7 + chunk - 1) / chunk);   // 7: values before the first that its chunk may hold
    const int n = std::max(1, std::min({chunks, kVerMaxSegs, want})), each = (chunks + n - 1) / n;
    *segs = (chunks + each - 1) / each;
    *per = (int)std::min<int64_t>((int64_t)each * chunk, 0x7fffffff);
}

template <int E>
static int verify_launch(Ctx* c, VerifyArgs a, bool greedy)
{
    const int targets = a.seqs * (a.n + 1), rows = targets + (a.draft.x ? a.seqs * a.n : 0);
    cut_row(a.vocab, kVerThreads * E, (kVerTarget + rows - 1) / rows, &a.segs, &a.per);
    cut_row(a.vocab, kVerThreads * E, (kVerTarget + a.seqs - 1) / a.seqs, &a.draw_segs, &a.draw_per);
    const size_t stats = (size_t)rows * a.segs * 2;
    IAM_TRY(ensure_verify_scratch(c, stats + (size_t)a.seqs * a.draw_segs * kVerWaves, (size_t)a.seqs));
    a.stat = c->ver_part;
    a.part = c->ver_part + stats;
    a.ctr = c->ver_ctr;
    // rows [r0, r1), at most 2^22 workgroups a launch
    auto pass = [&](int r0, int r1, int type) {
        const int most = (1 << 22) / a.segs;
        for (; r0 < r1; r0 += most) {
            const dim3 grid((unsigned)(std::min(most, r1 - r0) * a.segs)), block(kVerThreads);
            if (greedy) IAM_TRY(launch(c, "verify_best", k_verify_best<E>, grid, block, 0, a, r0));
            else if (type == IAM_F32) IAM_TRY(launch(c, "verify_rows", k_verify_rows<float, E>, grid, block, 0, a, r0));
            else if (type == IAM_F16) IAM_TRY(launch(c, "verify_rows", k_verify_rows<_Float16, E>, grid, block, 0, a, r0));
            else IAM_TRY(launch(c, "verify_rows", k_verify_rows<__bf16, E>, grid, block, 0, a, r0));
        }
        return IAM_OK;
    };
    const bool one = rows == targets || a.draft.type == a.target.type;
    IAM_TRY(pass(0, one ? rows : targets, a.target.type));
    if (!one) IAM_TRY(pass(targets, rows, a.draft.type));
    if (greedy) return launch(c, "verify_greedy", k_verify_greedy, dim3((unsigned)a.seqs), dim3(64), 0, a);
    return launch(c, "verify_pick", k_verify_pick<E>, dim3((unsigned)(a.seqs * a.draw_segs)), dim3(kVerThreads), 0, a);
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
    // Smaller chunks where there are few values in all (one sequence, 5 rows of
    // 32000: 12.2 us, 13.0 with larger ones).
    const int64_t values = (int64_t)S * (n + 1) * vocab;
    return values <= ((int64_t)1 << 21) ? verify_launch<8>(c, a, greedy) : verify_launch<16>(c, a, greedy);
}
