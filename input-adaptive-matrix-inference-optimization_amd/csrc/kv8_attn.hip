// Attention over the 8-bit KV cache: one token a sequence, or many.
//
// With q' = q * scale * log2(e), one KV head's rows of queries r (its n_heads /
// n_kv query heads of each token) and positions t:
//   s[t][r] = (k8[t] . q'[r]) * k_scale[block of t],  hidden positions -inf
//   p = 2^(s - m),  l[r] = sum p,  o[r] = sum over blocks v_scale * (sum p v8[t]),
// in one pass with the running maximum m[r] of the rows, o / l at the end.
#include <cmath>

#include "accum.h"
#include "kv8.h"
#include "wave.h"

namespace iam {

// A wave takes blocks of 64 positions, each 2 * 64 * head_dim bytes straight
// from memory into registers in the order of the matrix instructions (16x16x32
// in fp16, fp32 sums; 8-bit numbers are exact in fp16), no LDS:
//   S^T = K Q^T  A: 16 positions of K, B: 16 query rows; lane (g, r) then
//                holds positions 4 g .. 4 g + 3 of each 16 for row r
//   O^T = V^T P^T  A: 16 dimensions of V, its 32 positions in the order in
//                which B, the lane's own p, has them: p goes from the
//                softmax's registers into the product without moving lanes.
// Rows are in lanes (r), so the rescaling by 2^(m - m') is one factor a lane.
// Precision: q and p are fp32; each is split into two fp16 parts, high and
// low (22 bits), after a power of two that brings them near the top of fp16's
// range, and both are multiplied (an fp16 or bf16 q needs one part).
constexpr int kAttn8Threads = 256, kAttn8Waves = 4;
constexpr float kProbShift = 12.0f;   // p is held as 2^12 p: its low part stays a normal number

struct Attn8Args {
    const void* q;
    void* out;
    const uint8_t* kt;
    const uint8_t* vt;
    const float* ks;
    const float* vs;
    const uint16_t* ko;
    const uint16_t* vo;
    const int* pos;
    const int* count;
    Kv8Geometry g;
    int type;
    int heads, rep;          // query heads; of them per KV head
    int tokens, rows;        // of a sequence; rows = tokens * rep
    int groups;              // row groups of a sequence
    int items;               // n_seq * groups
    int planned;             // blocks dealt out over the context (else one workgroup an item and KV head)
    int target;              // planned: workgroups per KV head to aim at
    size_t q_stride, out_stride;
    int window;
    float scale_log2;
    float* part;             // partial results of the split items
    uint32_t* ctr;           // [items * n_kv] arrivals, zero on entry (left zero)
};

struct Span {
    int seq, first_row, n_rows;   // rows of the item that are there
    int b0, nb;                   // blocks they see
    int p0;
};

// what item `it` has to read
__device__ __forceinline__ Span span_of(const Attn8Args& a, int it, int rows_per_item)
{
    Span s;
    s.seq = it / a.groups;
    s.first_row = (it - s.seq * a.groups) * rows_per_item;
    s.p0 = a.pos[s.seq];
    const int n = a.count ? min(a.tokens, a.count[s.seq]) : a.tokens;
    s.n_rows = max(0, min(s.first_row + rows_per_item, n * a.rep) - s.first_row);
    s.b0 = s.nb = 0;
    if (s.n_rows > 0 && s.p0 >= 0) {
        const int top = a.g.max_ctx - 1;
        const int t0 = s.first_row / a.rep, t1 = (s.first_row + s.n_rows - 1) / a.rep;
        const int hi = s.p0 > top - t1 ? top : s.p0 + t1, lo_p = s.p0 > top - t0 ? top : s.p0 + t0;
        const int lo = a.window > 0 ? max(0, lo_p - a.window + 1) : 0;
        s.b0 = lo / kBlk;
        s.nb = hi / kBlk - s.b0 + 1;
    }
    return s;
}

__device__ __forceinline__ int block_sum_scan(int v, int* wsum, int& total)
{
    const int w = threadIdx.x >> 6;
    const int incl = wave_incl_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wsum[w] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kAttn8Waves; i++) {
        before += i < w ? wsum[i] : 0;
        total += wsum[i];
    }
    return before + incl - v;
}

struct Share {
    int item, split, splits, per, slot0;   // per: blocks of a workgroup
};

// Every workgroup finds its share of the work from the positions on the
// device: G blocks a workgroup such that the total fills `target` workgroups a
// KV head; item i takes ceil(nb_i / G) of them (one at least).
__device__ __forceinline__ bool find_share(const Attn8Args& a, int j, int rows_per_item, Share* out)
{
    __shared__ int wsum[kAttn8Waves];
    __shared__ Share found;
    const int tid = threadIdx.x;
    const int per = (a.items + kAttn8Threads - 1) / kAttn8Threads;
    const int i0 = tid * per, i1 = min(a.items, i0 + per);
    int mine = 0, total;
    for (int i = i0; i < i1; i++) mine += span_of(a, i, rows_per_item).nb;
    block_sum_scan(mine, wsum, total);
    const int G = max(kAttn8Waves, (total + a.target - 1) / a.target);
    int ws = 0, slots = 0, all_ws, all_slots;
    for (int i = i0; i < i1; i++) {
        const int n = max(1, (span_of(a, i, rows_per_item).nb + G - 1) / G);
        ws += n;
        slots += n > 1 ? n : 0;
    }
    int w0 = block_sum_scan(ws, wsum, all_ws), s0 = block_sum_scan(slots, wsum, all_slots);
    if (j >= all_ws) return false;
    if (j >= w0 && j < w0 + ws)
        for (int i = i0; i < i1; i++) {
            const int n = max(1, (span_of(a, i, rows_per_item).nb + G - 1) / G);
            if (j < w0 + n) {
                found = {i, j - w0, n, G, s0};
                break;
            }
            w0 += n;
            s0 += n > 1 ? n : 0;
        }
    __syncthreads();
    *out = found;
    return true;
}

// 8 numbers of a tile's run (half 0 or 1) as an operand
template <int FMT>
__device__ __forceinline__ half8 operand(const uint4& w, int h)
{
    half2v a, b, c, d;
    widen4<FMT>(h ? w.z : w.x, a, b);
    widen4<FMT>(h ? w.w : w.y, c, d);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ void load_row8(const void* q, size_t at, float* v)
{
    const Pack<T, 8, (int)sizeof(T)> r = *reinterpret_cast<const Pack<T, 8, (int)sizeof(T)>*>(reinterpret_cast<const T*>(q) + at);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = to_f32(r.v[e]);
}

template <typename T>
__device__ __forceinline__ void store_row4(void* o, size_t at, floatx4 v)
{
    Pack<T, 4, (int)sizeof(T)> r;
#pragma unroll
    for (int e = 0; e < 4; e++) r.v[e] = from_f32<T>(v[e]);
    *reinterpret_cast<Pack<T, 4, (int)sizeof(T)>*>(reinterpret_cast<T*>(o) + at) = r;
}

// four floats handed to another workgroup (two 8-byte words)
__device__ __forceinline__ void put4(float* p, floatx4 v)
{
    typedef unsigned long long ull2 __attribute__((ext_vector_type(2)));
    const ull2 u = __builtin_bit_cast(ull2, v);
    acc_put(reinterpret_cast<unsigned long long*>(p), u[0]);
    acc_put(reinterpret_cast<unsigned long long*>(p) + 1, u[1]);
}
__device__ __forceinline__ floatx4 peek4(float* p)
{
    typedef unsigned long long ull2 __attribute__((ext_vector_type(2)));
    ull2 u;
    u[0] = acc_peek(reinterpret_cast<unsigned long long*>(p));
    u[1] = acc_peek(reinterpret_cast<unsigned long long*>(p) + 1);
    return __builtin_bit_cast(floatx4, u);
}

// SPLIT: q is fp32, in two parts.  NT: tiles of 16 query rows an item has.
template <int HD, int FMT, bool SPLIT, int NT>
__global__ __launch_bounds__(kAttn8Threads) void k_kv8_attn(Attn8Args a)
{
    constexpr int KS = HD / 32, DT = HD / 16, R = 16 * NT;
    constexpr int DC = NT * DT <= 8 ? DT : 8 / NT;   // dimension tiles the waves' sums meet in at a time
    constexpr int RUNS = HD / 16;                    // 16-byte runs of a tile per lane
    __shared__ floatx4 meet[kAttn8Waves][NT * DC][64];
    __shared__ float sm[kAttn8Waves][R], sl[kAttn8Waves][R];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r16 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.g.n_kv, j = blockIdx.x / a.g.n_kv;
    Share sh;
    if (a.planned) {
        if (!find_share(a, j, R, &sh)) return;
    } else {
        // the row groups with the longest contexts first
        sh = {a.items - 1 - j, 0, 1, 1 << 30, 0};
    }
    const Span sp = span_of(a, sh.item, R);
    if (sp.n_rows == 0) return;
    const int bs = sp.b0 + (int)min((long long)sh.split * sh.per, (long long)sp.nb);
    const int be = sp.b0 + (int)min((long long)(sh.split + 1) * sh.per, (long long)sp.nb);

    // this lane's rows: positions they see, their queries
    int hi[NT], lo[NT];
    float mult[NT];
    half8 qh[NT][KS], ql[SPLIT ? NT : 1][SPLIT ? KS : 1];
    const size_t qrow0 = (size_t)sp.seq * a.tokens;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int row = sp.first_row + n * 16 + r16;
        const bool there = n * 16 + r16 < sp.n_rows;
        const int t = there ? row / a.rep : 0, head = kvh * a.rep + (there ? row - t * a.rep : 0);
        hi[n] = there && sp.p0 >= 0 ? (sp.p0 > a.g.max_ctx - 1 - t ? a.g.max_ctx - 1 : sp.p0 + t) : -1;
        lo[n] = a.window > 0 ? max(0, hi[n] - a.window + 1) : 0;
        float v[KS][8], top = 0.0f;
        const size_t at = (qrow0 + t) * a.q_stride + (size_t)head * HD;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            // instruction k of the dimensions 64 (k/2) + 16 g + 8 (k%2) ..
            const size_t ad = at + (k >> 1) * 64 + g * 16 + (k & 1) * 8;
            if (!there) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[k][e] = 0.0f;
            } else if (SPLIT) {
                load_row8<float>(a.q, ad, v[k]);
            } else if (a.type == IAM_F16) {
                load_row8<_Float16>(a.q, ad, v[k]);
            } else {
                load_row8<__bf16>(a.q, ad, v[k]);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(v[k][e]));
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // the power of two that brings the row's largest value into [2^9, 2^10)
        int ex = 10;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &ex);
        mult[n] = ldexpf(a.scale_log2, ex - 10);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = ldexpf(v[k][e], 10 - ex);
                const _Float16 h = (_Float16)x;
                qh[n][k][e] = h;
                if constexpr (SPLIT) ql[n][k][e] = (_Float16)(x - (float)h);
            }
    }

    float m[NT], l[NT];
    floatx4 o[NT][DT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[n][d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // positions that every row there sees: below lo_all and past hi_all a mask is needed
    const int top_ctx = a.g.max_ctx - 1;
    const int t_first = sp.first_row / a.rep, t_last = (sp.first_row + sp.n_rows - 1) / a.rep;
    const int hi_all = sp.p0 > top_ctx - t_first ? top_ctx : sp.p0 + t_first;
    const int hi_max = sp.p0 > top_ctx - t_last ? top_ctx : sp.p0 + t_last;
    const int lo_all = a.window > 0 ? max(0, hi_max - a.window + 1) : 0;

    // one block: getk / getv give the operands, bad the positions (a bit for
    // each of the lane's 16) whose V is not finite (open block)
    auto block_step = [&](int b, float ksc, float vsc, auto&& getk, auto&& getv, uint32_t bad, auto&& after_k)
                          __attribute__((always_inline)) {
        floatx4 s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < 4; t++) s[n][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const half8 ka = getk(t, k);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    s[n][t] = mfma(ka, qh[n][k], s[n][t]);
                    if constexpr (SPLIT) s[n][t] = mfma(ka, ql[n][k], s[n][t]);
                }
            }
        after_k();
        const bool edge = b * kBlk + kBlk - 1 > hi_all || b * kBlk < lo_all;
        half8 ph[NT][2], pl[NT][2];
        float alpha[NT], vsr[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float f = mult[n] * ksc;
            float top = -INFINITY;
            vsr[n] = vsc;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[n][t][i] * f;
                    if (bad >> (t * 4 + i) & 1) x = NAN;
                    if (edge) {
                        const int p = b * kBlk + t * 16 + g * 4 + i;
                        x = p >= lo[n] && p <= hi[n] ? x : -INFINITY;
                    }
                    s[n][t][i] = x;
                    top = fmaxf(top, x);
                }
            // a block that the row does not see adds nothing, whatever its scale
            if (edge && (b * kBlk > hi[n] || b * kBlk + kBlk - 1 < lo[n])) vsr[n] = 0.0f;
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(m[n], top);
            const float safe = mn == -INFINITY ? 0.0f : mn;
            alpha[n] = __builtin_amdgcn_exp2f(m[n] - safe);
            m[n] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(s[n][t][i] - safe + kProbShift);
                    sum += p;
                    const _Float16 h = (_Float16)p;
                    ph[n][t >> 1][(t & 1) * 4 + i] = h;
                    pl[n][t >> 1][(t & 1) * 4 + i] = (_Float16)(p - (float)h);
                }
            l[n] = l[n] * alpha[n] + sum;
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const half8 v0 = getv(d, 0), v1 = getv(d, 1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                x = mfma(v0, ph[n][0], x);
                x = mfma(v1, ph[n][1], x);
                x = mfma(v0, pl[n][0], x);
                x = mfma(v1, pl[n][1], x);
#pragma unroll
                for (int i = 0; i < 4; i++) o[n][d][i] = __builtin_fmaf(x[i], vsr[n], o[n][d][i] * alpha[n]);
            }
        }
    };

    uint4 kr[RUNS], vr[RUNS];
    float ksc = 0.0f, vsc = 0.0f;
    auto cell_of = [&](int b) { return kv8_cell(a.g, sp.seq, b, kvh); };
    auto load_k = [&](int b) __attribute__((always_inline)) {
        const size_t cell = cell_of(b);
        const uint4* p = reinterpret_cast<const uint4*>(a.kt + cell * (size_t)(kBlk * HD)) + lane;
#pragma unroll
        for (int i = 0; i < RUNS; i++) kr[i] = p[i * 64];
    };
    auto load_v = [&](int b) __attribute__((always_inline)) {
        const size_t cell = cell_of(b);
        const uint4* p = reinterpret_cast<const uint4*>(a.vt + cell * (size_t)(kBlk * HD)) + lane;
#pragma unroll
        for (int i = 0; i < RUNS; i++) vr[i] = p[i * 64];
    };
    int b = bs + w;
    if (b < be) {
        load_k(b);
        load_v(b);
        ksc = a.ks[cell_of(b)];
        vsc = a.vs[cell_of(b)];
    }
    while (b < be) {
        const int next = b + kAttn8Waves;
        float ksn = 0.0f, vsn = 0.0f;
        if (next < be) {
            ksn = a.ks[cell_of(next)];
            vsn = a.vs[cell_of(next)];
        }
        if (!(ksc < 0.0f)) {
            block_step(
                b, ksc, vsc, [&](int t, int k) { return operand<FMT>(kr[t * (HD / 64) + (k >> 1)], k & 1); },
                [&](int d, int h) { return operand<FMT>(vr[d], h); }, 0u,
                [&]() {
                    if (next < be) load_k(next);
                });
        } else {
            // the open block: fp16 runs in the same order; positions past the
            // item's last one hold nothing yet, and what is not finite in V
            // goes by its positions' p
            const size_t ob = ((size_t)sp.seq * a.g.n_kv + kvh) * (size_t)(kBlk * HD);
            const half8* ko = reinterpret_cast<const half8*>(a.ko + ob) + lane * 2;
            const half8* vo = reinterpret_cast<const half8*>(a.vo + ob) + lane * 2;
            uint32_t bad = 0;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint16_t x = __builtin_bit_cast(uint16_t, (_Float16)vo[d * 128 + h][e]);
                        if ((x & 0x7c00) == 0x7c00) bad |= 1u << ((h * 2 + (e >> 2)) * 4 + (e & 3));
                    }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) bad |= (uint32_t)__shfl_xor((int)bad, x, 64);
            block_step(
                b, 1.0f, 1.0f, [&](int t, int k) { return ko[(t * (HD / 64) + (k >> 1)) * 128 + (k & 1)]; },
                [&](int d, int h) {
                    half8 x = vo[d * 128 + h];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint16_t y = __builtin_bit_cast(uint16_t, (_Float16)x[e]);
                        x[e] = (y & 0x7c00) == 0x7c00 ? (_Float16)0.0f : x[e];
                    }
                    return x;
                },
                bad,
                [&]() {
                    if (next < be) load_k(next);
                });
        }
        if (next < be) load_v(next);
        ksc = ksn;
        vsc = vsn;
        b = next;
    }

    // the waves' rows meet: one maximum, the sums scaled to it
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] += __shfl_xor(l[n], 16, 64);
        l[n] += __shfl_xor(l[n], 32, 64);
        if (g == 0) {
            sm[w][n * 16 + r16] = m[n];
            sl[w][n * 16 + r16] = l[n];
        }
    }
    __syncthreads();
    float big[NT], sum[NT], mine[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float t = sm[0][n * 16 + r16];
#pragma unroll
        for (int v = 1; v < kAttn8Waves; v++) t = fmaxf(t, sm[v][n * 16 + r16]);
        big[n] = t;
        const float safe = t == -INFINITY ? 0.0f : t;
        sum[n] = 0.0f;
#pragma unroll
        for (int v = 0; v < kAttn8Waves; v++)
            sum[n] += sl[v][n * 16 + r16] * __builtin_amdgcn_exp2f(sm[v][n * 16 + r16] - safe);
        mine[n] = __builtin_amdgcn_exp2f(m[n] - safe);
    }
    const bool whole = sh.splits == 1;
    constexpr int kPartWords = R * HD + 2 * R;
    float* part = whole ? nullptr : a.part + ((size_t)(sh.slot0 + sh.split) * a.g.n_kv + kvh) * kPartWords;

    // rows n * 16 + r16, dimensions 16 d + 4 g .. of the item to out
    auto put = [&](int n, int d, floatx4 x, float total) __attribute__((always_inline)) {
        const int row = n * 16 + r16;
        if (row >= sp.n_rows) return;
        const int rr = sp.first_row + row, t = rr / a.rep, head = kvh * a.rep + rr - t * a.rep;
        const size_t at = (qrow0 + t) * a.out_stride + (size_t)head * HD + d * 16 + g * 4;
        // nothing seen: zeros
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = total == 0.0f ? 0.0f : x[i] / total;
        if (SPLIT) store_row4<float>(a.out, at, x);
        else if (a.type == IAM_F16) store_row4<_Float16>(a.out, at, x);
        else store_row4<__bf16>(a.out, at, x);
    };
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += DC) {
        if (d0) __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int d = 0; d < DC; d++) meet[w][n * DC + d][lane] = o[n][d0 + d] * mine[n];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NT * DC / kAttn8Waves; u++) {
            const int nd = u * kAttn8Waves + w, n = nd / DC, d = d0 + nd % DC;
            floatx4 x = meet[0][nd][lane];
#pragma unroll
            for (int v = 1; v < kAttn8Waves; v++) x += meet[v][nd][lane];
            float tot = sum[0];
#pragma unroll
            for (int q = 1; q < NT; q++) tot = n == q ? sum[q] : tot;
            if (whole) put(n, d, x, tot);
            else put4(part + ((n * DT + d) * 64 + lane) * 4, x);
        }
    }
    if (whole) return;
    if (w == 0 && g == 0)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            acc_put(part + R * HD + n * 16 + r16, big[n]);
            acc_put(part + R * HD + R + n * 16 + r16, sum[n]);
        }
    // the last of the item's workgroups to arrive joins their results
    uint32_t* ctr = a.ctr + (size_t)sh.item * a.g.n_kv + kvh;
    if (!acc_arrive(ctr, (uint32_t)sh.splits, &s_last)) return;
    float* parts = a.part + ((size_t)sh.slot0 * a.g.n_kv + kvh) * kPartWords;
    const size_t step = (size_t)a.g.n_kv * kPartWords;
#pragma unroll 1
    for (int nd = w; nd < NT * DT; nd += kAttn8Waves) {
        const int n = nd / DT, row = n * 16 + r16;
        float t = -INFINITY;
        for (int k = 0; k < sh.splits; k++) t = fmaxf(t, acc_peek(parts + k * step + R * HD + row));
        const float safe = t == -INFINITY ? 0.0f : t;
        float tot = 0.0f;
        floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < sh.splits; k++) {
            const float f = __builtin_amdgcn_exp2f(acc_peek(parts + k * step + R * HD + row) - safe);
            tot += acc_peek(parts + k * step + R * HD + R + row) * f;
            x += peek4(parts + k * step + (nd * 64 + lane) * 4) * f;
        }
        put(n, nd - n * DT, x, tot);
    }
    if (tid == 0) *ctr = 0u;
}

// ------------------------------------------------------------------ host ---
constexpr int kTargetGroups = 512;     // workgroups that fill the card: two on each of 256 CUs
constexpr int kMaxPlanned = 4096;      // items * n_kv up to which the context is split

template <int HD, int FMT, bool SPLIT, int NT>
static int attn8_launch(Ctx* c, Attn8Args a)
{
    constexpr int R = 16 * NT;
    a.groups = (int)(((int64_t)a.rows + R - 1) / R);
    const int64_t items = (int64_t)a.groups * a.g.n_seq;
    IAM_REQUIRE(items * a.g.n_kv < ((int64_t)1 << 31), "attention_kv8: too many rows");
    a.items = (int)items;
    a.target = (kTargetGroups + a.g.n_kv - 1) / a.g.n_kv;
    const int most = (kv8_blocks(a.g.max_ctx) + kAttn8Waves - 1) / kAttn8Waves;   // workgroups an item can use
    a.planned = items * a.g.n_kv <= kMaxPlanned && most > 1;
    int64_t per_head = items;
    if (a.planned) {
        per_head = std::min<int64_t>(a.target + items, items * most);
        // split items share at most 2 * target slots: each takes fewer than twice nb / G
        const size_t slots = (size_t)std::min<int64_t>(2 * (int64_t)a.target, items * most) * a.g.n_kv;
        IAM_TRY(ensure_kv8_scratch(c, slots * (R * HD + 2 * R), (size_t)items * a.g.n_kv));
        a.part = c->kv8_part;
        a.ctr = c->kv8_ctr;
    }
    const dim3 grid((unsigned)(per_head * a.g.n_kv));
    return launch(c, "kv8_attention", k_kv8_attn<HD, FMT, SPLIT, NT>, grid, dim3(kAttn8Threads), 0, a);
}

template <int HD, int FMT, bool SPLIT>
static int attn8_rows(Ctx* c, const Attn8Args& a)
{
    return a.rows <= 16 ? attn8_launch<HD, FMT, SPLIT, 1>(c, a) : attn8_launch<HD, FMT, SPLIT, 2>(c, a);
}

template <int HD>
static int attn8_dim(Ctx* c, const Attn8Args& a, int format)
{
    if (format == IAM_KV8_INT8)
        return a.type == IAM_F32 ? attn8_rows<HD, IAM_KV8_INT8, true>(c, a) : attn8_rows<HD, IAM_KV8_INT8, false>(c, a);
    return a.type == IAM_F32 ? attn8_rows<HD, IAM_KV8_E4M3, true>(c, a) : attn8_rows<HD, IAM_KV8_E4M3, false>(c, a);
}

}  // namespace iam

using namespace iam;

extern "C" int iam_attention_kv8(iam_ctx* c, const iam_kv8_cache* k, const void* q, int type, int n_heads, int n_tokens,
                                 size_t q_stride, const int* pos, const int* count, int window, float scale, void* out,
                                 size_t out_stride)
{
    if (!c || !k || !q || !pos || !out) return fail(IAM_E_INVALID, "attention_kv8: null argument");
    IAM_TRY(kv8_check(c, k, "attention_kv8"));
    IAM_REQUIRE(type == IAM_F32 || type == IAM_F16 || type == IAM_BF16, "attention_kv8: unknown type");
    IAM_REQUIRE(n_heads >= k->n_kv && n_heads <= 65536 && n_heads % k->n_kv == 0,
                "attention_kv8: n_heads must be a multiple of n_kv, at most 65536");
    IAM_REQUIRE(n_tokens >= 0 && (int64_t)n_tokens * (n_heads / k->n_kv) < ((int64_t)1 << 30),
                "attention_kv8: n_tokens must not be negative, n_tokens * n_heads / n_kv below 2^30");
    IAM_REQUIRE(window >= 0, "attention_kv8: the window must not be negative");
    IAM_REQUIRE(std::isfinite(scale) && scale >= 0.0f, "attention_kv8: the scale must be finite and not negative");
    const size_t width = (size_t)n_heads * k->head_dim, B = type_bytes(type);
    if (!q_stride) q_stride = width;
    if (!out_stride) out_stride = width;
    IAM_REQUIRE(q_stride >= width && out_stride >= width && q_stride < ((size_t)1 << 31) && out_stride < ((size_t)1 << 31),
                "attention_kv8: a stride must hold a row and be below 2^31");
    IAM_REQUIRE(aligned(q, B) && aligned(out, B) && aligned(pos, 4) && aligned(count, 4),
                "attention_kv8: q and out must be aligned to their type");
    if (n_tokens == 0) return IAM_OK;
    const size_t rows = (size_t)k->n_seq * n_tokens;
    const size_t qb = rows_bytes(rows, width, q_stride, B), ob = rows_bytes(rows, width, out_stride, B);
    IAM_TRY(check_dev_range(c, q, qb, "attention_kv8 q"));
    IAM_TRY(check_dev_range(c, out, ob, "attention_kv8 out"));
    IAM_TRY(check_dev_range(c, pos, (size_t)k->n_seq * 4, "attention_kv8 pos"));
    if (count) IAM_TRY(check_dev_range(c, count, (size_t)k->n_seq * 4, "attention_kv8 count"));
    IAM_REQUIRE((q == out && q_stride == out_stride) || !overlaps(q, qb, out, ob),
                "attention_kv8: q and out overlap without being the same rows");
    IAM_REQUIRE(!kv8_overlaps(k, out, ob) && !overlaps(pos, (size_t)k->n_seq * 4, out, ob) &&
                    !(count && overlaps(count, (size_t)k->n_seq * 4, out, ob)),
                "attention_kv8: out overlaps the cache, the positions or the counts");
    DeviceGuard on(c);
    Attn8Args a{};
    a.q = q;
    a.out = out;
    a.kt = k->k;
    a.vt = k->v;
    a.ks = k->k_scale;
    a.vs = k->v_scale;
    a.ko = k->k_open;
    a.vo = k->v_open;
    a.pos = pos;
    a.count = count;
    a.g = {k->n_seq, k->max_ctx, k->n_kv, kv8_blocks(k->max_ctx)};
    a.type = type;
    a.heads = n_heads;
    a.rep = n_heads / k->n_kv;
    a.tokens = n_tokens;
    a.rows = n_tokens * a.rep;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.window = window;
    a.scale_log2 = (float)((scale > 0.0f ? (double)scale : 1.0 / std::sqrt((double)k->head_dim)) * 1.4426950408889634);
    if (k->head_dim == 64) return attn8_dim<64>(c, a, k->format);
    if (k->head_dim == 128) return attn8_dim<128>(c, a, k->format);
    return attn8_dim<256>(c, a, k->format);
}
