// What the kernels of the attention over the 8-bit KV cache share: arguments,
// the dealing out of the work, operands and results.
//
// With q' = q * scale * log2(e), one KV head's rows of queries r (its n_heads /
// n_kv query heads of each token) and positions t:
//   s[t][r] = (k8[t] . q'[r]) * k_scale[block of t],  hidden positions -inf
//   p = 2^(s - m),  l[r] = sum p,  o[r] = sum over blocks v_scale * (sum p v8[t]),
// in one pass with the running maximum m[r] of the rows, o / l at the end.
#pragma once

#include "accum.h"
#include "kv8.h"
#include "wave.h"

namespace iam {

// A wave takes blocks of 64 positions for 16 rows at a time, K and V in the
// order of the matrix instructions (16x16x32 in fp16, fp32 sums; 8-bit numbers
// are exact in fp16):
//   S^T = K Q^T  A: 16 positions of K, B: 16 query rows; lane (g, r) then
//                holds positions 4 g .. 4 g + 3 of each 16 for row r
//   O^T = V^T P^T  A: 16 dimensions of V, its 32 positions in the order in
//                which B, the lane's own p, has them: p goes from the
//                softmax's registers into the product without moving lanes.
// Rows are in lanes (r), so the rescaling by 2^(m - m') is one factor a lane.
// Precision: q and p are fp32; each is split into two fp16 parts, high and
// low (22 bits of q, 21 of p), after a power of two that brings them near the
// top of fp16's range, and both are multiplied (an fp16 or bf16 q needs one
// part).
constexpr int kAttn8Threads = 256, kAttn8Waves = 4;
constexpr int kAlone = 2 * kAttn8Waves;   // blocks that one workgroup takes by itself: joining costs 4 us
constexpr int kMinBlocks = 8;         // blocks of a workgroup where an item is split,
constexpr int kFewParts = 16;         // or 4 while that makes no more parts than these (read in one go when joined)
constexpr int kPartsOver = 2;        // many rows: blocks that a part may be over an even share
constexpr int kMaxItems = 2048;       // items up to which they are dealt out by length
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
    int rep;                 // query heads of a KV head
    int tokens, rows;        // of a sequence; rows = tokens * rep
    int groups;              // row groups of a sequence
    int items;               // n_seq * groups
    int planned;             // blocks dealt out by length (else one workgroup an item and KV head)
    int target;              // planned: workgroups per KV head
    size_t q_stride, out_stride;
    int window;
    float scale_log2;
    float* part;             // partial results of the split items
    uint32_t* ctr;           // [(items + upper) * n_kv] arrivals, zero on entry (left zero)
    int upper;               // slots of partial results; the results of groups of them lie behind
    int4* joins;             // [items] many rows: parts of an item and where they are
};

struct Span {
    int seq, first_row, n_rows;   // rows of the item that are there
    int b0, nb;                   // blocks they see
    int p0;
};

// the token of row `row` of a sequence (no division for single tokens)
__device__ __forceinline__ int token_of(const Attn8Args& a, int row) { return a.tokens == 1 ? 0 : row / a.rep; }

// what item `it` has to read
__device__ __forceinline__ Span span_of(const Attn8Args& a, int it, int rows_per_item)
{
    Span s;
    s.seq = a.groups == 1 ? it : it / a.groups;
    s.first_row = (it - s.seq * a.groups) * rows_per_item;
    s.p0 = a.pos[s.seq];
    const int n = a.count ? min(a.tokens, a.count[s.seq]) : a.tokens;
    s.n_rows = max(0, min(s.first_row + rows_per_item, n * a.rep) - s.first_row);
    s.b0 = s.nb = 0;
    if (s.n_rows > 0 && s.p0 >= 0) {
        const int top = a.g.max_ctx - 1;
        const int t0 = token_of(a, s.first_row), t1 = token_of(a, s.first_row + s.n_rows - 1);
        const int hi = s.p0 > top - t1 ? top : s.p0 + t1, lo_p = s.p0 > top - t0 ? top : s.p0 + t0;
        const int lo = a.window > 0 ? max(0, lo_p - a.window + 1) : 0;
        s.b0 = lo / kBlk;
        s.nb = hi / kBlk - s.b0 + 1;
    }
    return s;
}

template <int WAVES>
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
    for (int i = 0; i < WAVES; i++) {
        before += i < w ? wsum[i] : 0;
        total += wsum[i];
    }
    return before + incl - v;
}

// A part of an item: of the blocks it reads, four (one a wave) from `from` on,
// then every `stride`-th, below `to`.  Split items leave `splits` partial
// results; part k of them is in slot (k ? base + k * step : first).
struct Share {
    int item, from, to, stride, splits;
    int slot, first, base, step;
};

// How the work is dealt out to the `target` workgroups of a KV head that the
// card holds at once, from the positions on the device; every workgroup
// finds its own share.  Few items, or little work: an item of n blocks is dealt
// to ceil(n / G) workgroups, four blocks at a time in turn (so that they read
// one window of the cache at any time), up to kAlone blocks to one.  Else
// the items' blocks are taken as one row and cut into `target` even pieces; a
// workgroup goes through the (parts of) items in its own.
struct Deal {
    int mode;             // 0: one part a workgroup; 1: a piece of the row
    int lo, hi;           // mode 1: this workgroup's piece
    int per, last;        // mode 1: blocks of a piece; whether it is the last one
    Share one;            // mode 0
    int item;             // mode 1: the next item
};

__device__ __forceinline__ int up_div(int x, int y) { return (int)((unsigned)(x + y - 1) / (unsigned)y); }
// G: kAttn8Waves where the card has workgroups to spare, else kMinBlocks or more
__device__ __forceinline__ int parts_of(int nb, int G)
{
    if (nb <= kAlone) return 1;
    return G > kAttn8Waves ? up_div(nb, G) : min(up_div(nb, kAttn8Waves), max(kFewParts, up_div(nb, kMinBlocks)));
}

// pre: LDS [items + 1], the items' blocks before each; least: 0, or mode 1 with
// pieces of at least so many blocks; false: no work
template <int WAVES = kAttn8Waves>
__device__ __forceinline__ bool find_deal(const Attn8Args& a, int j, int rows_per_item, int* pre, Deal& d, int least = 0)
{
    __shared__ int wsum[WAVES];
    __shared__ Share found;
    const int tid = threadIdx.x;
    const int per = (a.items + 64 * WAVES - 1) / (64 * WAVES);
    const int i0 = tid * per, i1 = min(a.items, i0 + per);
    int total;
    if (a.items == 1) {
        total = span_of(a, 0, rows_per_item).nb;
    } else {
        int mine = 0;
        for (int i = i0; i < i1; i++) mine += span_of(a, i, rows_per_item).nb;
        int at = block_sum_scan<WAVES>(mine, wsum, total);
        for (int i = i0; i < i1; i++) {
            pre[i] = at;
            at += span_of(a, i, rows_per_item).nb;
        }
        if (tid == 0) pre[a.items] = total;
        __syncthreads();
    }
    const int spare = a.target - a.items;
    const int need = spare > 0 ? up_div(total, spare) : 0;   // with parts of this many blocks all fit
    const int G = need <= kAttn8Waves ? kAttn8Waves : max(kMinBlocks, need);
    d.mode = least == 0 && spare > 0 && (G <= 2 * kMinBlocks || a.items <= a.target / 8) ? 0 : 1;
    if (d.mode == 0 && a.items == 1) {
        const int n = parts_of(total, G);
        if (j >= n) return false;
        d.one = {0, j * kAttn8Waves, total, n * kAttn8Waves, n, j, 0, 0, 1};
        return true;
    }
    if (d.mode == 0) {
        int ws = 0, slots = 0, all, all_slots;
        for (int i = i0; i < i1; i++) {
            const int n = parts_of(pre[i + 1] - pre[i], G);
            ws += n;
            slots += n > 1 ? n : 0;
        }
        int w0 = block_sum_scan<WAVES>(ws, wsum, all), s0 = block_sum_scan<WAVES>(slots, wsum, all_slots);
        if (j >= all) return false;
        if (j >= w0 && j < w0 + ws)
            for (int i = i0; i < i1; i++) {
                const int nb = pre[i + 1] - pre[i], n = parts_of(nb, G), k = j - w0;
                if (k < n) {
                    found = {i, k * kAttn8Waves, nb, n * kAttn8Waves, n, s0 + k, s0, s0, 1};
                    break;
                }
                w0 += n;
                s0 += n > 1 ? n : 0;
            }
        __syncthreads();
        d.one = found;
        return true;
    }
    if (a.items == 1) {
        if (tid < 2) pre[tid] = tid ? total : 0;
        __syncthreads();
    }
    d.per = max(max(1, least), up_div(total, a.target));
    // Many rows: parts of up to per, per + 1 .. blocks, if the workgroups are
    // enough for them.  An even cut of the row of blocks gives most workgroups
    // two items, with the rows' operands and results of both (500 tokens
    // behind 3600: fp32 88 us, bf16 81; by parts 80 and 73).
#pragma unroll 1
    for (int G = d.per; least && G <= d.per + kPartsOver; G++) {
        int ws = 0, slots = 0, all, all_slots;
#pragma unroll 1
        for (int i = i0; i < i1; i++) {
            const int n = max(1, up_div(pre[i + 1] - pre[i], G));
            ws += n;
            slots += n > 1 ? n : 0;
        }
        int w0 = block_sum_scan<WAVES>(ws, wsum, all);
        if (all > a.target) continue;
        int s0 = block_sum_scan<WAVES>(slots, wsum, all_slots);
        if (j >= all) return false;
        if (j >= w0 && j < w0 + ws)
            for (int i = i0; i < i1; i++) {
                const int nb = pre[i + 1] - pre[i], n = max(1, up_div(nb, G)), k = j - w0;
                if (k < n) {
                    const int q = nb / n, r = nb - q * n;   // the first r parts have q + 1
                    found = {i, k * q + min(k, r), (k + 1) * q + min(k + 1, r), 1, n, s0 + k, s0, s0, 1};
                    break;
                }
                w0 += n;
                s0 += n > 1 ? n : 0;
            }
        __syncthreads();
        d.mode = 0;
        d.one = found;
        return true;
    }
    d.lo = j * d.per;
    if (j > 0 && d.lo >= total) return false;
    d.last = total - d.lo <= d.per;
    d.hi = d.last ? total : d.lo + d.per;
    // the first item that ends past lo, or (of no blocks) lies at it
    int x = 0, y = a.items;
    while (x < y) {
        const int m = (x + y) >> 1;
        if (pre[m + 1] > d.lo || pre[m] >= d.lo) y = m;
        else x = m + 1;
    }
    d.item = x;
    return true;
}

// mode 1: the workgroup's part of item d.item, and on to the next; false: done
__device__ __forceinline__ bool next_share(const Attn8Args& a, const int* pre, int j, Deal& d, Share& s)
{
    const int i = d.item;
    if (i >= a.items) return false;
    const int p0 = pre[i], p1 = pre[i + 1];
    if (p0 >= d.hi && !d.last) return false;     // the next piece's
    d.item = i + 1;
    s.item = i;
    s.stride = kAttn8Waves;
    s.from = s.to = 0;
    s.splits = 1;
    if (p0 == p1) return true;                   // of no blocks: its rows are zeros
    s.from = max(d.lo - p0, 0);
    s.to = min(d.hi, p1) - p0;
    const int j0 = p0 / d.per, j1 = (p1 - 1) / d.per;
    s.splits = j1 - j0 + 1;
    s.step = 2;
    s.base = 2 * j0;
    s.first = 2 * j0 + (j0 * d.per < p0 ? 1 : 0);
    s.slot = j == j0 ? s.first : 2 * j;
    return true;
}

// 8 numbers of a tile's run (half 0 or 1) as an operand
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <int FMT>
__device__ __forceinline__ half8 operand(const u32x4& w, int h)
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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Two probabilities' high parts (towards zero) and what is left of them, in
// fp16: 21 bits together.
__device__ __forceinline__ void split2(float p0, float p1, half2v& high, half2v& low)
{
    high = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    low = half2v{(_Float16)__builtin_fmaf((float)high[0], -1.0f, p0), (_Float16)__builtin_fmaf((float)high[1], -1.0f, p1)};
}

// over the four lanes that hold one row (r16, r16 + 16, ...), in each of them
template <typename Op>
__device__ __forceinline__ float over_row(float v, Op op)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_max(float v)
{
    return over_row(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float row_sum(float v)
{
    return over_row(v, [](float x, float y) { return x + y; });
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
typedef unsigned long long ull2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put4(float* p, floatx4 v)
{
    const ull2 u = __builtin_bit_cast(ull2, v);
    acc_put(reinterpret_cast<unsigned long long*>(p), u[0]);
    acc_put(reinterpret_cast<unsigned long long*>(p) + 1, u[1]);
}
__device__ __forceinline__ floatx4 peek4(float* p)
{
    ull2 u;
    u[0] = acc_peek(reinterpret_cast<unsigned long long*>(p));
    u[1] = acc_peek(reinterpret_cast<unsigned long long*>(p) + 1);
    return __builtin_bit_cast(floatx4, u);
}

// what the rows of an item see: every row there [lo_all, hi_all], any [.., hi_max]
struct Sees {
    int hi_all, hi_max, lo_all;
};
__device__ __forceinline__ Sees sees_of(const Attn8Args& a, const Span& sp)
{
    const int top = a.g.max_ctx - 1;
    const int t0 = token_of(a, sp.first_row), t1 = token_of(a, sp.first_row + sp.n_rows - 1);
    Sees s;
    s.hi_all = sp.p0 > top - t0 ? top : sp.p0 + t0;
    s.hi_max = sp.p0 > top - t1 ? top : sp.p0 + t1;
    s.lo_all = a.window > 0 ? max(0, s.hi_max - a.window + 1) : 0;
    return s;
}

// One row of queries of an item as operands of the KS instructions: lane (g,
// r16) has row `row`, of instruction k the dimensions 64 (k/2) + 16 g + 8 (k%2)
// and on.
template <int HD, bool SPLIT>
struct Query {
    static constexpr int KS = HD / 32;
    float v[KS][8];
    int hi, lo;        // positions the row sees (none there: -1)

    __device__ __forceinline__ void load(const Attn8Args& a, const Span& sp, int kvh, int row, int g)
    {
        const bool there = row < sp.n_rows;
        const int rr = sp.first_row + row, top = a.g.max_ctx - 1;
        const int t = there ? token_of(a, rr) : 0, head = kvh * a.rep + (there ? rr - t * a.rep : 0);
        hi = there && sp.p0 >= 0 ? (sp.p0 > top - t ? top : sp.p0 + t) : -1;
        lo = a.window > 0 ? max(0, hi - a.window + 1) : 0;
        const size_t at = ((size_t)sp.seq * a.tokens + t) * a.q_stride + (size_t)head * HD;
#pragma unroll
        for (int k = 0; k < KS; k++) {
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
        }
    }
    // the operands' parts; the factor that takes the products to log2 units: NaN
    // where a value is infinite, as scores that are all -inf would else be a
    // row that sees nothing
    __device__ __forceinline__ float split(const Attn8Args& a, half8* high, half8* low)
    {
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(v[k][e]));
        top = row_max(top);
        // the power of two that brings the row's largest value into [2^9, 2^10)
        int ex = 10;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &ex);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = ldexpf(v[k][e], 10 - ex);
                const _Float16 h = (_Float16)x;
                high[k][e] = h;
                if constexpr (SPLIT) low[k][e] = (_Float16)(x - (float)h);
            }
        return top < INFINITY ? ldexpf(a.scale_log2, ex - 10) : NAN;
    }
};

// four values of row `row` of an item, from dimension d on, to out
template <int HD, bool SPLIT>
__device__ __forceinline__ void put_row(const Attn8Args& a, const Span& sp, int kvh, int row, int d, floatx4 x, float total)
{
    const int rr = sp.first_row + row, t = token_of(a, rr), head = kvh * a.rep + rr - t * a.rep;
    const size_t at = ((size_t)sp.seq * a.tokens + t) * a.out_stride + (size_t)head * HD + d;
    // nothing seen: zeros
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = total == 0.0f ? 0.0f : x[i] / total;
    if (SPLIT) store_row4<float>(a.out, at, x);
    else if (a.type == IAM_F16) store_row4<_Float16>(a.out, at, x);
    else store_row4<__bf16>(a.out, at, x);
}

// ------------------------------------------------------------------ host ---
// workgroups that the card holds at once
template <typename Kernel>
int attn8_resident(Kernel k, int threads)
{
    int per_cu = 0, dev = 0, cus = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, k, threads, 0) != hipSuccess ||
        hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        return 256;
    return std::max(per_cu, 1) * std::max(cus, 1);
}
// many rows (a prompt's chunk)
int attn8_rows(Ctx* c, const Attn8Args& a, int head_dim, int format);

}  // namespace iam
