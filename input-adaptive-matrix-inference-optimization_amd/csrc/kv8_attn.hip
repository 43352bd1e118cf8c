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

// A wave takes blocks of 64 positions, each 2 * 64 * head_dim bytes in the
// order of the matrix instructions (16x16x32 in fp16, fp32 sums; 8-bit numbers
// are exact in fp16):
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
constexpr int kAlone = 2 * kAttn8Waves;   // blocks that one workgroup takes by itself: joining costs 4 us
constexpr int kMinBlocks = 8;         // blocks of a workgroup where an item is split,
constexpr int kFewParts = 16;         // or 4 while that makes no more parts than these (read in one go when joined)
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
    int heads, rep;          // query heads; of them per KV head
    int tokens, rows;        // of a sequence; rows = tokens * rep
    int groups;              // row groups of a sequence
    int items;               // n_seq * groups
    int planned;             // blocks dealt out by length (else one workgroup an item and KV head)
    int target;              // planned: workgroups per KV head
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

// pre: LDS [items + 1], the items' blocks before each; false: no work
__device__ __forceinline__ bool find_deal(const Attn8Args& a, int j, int rows_per_item, int* pre, Deal& d)
{
    __shared__ int wsum[kAttn8Waves];
    __shared__ Share found;
    const int tid = threadIdx.x;
    const int per = (a.items + kAttn8Threads - 1) / kAttn8Threads;
    const int i0 = tid * per, i1 = min(a.items, i0 + per);
    int total;
    if (a.items == 1) {
        total = span_of(a, 0, rows_per_item).nb;
    } else {
        int mine = 0;
        for (int i = i0; i < i1; i++) mine += span_of(a, i, rows_per_item).nb;
        int at = block_sum_scan(mine, wsum, total);
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
    d.mode = spare > 0 && (G <= 2 * kMinBlocks || a.items <= a.target / 8) ? 0 : 1;
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
        int w0 = block_sum_scan(ws, wsum, all), s0 = block_sum_scan(slots, wsum, all_slots);
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
    d.per = max(1, up_div(total, a.target));
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

// A tile of RUNS * 1024 bytes from memory into the wave's own part of LDS, 16
// bytes a lane and instruction, without registers.  ONCE: past the caches'
// reuse (a tile that one workgroup reads): 42 us against 45 for a plain read
// of the 268 MB that 131000 tokens take.
template <int RUNS, bool ONCE>
__device__ __forceinline__ void fetch_tile(const uint8_t* src, char* lds)
{
    const uint8_t* p = src + (threadIdx.x & 63) * 16;
#pragma unroll
    for (int i = 0; i < RUNS; i++)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p + i * 1024),
                                         (__attribute__((address_space(3))) void*)(lds + i * 1024), 16, 0, ONCE ? 2 : 0);
}

// Four runs (i = 0 .. 3) of a tile in LDS into registers, once all but the
// wave's last YOUNGER vector memory instructions are done.  In one piece of
// assembly with its waits: the compiler, which cannot tell the tiles apart,
// would wait for every fetch in flight before any read.
template <int YOUNGER>
__device__ __forceinline__ void read_runs(uint32_t at, u32x4* r)
{
    asm volatile(
        "s_waitcnt vmcnt(%5)\n\t"
        "ds_read_b128 %0, %4\n\t"
        "ds_read_b128 %1, %4 offset:1024\n\t"
        "ds_read_b128 %2, %4 offset:2048\n\t"
        "ds_read_b128 %3, %4 offset:3072\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(at), "n"(YOUNGER)
        : "memory");
}
// the whole tile; `more`: a younger tile of RUNS instructions is in flight
template <int RUNS>
__device__ __forceinline__ void read_tile(uint32_t at, bool more, u32x4* r)
{
    if (more) read_runs<RUNS>(at, r);
    else read_runs<0>(at, r);
#pragma unroll
    for (int i = 4; i < RUNS; i += 4) read_runs<63>(at + i * 1024, r + i);
}

// SPLIT: q is fp32, in two parts.  NT: tiles of 16 query rows an item has.
// A wave's K and V tiles come through its own two places in LDS: a tile is
// read into registers as soon as it is there and its place fetched again at
// once, so that a block is in flight at any time whatever the arithmetic
// does (and no wave waits for another).  Bound by memory for single tokens.
template <int HD, int FMT, bool SPLIT, int NT>
__global__ __launch_bounds__(kAttn8Threads, HD * NT <= 128 ? 2 : 1) void k_kv8_attn(Attn8Args a)
{
    constexpr int KS = HD / 32, DT = HD / 16, R = 16 * NT;
    constexpr int RUNS = HD / 16, TILE = kBlk * HD;  // 16-byte runs of a tile per lane; its bytes
    constexpr int DC = NT * DT <= 8 ? DT : 8 / NT;   // dimension tiles the waves' sums meet in at a time
    constexpr int kPartWords = R * HD + 2 * R;       // a partial result: o of the rows there, m, l
    constexpr int PARTS = SPLIT ? 2 : 1;             // fp16 parts of q
    constexpr int MEET = kAttn8Waves * NT * DC * 64 * 16, RING = kAttn8Waves * 2 * TILE;
    static_assert(MEET >= kAttn8Threads * 24, "the joining sums fit");
    __shared__ __align__(1024) char lds[MEET > RING ? MEET : RING];
    __shared__ float sm[kAttn8Waves][R], sl[kAttn8Waves][R];
    __shared__ int pre[kMaxItems + 1];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r16 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.g.n_kv, j = blockIdx.x / a.g.n_kv;
    char* const place_k = lds + w * 2 * TILE;
    char* const place_v = place_k + TILE;
    const uint32_t at_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)place_k + lane * 16;
    const uint32_t at_v = at_k + TILE;
    floatx4(*const meet)[NT * DC][64] = reinterpret_cast<floatx4(*)[NT * DC][64]>(lds);
    Deal deal{};
    Share sh{};
    if (a.planned) {
        if (!find_deal(a, j, R, pre, deal)) return;
        if (deal.mode == 0) sh = deal.one;
        else if (!next_share(a, pre, j, deal, sh)) return;
    } else {
        sh.item = a.items - 1 - j;   // the row groups with the longest contexts first
        sh.splits = 1;
        sh.to = 1 << 30;
        sh.stride = kAttn8Waves;
    }
    for (;;) {
        const Span sp = span_of(a, sh.item, R);
        const int bs = sp.b0 + sh.from, be = sp.b0 + min(sh.to, sp.nb);
        if (sp.n_rows > 0) {
            // positions that every row there sees: below lo_all and past hi_all a mask is needed
            const int top_ctx = a.g.max_ctx - 1;
            const int t_first = token_of(a, sp.first_row), t_last = token_of(a, sp.first_row + sp.n_rows - 1);
            const int hi_all = sp.p0 > top_ctx - t_first ? top_ctx : sp.p0 + t_first;
            const int hi_max = sp.p0 > top_ctx - t_last ? top_ctx : sp.p0 + t_last;
            const int lo_all = a.window > 0 ? max(0, hi_max - a.window + 1) : 0;
            auto cell_of = [&](int b) { return kv8_cell(a.g, sp.seq, b, kvh); };
            // Where the last position does not end its block, the block is
            // open, unless more tokens came since: its scale says so.  The
            // workgroup with the block before `be` among its fours takes it.
            const bool end_inside = be > bs && be == sp.b0 + sp.nb && (hi_max + 1) % kBlk != 0 &&
                                    (unsigned)(be - 1 - bs) % (unsigned)sh.stride < kAttn8Waves;
            const float end_scale = end_inside ? a.ks[cell_of(be - 1)] : 0.0f;

            // this lane's rows: positions they see, their queries
            int hi[NT], lo[NT];
            float mult[NT];
            half8 qh[PARTS][NT][KS];
            const size_t qrow0 = (size_t)sp.seq * a.tokens;
            float qv[NT][KS][8];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int row = sp.first_row + n * 16 + r16;
                const bool there = n * 16 + r16 < sp.n_rows;
                const int t = there ? token_of(a, row) : 0, head = kvh * a.rep + (there ? row - t * a.rep : 0);
                hi[n] = there && sp.p0 >= 0 ? (sp.p0 > top_ctx - t ? top_ctx : sp.p0 + t) : -1;
                lo[n] = a.window > 0 ? max(0, hi[n] - a.window + 1) : 0;
                const size_t at = (qrow0 + t) * a.q_stride + (size_t)head * HD;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    // instruction k of the dimensions 64 (k/2) + 16 g + 8 (k%2) ..
                    const size_t ad = at + (k >> 1) * 64 + g * 16 + (k & 1) * 8;
                    if (!there) {
#pragma unroll
                        for (int e = 0; e < 8; e++) qv[n][k][e] = 0.0f;
                    } else if (SPLIT) {
                        load_row8<float>(a.q, ad, qv[n][k]);
                    } else if (a.type == IAM_F16) {
                        load_row8<_Float16>(a.q, ad, qv[n][k]);
                    } else {
                        load_row8<__bf16>(a.q, ad, qv[n][k]);
                    }
                }
            }
            int b = bs + w;
            float ksc = 0.0f, vsc = 0.0f;   // the scales of block b
            if (b < be) {   // (an open block's bytes are not looked at)
                fetch_tile<RUNS, NT == 1>(a.kt + cell_of(b) * (size_t)TILE, place_k);
                fetch_tile<RUNS, NT == 1>(a.vt + cell_of(b) * (size_t)TILE, place_v);
                ksc = a.ks[cell_of(b)];
                vsc = a.vs[cell_of(b)];
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(qv[n][k][e]));
                top = row_max(top);
                // the power of two that brings the row's largest value into [2^9, 2^10)
                int ex = 10;
                if (top > 0.0f && top < INFINITY) (void)frexpf(top, &ex);
                mult[n] = ldexpf(a.scale_log2, ex - 10);
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float x = ldexpf(qv[n][k][e], 10 - ex);
                        const _Float16 h = (_Float16)x;
                        qh[0][n][k][e] = h;
                        if constexpr (SPLIT) qh[PARTS - 1][n][k][e] = (_Float16)(x - (float)h);
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

            // The open block, fp16 runs in the tiles' order: each wave takes
            // 16 of its positions.  Those past the item's last one hold
            // nothing yet; V's values that are not finite are taken out, and
            // go by their positions' s.
            const bool open_end = end_scale < 0.0f;
            if (open_end) {
                const size_t ob = ((size_t)sp.seq * a.g.n_kv + kvh) * (size_t)TILE;
                const half8* ko = reinterpret_cast<const half8*>(a.ko + ob) + lane * 2 + w * (HD / 64) * 128;
                const half8* vo = reinterpret_cast<const half8*>(a.vo + ob) + lane * 2 + (w >> 1);
                half8 kk[KS], vv[DT];
#pragma unroll
                for (int k = 0; k < KS; k++) kk[k] = ko[(k >> 1) * 128 + (k & 1)];
#pragma unroll
                for (int d = 0; d < DT; d++) vv[d] = vo[d * 128];
                const int at = (be - 1) * kBlk + w * 16 + g * 4;   // the lane's 4 positions:
                const bool upper = w & 1;                          // the second 4 of an operand's 8, or the first
                uint32_t bad = 0;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if ((__builtin_bit_cast(uint16_t, (_Float16)vv[d][e]) & 0x7c00) == 0x7c00) {
                            bad |= 1u << e;
                            vv[d][e] = (_Float16)0.0f;
                        }
#pragma unroll
                for (int x = 1; x < 16; x <<= 1) bad |= (uint32_t)__shfl_xor((int)bad, x, 64);
                bad = upper ? bad >> 4 : bad;
                half8 ph[NT], pl[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    floatx4 s = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int x = 0; x < PARTS; x++) s = mfma(kk[k], qh[x][n][k], s);
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s[i] = bad >> i & 1 ? NAN : s[i] * mult[n];
                        s[i] = at + i >= lo[n] && at + i <= hi[n] ? s[i] : -INFINITY;
                        top = fmaxf(top, s[i]);
                    }
                    top = row_max(top);
                    m[n] = top;
                    const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = exp2_fast(s[i] - safe + kProbShift);
                        l[n] += p;
                        const _Float16 h = (_Float16)p, r = (_Float16)(p - (float)h);
                        ph[n][i] = upper ? (_Float16)0.0f : h;
                        ph[n][4 + i] = upper ? h : (_Float16)0.0f;
                        pl[n][i] = upper ? (_Float16)0.0f : r;
                        pl[n][4 + i] = upper ? r : (_Float16)0.0f;
                    }
                }
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[n][d] = mfma(vv[d], ph[n], o[n][d]);
                        o[n][d] = mfma(vv[d], pl[n], o[n][d]);
                    }
            }

            const int bend = open_end ? be - 1 : be;
            while (b < bend) {
                const int next = b + sh.stride;
                const bool more = next < bend;
                const float kscale = ksc, vscale = vsc;
                if (more) {
                    ksc = a.ks[cell_of(next)];
                    vsc = a.vs[cell_of(next)];
                }
                u32x4 run[RUNS];
                read_tile<RUNS>(at_k, true, run);      // the V tile is younger
                if (more) fetch_tile<RUNS, NT == 1>(a.kt + cell_of(next) * (size_t)TILE, place_k);
                floatx4 s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int t = 0; t < 4; t++) s[n][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        const half8 ka = operand<FMT>(run[t * (HD / 64) + (k >> 1)], k & 1);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int x = 0; x < PARTS; x++) s[n][t] = mfma(ka, qh[x][n][k], s[n][t]);
                    }
                const bool edge = b * kBlk + kBlk - 1 > hi_all || b * kBlk < lo_all;
                half8 ph[NT][2], pl[NT][2];
                float alpha[NT], vsr[NT];
                bool grown = false;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float f = mult[n] * kscale;
                    vsr[n] = vscale;
                    uint32_t hidden = 0;   // a bit for each of the lane's 16 positions
                    if (edge) {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int p = b * kBlk + t * 16 + g * 4 + i;
                                if (p < lo[n] || p > hi[n]) {
                                    hidden |= 1u << (t * 4 + i);
                                    s[n][t][i] = -INFINITY;
                                }
                            }
                        // a block that the row does not see adds nothing, whatever its scale
                        if (b * kBlk > hi[n] || b * kBlk + kBlk - 1 < lo[n]) vsr[n] = 0.0f;
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) top = fmaxf(top, s[n][t][i]);
                    top = row_max(top);
                    // f is not negative: the scaled maximum is the maximum scaled
                    const float mn = fmaxf(m[n], top == -INFINITY ? top : top * f);
                    const float safe = mn == -INFINITY ? 0.0f : mn;
                    alpha[n] = exp2_fast(m[n] - safe);
                    grown |= mn != m[n];
                    m[n] = mn;
                    const float shift = kProbShift - safe;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[n][t][i] = exp2_fast(__builtin_fmaf(s[n][t][i], f, shift));
                    if (edge) {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (hidden >> (t * 4 + i) & 1) s[n][t][i] = 0.0f;   // also where f is 0 or NaN
                    }
                    float sum = 0.0f;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float p = s[n][t][i];
                            sum += p;
                            const _Float16 h = (_Float16)p;
                            ph[n][t >> 1][(t & 1) * 4 + i] = h;
                            pl[n][t >> 1][(t & 1) * 4 + i] = (_Float16)(p - (float)h);
                        }
                    l[n] = l[n] * alpha[n] + sum;
                }
                if (__any(grown)) {   // most blocks do not raise any row's maximum
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int d = 0; d < DT; d++) o[n][d] *= alpha[n];
                }
                read_tile<RUNS>(at_v, more, run);
                if (more) fetch_tile<RUNS, NT == 1>(a.vt + cell_of(next) * (size_t)TILE, place_v);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const half8 v0 = operand<FMT>(run[d], 0), v1 = operand<FMT>(run[d], 1);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                        x = mfma(v0, ph[n][0], x);
                        x = mfma(v1, ph[n][1], x);
                        x = mfma(v0, pl[n][0], x);
                        x = mfma(v1, pl[n][1], x);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[n][d][i] = __builtin_fmaf(x[i], vsr[n], o[n][d][i]);
                    }
                }
                b = next;
            }

            // the waves' rows meet: one maximum, the sums scaled to it (a
            // tile that was fetched for nothing has landed before LDS is used)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int n = 0; n < NT; n++) {
                l[n] = row_sum(l[n]);
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
                for (int v = 0; v < kAttn8Waves; v++) sum[n] += sl[v][n * 16 + r16] * exp2_fast(sm[v][n * 16 + r16] - safe);
                mine[n] = exp2_fast(m[n] - safe);
            }
            const bool whole = sh.splits == 1;
            const size_t step = (size_t)a.g.n_kv * kPartWords;
            float* part = whole ? nullptr : a.part + sh.slot * step + (size_t)kvh * kPartWords;

            // four values of row `row` of the item, from dimension d on, to out
            auto put = [&](int row, int d, floatx4 x, float total) __attribute__((always_inline)) {
                const int rr = sp.first_row + row, t = token_of(a, rr), head = kvh * a.rep + rr - t * a.rep;
                const size_t at = (qrow0 + t) * a.out_stride + (size_t)head * HD + d;
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
                    const int nd = u * kAttn8Waves + w, n = nd / DC, d = d0 + nd % DC, row = n * 16 + r16;
                    if (row >= sp.n_rows) continue;
                    floatx4 x = meet[0][nd][lane];
#pragma unroll
                    for (int v = 1; v < kAttn8Waves; v++) x += meet[v][nd][lane];
                    float tot = sum[0];
#pragma unroll
                    for (int q = 1; q < NT; q++) tot = n == q ? sum[q] : tot;
                    if (whole) put(row, d * 16 + g * 4, x, tot);
                    else put4(part + row * HD + d * 16 + g * 4, x);
                }
            }
            if (!whole) {
                if (w == 0 && g == 0)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        acc_put(part + R * HD + n * 16 + r16, big[n]);
                        acc_put(part + R * HD + R + n * 16 + r16, sum[n]);
                    }
                // The last of the item's workgroups to arrive joins their
                // results: thread (k0, four values e) takes every KP-th
                // one, 8 of their loads in flight, joined as blocks are; then
                // the KP sums meet.
                uint32_t* ctr = a.ctr + (size_t)sh.item * a.g.n_kv + kvh;
                if (acc_arrive(ctr, (uint32_t)sh.splits, &s_last)) {
                    constexpr int U = 8, Q = HD / 4;
                    float* parts = a.part + (size_t)kvh * kPartWords;
                    const int E = sp.n_rows * Q, KP = max(1, min(kAttn8Threads / E, sh.splits));
                    floatx4* jo = reinterpret_cast<floatx4*>(lds);
                    float* jml = reinterpret_cast<float*>(jo + kAttn8Threads);
                    for (int e0 = 0; e0 < E; e0 += kAttn8Threads) {
                        const int kp = KP > 1 ? tid / E : 0, e = KP > 1 ? tid - kp * E : e0 + tid;
                        const bool on = kp < KP && e < E;
                        const int row = on ? e / Q : 0;
                        float jm = -INFINITY, jl = 0.0f;
                        floatx4 jx = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (on)
                            for (int k0 = kp; k0 < sh.splits; k0 += U * KP) {
                                float pm[U], pl[U];
                                floatx4 px[U];
#pragma unroll
                                for (int u = 0; u < U; u++) {
                                    const int k = min(k0 + u * KP, sh.splits - 1);
                                    float* p = parts + (k ? sh.base + k * sh.step : sh.first) * step;
                                    pm[u] = acc_peek(p + R * HD + row);
                                    pl[u] = acc_peek(p + R * HD + R + row);
                                    px[u] = peek4(p + e * 4);
                                }
                                float t = jm;
#pragma unroll
                                for (int u = 0; u < U; u++) t = fmaxf(t, pm[u]);
                                const float safe = t == -INFINITY ? 0.0f : t, f0 = exp2_fast(jm - safe);
                                jm = t;
                                jl *= f0;
                                jx *= f0;
#pragma unroll
                                for (int u = 0; u < U; u++)
                                    if (k0 + u * KP < sh.splits) {
                                        const float f = exp2_fast(pm[u] - safe);
                                        jl += pl[u] * f;
                                        jx += px[u] * f;
                                    }
                            }
                        if (KP > 1) {
                            jo[tid] = jx;
                            jml[2 * tid] = jm;
                            jml[2 * tid + 1] = jl;
                            __syncthreads();
                            if (kp == 0 && on) {
                                float t = jm;
                                for (int k = 1; k < KP; k++) t = fmaxf(t, jml[2 * (tid + k * E)]);
                                const float safe = t == -INFINITY ? 0.0f : t, f0 = exp2_fast(jm - safe);
                                jl *= f0;
                                jx *= f0;
                                for (int k = 1; k < KP; k++) {
                                    const float f = exp2_fast(jml[2 * (tid + k * E)] - safe);
                                    jl += jml[2 * (tid + k * E) + 1] * f;
                                    jx += jo[tid + k * E] * f;
                                }
                            }
                        }
                        if (on && kp == 0) put(row, (e - row * Q) * 4, jx, jl);
                    }
                    if (tid == 0) *ctr = 0u;
                }
            }
        }
        if (!a.planned || deal.mode == 0 || !next_share(a, pre, j, deal, sh)) return;
        // LDS is used again, and fetches are counted from here
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
}

// ------------------------------------------------------------------ host ---
template <int HD, int FMT, bool SPLIT, int NT>
static int attn8_launch(Ctx* c, Attn8Args a)
{
    constexpr int R = 16 * NT;
    a.groups = (int)(((int64_t)a.rows + R - 1) / R);
    const int64_t items = (int64_t)a.groups * a.g.n_seq;
    IAM_REQUIRE(items * a.g.n_kv < ((int64_t)1 << 31), "attention_kv8: too many rows");
    a.items = (int)items;
    // workgroups that the card holds at once
    static const int resident = [] {
        int per_cu = 0, dev = 0, cus = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, k_kv8_attn<HD, FMT, SPLIT, NT>, kAttn8Threads, 0) != hipSuccess ||
            hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
            return 256;
        return std::max(per_cu, 1) * std::max(cus, 1);
    }();
    a.target = (resident + a.g.n_kv - 1) / a.g.n_kv;
    a.planned = items <= kMaxItems;
    int64_t per_head = items;
    if (a.planned) {
        per_head = a.target;
        const int most = (kv8_blocks(a.g.max_ctx) + kAttn8Waves - 1) / kAttn8Waves;   // parts that an item can have
        if (items <= a.target / 8) per_head = std::min<int64_t>(per_head, items * most);
        IAM_TRY(ensure_kv8_scratch(c, 2 * (size_t)per_head * a.g.n_kv * (R * HD + 2 * R), (size_t)items * a.g.n_kv));
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
