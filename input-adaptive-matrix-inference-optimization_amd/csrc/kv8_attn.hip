// Attention over the 8-bit KV cache for few rows of queries a sequence: single
// tokens, above all.  Its entry point.
#include <cmath>

#include "kv8_attn.h"

namespace iam {

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
constexpr int kRun = 64 * 16;   // bytes of a wave's load
template <int YOUNGER>
__device__ __forceinline__ void read_runs(uint32_t at, u32x4* r)
{
    asm volatile(
        "s_waitcnt vmcnt(%5)\n\t"
        "ds_read_b128 %0, %4\n\t"
        "ds_read_b128 %1, %4 offset:%6\n\t"
        "ds_read_b128 %2, %4 offset:%7\n\t"
        "ds_read_b128 %3, %4 offset:%8\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(at), "n"(YOUNGER), "n"(kRun), "n"(2 * kRun), "n"(3 * kRun)
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

constexpr int kRounds = 6;   // rounds of loads that one workgroup joins results in (2 to 8 alike, but for few parts)

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
    constexpr int DD = 4 / NT;                       // dimension tiles whose products run side by side
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
            const Sees see = sees_of(a, sp);   // past these a block needs a mask
            auto cell_of = [&](int b) { return kv8_cell(a.g, sp.seq, b, kvh); };
            // Where the last position does not end its block, the block is
            // open, unless more tokens came since: its scale says so.  The
            // workgroup with the block before `be` among its fours takes it.
            const bool end_inside = be > bs && be == sp.b0 + sp.nb && (see.hi_max + 1) % kBlk != 0 &&
                                    (unsigned)(be - 1 - bs) % (unsigned)sh.stride < kAttn8Waves;
            const float end_scale = end_inside ? a.ks[cell_of(be - 1)] : 0.0f;

            // Its loads do not depend on its scale (as compiled, they wait for
            // the scale's comparison all the same: a link of 0.8 us in the
            // chain before the first tile).
            half8 kk[KS], vv[DT];
            if (end_inside) {
                const size_t ob = ((size_t)sp.seq * a.g.n_kv + kvh) * (size_t)TILE;
                const half8* ko = reinterpret_cast<const half8*>(a.ko + ob) + lane * 2 + w * (HD / 64) * 128;
                const half8* vo = reinterpret_cast<const half8*>(a.vo + ob) + lane * 2 + (w >> 1);
#pragma unroll
                for (int k = 0; k < KS; k++) kk[k] = ko[(k >> 1) * 128 + (k & 1)];
#pragma unroll
                for (int d = 0; d < DT; d++) vv[d] = vo[d * 128];
            }

            Query<HD, SPLIT> query[NT];        // this lane's rows
#pragma unroll
            for (int n = 0; n < NT; n++) query[n].load(a, sp, kvh, n * 16 + r16, g);
            int b = bs + w;
            float ksc = 0.0f, vsc = 0.0f;   // the scales of block b
            if (b < be) {   // (an open block's bytes are not looked at)
                fetch_tile<RUNS, NT == 1>(a.kt + cell_of(b) * (size_t)TILE, place_k);
                asm volatile("" ::: "memory");   // K's first: its wait counts V's as the younger ones
                fetch_tile<RUNS, NT == 1>(a.vt + cell_of(b) * (size_t)TILE, place_v);
                ksc = a.ks[cell_of(b)];
                vsc = a.vs[cell_of(b)];
            }
            int hi[NT], lo[NT];
            float mult[NT];
            half8 qh[PARTS][NT][KS];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                hi[n] = query[n].hi;
                lo[n] = query[n].lo;
                mult[n] = query[n].split(a, qh[0][n], qh[PARTS - 1][n]);
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
                const int at = (be - 1) * kBlk + w * 16 + g * 4;   // the lane's 4 positions:
                const bool upper = w & 1;                          // the second 4 of an operand's 8, or the first
                // an exponent of all ones carries into its half's top bit
                uint32_t ones = 0;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const u32x4 x = __builtin_bit_cast(u32x4, vv[d]);
#pragma unroll
                    for (int e = 0; e < 4; e++) ones |= (x[e] & 0x7c007c00u) + 0x04000400u;
                }
                uint32_t bad = 0;
                if (__any((ones & 0x80008000u) != 0)) {
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
                }
                half8 ph[NT], pl[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    floatx4 sk[2] = {floatx4{0.0f, 0.0f, 0.0f, 0.0f}, floatx4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int x = 0; x < PARTS; x++) sk[k & 1] = mfma(kk[k], qh[x][n][k], sk[k & 1]);
                    floatx4 s = sk[0] + sk[1];
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // an infinite K (its sum of -inf would drop the position): NaN, by 0 * inf
                        s[i] = __builtin_fmaf(s[i], 0.0f, s[i]);
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
                // (sums of other tiles between two that add onto one)
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    half8 ka[4];
#pragma unroll
                    for (int t = 0; t < 4; t++) ka[t] = operand<FMT>(run[t * (HD / 64) + (k >> 1)], k & 1);
#pragma unroll
                    for (int x = 0; x < PARTS; x++)
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int n = 0; n < NT; n++) s[n][t] = mfma(ka[t], qh[x][n][k], s[n][t]);
                }
                const bool edge = b * kBlk + kBlk - 1 > see.hi_all || b * kBlk < see.lo_all;
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
                        for (int i = 0; i < 4; i += 2) {
                            sum += s[n][t][i] + s[n][t][i + 1];
                            half2v h, r;
                            split2(s[n][t][i], s[n][t][i + 1], h, r);
                            const int e = (t & 1) * 4 + i;
                            ph[n][t >> 1][e] = h[0];
                            ph[n][t >> 1][e + 1] = h[1];
                            pl[n][t >> 1][e] = r[0];
                            pl[n][t >> 1][e + 1] = r[1];
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
                for (int d = 0; d < DT; d += DD) {
                    half8 v[2][DD];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < DD; e++) v[h][e] = operand<FMT>(run[d + e], h);
                    floatx4 x[NT][DD];
#pragma unroll
                    for (int y = 0; y < 4; y++)
#pragma unroll
                        for (int e = 0; e < DD; e++)
#pragma unroll
                            for (int n = 0; n < NT; n++)
                                x[n][e] = mfma(v[y & 1][e], (y < 2 ? ph : pl)[n][y & 1], y ? x[n][e] : floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < DD; e++)
#pragma unroll
                            for (int i = 0; i < 4; i++) o[n][d + e][i] = __builtin_fmaf(x[n][e][i], vsr[n], o[n][d + e][i]);
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

            auto put = [&](int row, int d, floatx4 x, float total) __attribute__((always_inline)) {
                put_row<HD, SPLIT>(a, sp, kvh, row, d, x, total);
            };
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += DC) {
                if (d0) __syncthreads();
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int d = 0; d < DC; d++)
                        if (n * 16 + r16 < sp.n_rows) meet[w][n * DC + d][lane] = o[n][d0 + d] * mine[n];
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
                // the KP sums meet.  Where that would take one workgroup many
                // rounds of loads, groups of about the root of their number
                // are joined first, each by its last one (1 KV head of 256, 8
                // query heads, 73769 tokens: 50 us, in groups 28.5; 1 of 128, 16
                // query heads, 131000 tokens: 68 and 23).
                constexpr int U = 8, Q = HD / 4;
                // offsets in 32 bits: the results of a full card are far smaller
                const uint32_t step32 = (uint32_t)step;
                auto slot_of = [&](int k) { return k ? sh.base + k * sh.step : sh.first; };
                const int E = sp.n_rows * Q, passes = (E + kAttn8Threads - 1) / kAttn8Threads;
                const int wide = max(1, kAttn8Threads / E) * U;   // results that a round takes
                const bool tree = passes * sh.splits > kRounds * wide;
                int group = 1, groups = 1, q = 0;   // results of a group, groups, this one's
                if (tree) {
                    group = (int)ceilf(sqrtf((float)sh.splits));
                    groups = up_div(sh.splits, group);
                    q = (sh.slot == sh.first ? 0 : (sh.slot - sh.base) / sh.step) / group;
                }
                floatx4* jo = reinterpret_cast<floatx4*>(lds);
                float* jml = reinterpret_cast<float*>(jo + kAttn8Threads);
#pragma unroll 1
                for (int level = tree ? 0 : 1; level < 2; level++) {
                    const int n = level == 0 ? min(group, sh.splits - q * group) : tree ? groups : sh.splits;
                    uint32_t* ctr = level == 0 ? a.ctr + ((size_t)a.items + slot_of(q * group)) * a.g.n_kv + kvh
                                               : a.ctr + (size_t)sh.item * a.g.n_kv + kvh;
                    if (!acc_arrive(ctr, (uint32_t)n, &s_last)) break;
                    // the k-th result to join
                    const int stride = level == 1 && tree ? group : 1, from = level == 0 ? q * group : 0;
                    const int off = level == 1 && tree ? a.upper : 0;
                    const int KP = max(1, min(kAttn8Threads / E, n));
                    for (int e0 = 0; e0 < E; e0 += kAttn8Threads) {
                        const int kp = KP > 1 ? tid / E : 0, e = KP > 1 ? tid - kp * E : e0 + tid;
                        const bool on = kp < KP && e < E;
                        const int row = on ? e / Q : 0;
                        float jm = -INFINITY, jl = 0.0f;
                        floatx4 jx = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (on)
                            for (int k0 = kp; k0 < n; k0 += U * KP) {
                                float pm[U], pl[U];
                                floatx4 px[U];
#pragma unroll
                                for (int u = 0; u < U; u++) {
                                    const int k = from + min(k0 + u * KP, n - 1) * stride;
                                    const uint32_t at = (uint32_t)kvh * kPartWords + (uint32_t)(off + slot_of(k)) * step32;
                                    pm[u] = acc_peek(a.part + (at + R * HD + row));
                                    pl[u] = acc_peek(a.part + (at + R * HD + R + row));
                                    px[u] = peek4(a.part + (at + e * 4));
                                }
                                float t = jm;
#pragma unroll
                                for (int u = 0; u < U; u++) t = fmaxf(t, pm[u]);
                                const float safe = t == -INFINITY ? 0.0f : t, f0 = exp2_fast(jm - safe);
                                jm = t;
                                jl *= f0;
                                jx *= f0;
#pragma unroll
                                for (int u = 0; u < U; u++) {
                                    const float f = k0 + u * KP < n ? exp2_fast(pm[u] - safe) : 0.0f;
                                    jl = __builtin_fmaf(pl[u], f, jl);
#pragma unroll
                                    for (int i = 0; i < 4; i++) jx[i] = __builtin_fmaf(px[u][i], f, jx[i]);
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
                                jm = t;
                                jl *= f0;
                                jx *= f0;
                                for (int k = 1; k < KP; k++) {
                                    const float f = exp2_fast(jml[2 * (tid + k * E)] - safe);
                                    jl += jml[2 * (tid + k * E) + 1] * f;
                                    jx += jo[tid + k * E] * f;
                                }
                            }
                        }
                        if (on && kp == 0) {
                            if (level == 1) {
                                put(row, (e - row * Q) * 4, jx, jl);
                            } else {
                                float* up = a.part + (uint32_t)kvh * kPartWords + (size_t)(a.upper + slot_of(q * group)) * step32;
                                put4(up + e * 4, jx);
                                if (e == row * Q) {
                                    acc_put(up + R * HD + row, jm);
                                    acc_put(up + R * HD + R + row, jl);
                                }
                            }
                        }
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
    IAM_REQUIRE(items * a.g.n_kv < ((int64_t)1 << 24), "attention_kv8: too many rows");
    a.items = (int)items;
    static const int resident = attn8_resident(k_kv8_attn<HD, FMT, SPLIT, NT>, kAttn8Threads);
    a.target = (resident + a.g.n_kv - 1) / a.g.n_kv;
    a.planned = items <= kMaxItems;
    int64_t per_head = items;
    if (a.planned) {
        per_head = a.target;
        const int most = (kv8_blocks(a.g.max_ctx) + kAttn8Waves - 1) / kAttn8Waves;   // parts that an item can have
        if (items <= a.target / 8) per_head = std::min<int64_t>(per_head, items * most);
        // two results a workgroup, and as many of groups
        a.upper = (int)(2 * per_head);
        IAM_TRY(ensure_kv8_scratch(c, 2 * (size_t)a.upper * a.g.n_kv * (R * HD + 2 * R), (size_t)(items + a.upper) * a.g.n_kv));
        a.part = c->kv8_part;
        a.ctr = c->kv8_ctr;
    }
    const dim3 grid((unsigned)(per_head * a.g.n_kv));
    return launch(c, "kv8_attention", k_kv8_attn<HD, FMT, SPLIT, NT>, grid, dim3(kAttn8Threads), 0, a);
}

template <int HD, int FMT, bool SPLIT>
static int attn8_few(Ctx* c, const Attn8Args& a)
{
    if constexpr (HD <= 128) {
        if (a.rows > 16) return attn8_launch<HD, FMT, SPLIT, 2>(c, a);
    }
    return attn8_launch<HD, FMT, SPLIT, 1>(c, a);
}

// Up to this many rows of a sequence (tokens * query heads of a KV head) every
// wave takes blocks of its own (this file), with more it takes rows of its own:
// 16, one tile, or 64 where sequences and KV heads alone give the card enough
// to do, so that the widening is not what counts (heads of 128, 8 KV heads,
// 2000 tokens, 32 rows, us here and by rows: 1 to 2 sequences 25 and 19, 8
// sequences 31 and 30, 16 36 and 41, 32 46 and 70; 64 rows of 16 sequences 43
// and 53; 96 rows 83 and 61), and for heads of 64, where it costs half (32
// rows, 1 KV head, 2048 tokens 11.5 and 14, 32768 17 and 28; 64 rows, 8 KV
// heads, 8192 tokens 20 and 20).
// Where no row sees more than 4 blocks (a small cache or window), parts and
// their joining cost more than the widening: up to 128 rows, as long as they are
// a workgroup a CU (256 tokens, 8 KV heads of 128: 20 to 128 rows of 4
// sequences 14 and 16 to 19; 64 rows of 32 sequences, two a CU, 28 and 28).
static int few_rows(const Attn8Args& a, int head_dim)
{
    const int64_t pairs = (int64_t)a.g.n_seq * a.g.n_kv;
    const int64_t span = a.window > 0 ? ((int64_t)a.window + a.tokens + 2 * kBlk - 2) / kBlk : a.g.blocks;
    const int tile = head_dim == 256 ? 16 : 32;
    if (std::min<int64_t>(span, a.g.blocks) <= 4 && pairs * ((a.rows + tile - 1) / tile) <= 256) return 128;
    return head_dim == 64 || (head_dim == 128 && pairs >= 64) ? 64 : 16;
}

template <int HD>
static int attn8_dim(Ctx* c, const Attn8Args& a, int format)
{
    if (format == IAM_KV8_INT8)
        return a.type == IAM_F32 ? attn8_few<HD, IAM_KV8_INT8, true>(c, a) : attn8_few<HD, IAM_KV8_INT8, false>(c, a);
    return a.type == IAM_F32 ? attn8_few<HD, IAM_KV8_E4M3, true>(c, a) : attn8_few<HD, IAM_KV8_E4M3, false>(c, a);
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
    a.rep = n_heads / k->n_kv;
    a.tokens = n_tokens;
    a.rows = n_tokens * a.rep;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.window = window;
    a.scale_log2 = (float)((scale > 0.0f ? (double)scale : 1.0 / std::sqrt((double)k->head_dim)) * 1.4426950408889634);
    if (a.rows > few_rows(a, k->head_dim)) return attn8_rows(c, a, k->head_dim, k->format);
    if (k->head_dim == 64) return attn8_dim<64>(c, a, k->format);
    if (k->head_dim == 128) return attn8_dim<128>(c, a, k->format);
    return attn8_dim<256>(c, a, k->format);
}
