// Attention over the 8-bit KV cache for many rows of queries a sequence: a
// prompt's chunk.
#include "kv8_attn.h"

namespace iam {

// An item is 128 rows.  The workgroup brings one block of K and V at a time
// into LDS as fp16 operands, each wave its share (so that the widening of a
// number is paid once for 128 rows); the next block's bytes are on their way
// meanwhile.  Bound by the softmax and the matrix instructions (48 to 64 a block
// and 16 rows): of 67 us (500 tokens behind 3.6k, fp32) a SIMD's vector
// instructions are busy 36 and its matrix units 26, and two workgroups of a CU
// overlap little of them.  Beside its blocks a call takes 25 us, half of that
// partial results.
// The low parts of an fp32 q are in LDS, or two workgroups would not fit the
// registers.  v_scale is taken into the probabilities' shift: o is kept in units
// of one block's v_scale (v_unit), so that the products add onto o itself.
// Waves and tiles of 16 rows of each: two tiles share every operand read from
// LDS, where the registers of two workgroups a CU hold them, nearly: with heads
// of 128 and an fp32 q, 4 (int8) and 2 (e4m3) vector registers are spilled (500
// tokens behind 3.6k, heads of 128: 81 us; 8 waves of one tile took 12 % more.
// Heads of 256, one KV head: two tiles 94 us, 8 waves of one 66).
template <int HD>
struct RowsShape {
    static constexpr int TILES = HD <= 128 ? 2 : 1, WAVES = HD <= 128 ? 4 : 8;
};
constexpr int kRowsItem = 128;
constexpr int kRowsLeast = 2;   // blocks of a workgroup where an item is split (4 and 8 were no faster)

template <int HD, int FMT, bool SPLIT>
__global__ __launch_bounds__(64 * RowsShape<HD>::WAVES, 2) void k_kv8_attn_rows(Attn8Args a)
{
    constexpr int NT = RowsShape<HD>::TILES, W = RowsShape<HD>::WAVES, KS = HD / 32, DT = HD / 16, R = kRowsItem;
    static_assert(16 * NT * W == R, "the waves' rows");
    constexpr int RUNS = HD / 16, TILE = kBlk * HD, MINE = 2 * RUNS / W;
    constexpr int kPartWords = R * HD + 2 * R;
    __shared__ half8 tiles[4 * RUNS][64];        // K: operand (t, k) at KS t + k; V: (d, h) at 2 RUNS + 2 d + h
    __shared__ half8 low[SPLIT ? W : 1][SPLIT ? NT : 1][SPLIT ? KS : 1][64];
    __shared__ int pre[kMaxItems + 1];
    __shared__ unsigned long long bad_s;         // open block: positions whose V is not finite
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r16 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.g.n_kv, j = blockIdx.x / a.g.n_kv;
    Deal deal{};
    Share sh{};
    if (a.planned) {
        if (!find_deal<W>(a, j, R, pre, deal, kRowsLeast)) return;
        if (deal.mode == 0) sh = deal.one;
        else if (!next_share(a, pre, j, deal, sh)) return;
    } else {
        sh.item = a.items - 1 - j;   // the row groups with the longest contexts first
        sh.splits = 1;
        sh.to = 1 << 30;
    }
    for (;;) {
        const Span sp = span_of(a, sh.item, R);
        const int bs = sp.b0 + sh.from, be = sp.b0 + min(sh.to, sp.nb);
        if (sp.n_rows > 0) {
            const Sees see = sees_of(a, sp);
            auto cell_of = [&](int b) { return kv8_cell(a.g, sp.seq, b, kvh); };
            // the last block is open where its scale says so (see k_kv8_attn)
            const bool end_inside = be > bs && be == sp.b0 + sp.nb && (see.hi_max + 1) % kBlk != 0;
            const int open_at = end_inside && a.ks[cell_of(be - 1)] < 0.0f ? be - 1 : -1;
            if (tid == 0) bad_s = 0;
            __syncthreads();

            u32x4 raw[MINE];   // runs w, w + W, ... of K's and then V's
            float ks_next = 0.0f, vs_next = 0.0f;
            auto fetch = [&](int b) __attribute__((always_inline)) {
                const size_t at = cell_of(b) * (size_t)TILE + lane * 16;
                ks_next = a.ks[cell_of(b)];
                vs_next = a.vs[cell_of(b)];
#pragma unroll
                for (int i = 0; i < MINE; i++) {
                    const int run = i * W + w;
                    const uint8_t* t = run < RUNS ? a.kt : a.vt;
                    raw[i] = *reinterpret_cast<const u32x4*>(t + at + (size_t)(run % RUNS) * 1024);
                }
            };
            auto store = [&](int b) __attribute__((always_inline)) {
                if (b == open_at) {
                    // fp16 as it is; what is not finite in V is taken out, and
                    // goes by its positions' s
                    const size_t ob = ((size_t)sp.seq * a.g.n_kv + kvh) * (size_t)TILE;
                    uint32_t bad = 0;
#pragma unroll
                    for (int i = 0; i < MINE; i++) {
                        const int run = i * W + w;
                        const half8* o = reinterpret_cast<const half8*>((run < RUNS ? a.ko : a.vo) + ob) + run % RUNS * 128 + lane * 2;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            half8 x = o[h];
                            if (run >= RUNS) {
#pragma unroll
                                for (int e = 0; e < 8; e++)
                                    if ((__builtin_bit_cast(uint16_t, (_Float16)x[e]) & 0x7c00) == 0x7c00) {
                                        bad |= 1u << (h * 8 + e);
                                        x[e] = (_Float16)0.0f;
                                    }
                            }
                            tiles[2 * run + h][lane] = x;
                        }
                    }
                    if (bad) {
                        // (the lane's run holds positions 4 g .. of each 16)
                        const unsigned long long m = (unsigned long long)(bad & 15) | (unsigned long long)(bad >> 4 & 15) << 16 |
                                                     (unsigned long long)(bad >> 8 & 15) << 32 | (unsigned long long)(bad >> 12) << 48;
                        atomicOr(&bad_s, m << (g * 4));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < MINE; i++) {
                        const int run = i * W + w;
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            tiles[2 * run + h][lane] = operand<FMT>(raw[i], h);
                    }
                }
            };
            if (bs < be) fetch(bs);

            int hi[NT], lo[NT];
            float mult[NT];
            half8 qh[NT][KS];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                Query<HD, SPLIT> query;
                query.load(a, sp, kvh, (w * NT + n) * 16 + r16, g);
                hi[n] = query.hi;
                lo[n] = query.lo;
                half8 ql[KS];
                mult[n] = query.split(a, qh[n], ql);
                if constexpr (SPLIT) {
#pragma unroll
                    for (int k = 0; k < KS; k++) low[w][n][k][lane] = ql[k];
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
            float v_unit = 1.0f;
            const bool mine_there = w * 16 * NT < sp.n_rows;   // the wave has rows
            for (int b = bs; b < be; b++) {
                store(b);
                // (they came with the bytes: a wait for them here would wait for
                // the next block's, too)
                float ksc = ks_next, vsc = vs_next;
                if (b + 1 < be) fetch(b + 1);
                __syncthreads();
                if (mine_there) {
                    uint32_t bad = 0;   // a bit for each of the lane's 16 positions
                    if (b == open_at) {
                        ksc = vsc = 1.0f;
                        const unsigned long long m = bad_s >> (g * 4);
                        bad = (uint32_t)(m & 15) | (uint32_t)(m >> 12 & 0xf0) | (uint32_t)(m >> 24 & 0xf00) | (uint32_t)(m >> 36 & 0xf000);
                    }
                    const half8(*tv)[64] = tiles + 2 * RUNS;
                    floatx4 s[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int t = 0; t < 4; t++) s[n][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        half8 ql[NT];
                        if constexpr (SPLIT) {
#pragma unroll
                            for (int n = 0; n < NT; n++) ql[n] = low[w][n][k][lane];
                        }
                        half8 ka[4];
#pragma unroll
                        for (int t = 0; t < 4; t++) ka[t] = tiles[t * KS + k][lane];
                        // sums of other tiles between two that add onto one
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int n = 0; n < NT; n++) s[n][t] = mfma(ka[t], qh[n][k], s[n][t]);
                        if constexpr (SPLIT) {
#pragma unroll
                            for (int t = 0; t < 4; t++)
#pragma unroll
                                for (int n = 0; n < NT; n++) s[n][t] = mfma(ka[t], ql[n], s[n][t]);
                        }
                    }
                    const bool edge = b * kBlk + kBlk - 1 > see.hi_all || b * kBlk < see.lo_all;
                    // The probabilities carry vsc / v_unit, kept within [2^-6,
                    // 2^3] (a block of zeros: any): o's unit changes seldom.
                    float turn = 1.0f;
                    if (vsc != vsc) {
                        ksc = vsc;                 // NaN, for the rows that see the block
                    } else if (vsc > 0.0f && !(vsc <= 8.0f * v_unit && vsc >= 0.015625f * v_unit)) {
                        turn = v_unit / vsc;       // o into the new unit
                        v_unit = vsc;
                    }
                    const float ratio = vsc > 0.0f ? vsc / v_unit : 1.0f;
                    const float bias = kProbShift + log2f(ratio), back = 1.0f / ratio;
                    half8 ph[NT][2], pl[NT][2];
                    float alpha[NT];
                    bool grown = turn != 1.0f;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float f = mult[n] * ksc;
                        uint32_t hidden = 0;   // bits as in bad
                        if (edge) {
                            const int from = lo[n] - (b * kBlk + g * 4), to = hi[n] - (b * kBlk + g * 4);
#pragma unroll
                            for (int t = 0; t < 4; t++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    // an infinite K (its sum of -inf would drop the position): NaN, by 0 * inf
                                    s[n][t][i] = __builtin_fmaf(s[n][t][i], 0.0f, s[n][t][i]);
                                    if (bad & 1u << (t * 4 + i)) s[n][t][i] = NAN;
                                    if (t * 16 + i < from || t * 16 + i > to) {
                                        hidden |= 1u << (t * 4 + i);
                                        s[n][t][i] = -INFINITY;
                                    }
                                }
                        }
                        float top = -INFINITY;
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) top = fmaxf(top, s[n][t][i]);
                        top = row_max(top);
                        const float mn = fmaxf(m[n], top == -INFINITY ? top : top * f);
                        const float safe = mn == -INFINITY ? 0.0f : mn;
                        alpha[n] = exp2_fast(m[n] - safe);
                        grown |= mn != m[n];
                        m[n] = mn;
                        const float shift = bias - safe;
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) s[n][t][i] = exp2_fast(__builtin_fmaf(s[n][t][i], f, shift));
                        if (edge) {
#pragma unroll
                            for (int t = 0; t < 4; t++)
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (hidden & 1u << (t * 4 + i)) s[n][t][i] = 0.0f;   // also where f is 0 or NaN
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
                        l[n] = l[n] * alpha[n] + sum * back;
                    }
                    if (__any(grown)) {   // most blocks do not raise any row's maximum
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int d = 0; d < DT; d++) o[n][d] *= alpha[n] * turn;
                    }
#pragma unroll
                    for (int d = 0; d < DT; d += 2) {
                        half8 v[2][2];
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int e = 0; e < 2; e++) v[h][e] = tv[2 * (d + e) + h][lane];
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int x = 0; x < 2; x++)
#pragma unroll
                                for (int n = 0; n < NT; n++)
#pragma unroll
                                    for (int e = 0; e < 2; e++)
                                        o[n][d + e] = mfma(v[h][e], x ? pl[n][h] : ph[n][h], o[n][d + e]);
                    }
                }
                __syncthreads();
            }

            const bool whole = sh.splits == 1;
            const size_t step = (size_t)a.g.n_kv * kPartWords;
            float* part = whole ? nullptr : a.part + sh.slot * step + (size_t)kvh * kPartWords;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int row = (w * NT + n) * 16 + r16;
                l[n] = row_sum(l[n]);
                if (row >= sp.n_rows) continue;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const floatx4 x = o[n][d] * v_unit;
                    if (whole) put_row<HD, SPLIT>(a, sp, kvh, row, d * 16 + g * 4, x, l[n]);
                    else *reinterpret_cast<floatx4*>(part + row * HD + d * 16 + g * 4) = x;
                }
                if (!whole && g == 0) {
                    part[R * HD + row] = m[n];
                    part[R * HD + R + row] = l[n];
                }
            }
        }
        if (a.planned && kvh == 0 && sh.from == 0 && tid == 0) a.joins[sh.item] = make_int4(sh.splits, sh.first, sh.base, sh.step);
        if (!a.planned || deal.mode == 0 || !next_share(a, pre, j, deal, sh)) return;
        __syncthreads();   // LDS is used again
    }
}

// The split items' results joined: 256 threads take 1024 values of an item and
// KV head, a thread four, 8 of the partial results' loads in flight; PARTS
// such groups take every PARTS-th result (4 where an item has more than 8 in
// the mean: 32 rows over 32768 tokens 52 us with 1, 28 with 4; 500 tokens
// behind 3600 80 and 85).  A launch of its own, since a chunk's partial results are many (an item's 64 KB
// a workgroup): joined by the last workgroup to arrive, as for single tokens,
// they took 100 us for 64 tokens behind 4000.
constexpr int kJoinThreads = 256;
template <int HD, bool SPLIT, int PARTS>
__global__ __launch_bounds__(kJoinThreads * PARTS) void k_kv8_join(Attn8Args a)
{
    constexpr int R = kRowsItem, Q = HD / 4, ROWS = kJoinThreads / Q, U = 8;
    constexpr int kPartWords = R * HD + 2 * R;
    __shared__ floatx4 sx[PARTS > 1 ? PARTS : 1][PARTS > 1 ? kJoinThreads : 1];
    __shared__ float sm[PARTS > 1 ? PARTS : 1][PARTS > 1 ? kJoinThreads : 1], sl[PARTS > 1 ? PARTS : 1][PARTS > 1 ? kJoinThreads : 1];
    const int kvh = blockIdx.x % a.g.n_kv, u = blockIdx.x / a.g.n_kv, it = blockIdx.y;
    const int4 jn = a.joins[it];    // splits, first, base, step
    const int tid = threadIdx.x % kJoinThreads, part = threadIdx.x / kJoinThreads;
    if (jn.x <= 1) return;
    const Span sp = span_of(a, it, R);
    if (u * ROWS >= sp.n_rows) return;
    const int row = u * ROWS + tid / Q, d = tid % Q * 4;
    const bool there = row < sp.n_rows;
    const size_t step = (size_t)a.g.n_kv * kPartWords;
    const float* parts = a.part + (size_t)kvh * kPartWords;
    float jm = -INFINITY, jl = 0.0f;
    floatx4 jx = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = part; there && k0 < jn.x; k0 += U * PARTS) {
        float pm[U], pl[U];
        floatx4 px[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int k = min(k0 + i * PARTS, jn.x - 1);
            const float* p = parts + (k ? jn.z + k * jn.w : jn.y) * step;
            pm[i] = p[R * HD + row];
            pl[i] = p[R * HD + R + row];
            px[i] = *reinterpret_cast<const floatx4*>(p + row * HD + d);
        }
        float t = jm;
#pragma unroll
        for (int i = 0; i < U; i++) t = fmaxf(t, pm[i]);
        const float safe = t == -INFINITY ? 0.0f : t, f0 = exp2_fast(jm - safe);
        jm = t;
        jl *= f0;
        jx *= f0;
#pragma unroll
        for (int i = 0; i < U; i++)
            if (k0 + i * PARTS < jn.x) {
                const float f = exp2_fast(pm[i] - safe);
                jl += pl[i] * f;
                jx += px[i] * f;
            }
    }
    if constexpr (PARTS > 1) {
        sx[part][tid] = jx;
        sm[part][tid] = jm;
        sl[part][tid] = jl;
        __syncthreads();
        if (part > 0) return;
        float t = jm;
#pragma unroll
        for (int k = 1; k < PARTS; k++) t = fmaxf(t, sm[k][tid]);
        const float safe = t == -INFINITY ? 0.0f : t, f0 = exp2_fast(jm - safe);
        jl *= f0;
        jx *= f0;
#pragma unroll
        for (int k = 1; k < PARTS; k++) {
            const float f = exp2_fast(sm[k][tid] - safe);
            jl += sl[k][tid] * f;
            jx += sx[k][tid] * f;
        }
    }
    if (there) put_row<HD, SPLIT>(a, sp, kvh, row, d, jx, jl);
}

// ------------------------------------------------------------------ host ---
template <int HD, int FMT, bool SPLIT>
static int rows_launch(Ctx* c, Attn8Args a)
{
    constexpr int R = kRowsItem;
    a.groups = (int)(((int64_t)a.rows + R - 1) / R);
    const int64_t items = (int64_t)a.groups * a.g.n_seq;
    IAM_REQUIRE(items * a.g.n_kv < ((int64_t)1 << 23), "attention_kv8: too many rows");
    a.items = (int)items;
    static const int resident = attn8_resident(k_kv8_attn_rows<HD, FMT, SPLIT>, 64 * RowsShape<HD>::WAVES);
    a.target = (resident + a.g.n_kv - 1) / a.g.n_kv;
    a.planned = items <= kMaxItems;
    int64_t per_head = items;
    if (a.planned) {
        per_head = std::min<int64_t>(a.target, items * ((kv8_blocks(a.g.max_ctx) + kRowsLeast - 1) / kRowsLeast));
        // the joins' records lie behind the partial results
        const size_t words = 2 * (size_t)per_head * a.g.n_kv * (R * HD + 2 * R);
        IAM_TRY(ensure_kv8_scratch(c, words + 4 * (size_t)items, 1));
        a.part = c->kv8_part;
        a.joins = reinterpret_cast<int4*>(a.part + words);
    }
    const dim3 grid((unsigned)(per_head * a.g.n_kv));
    IAM_TRY(launch(c, "kv8_attention", k_kv8_attn_rows<HD, FMT, SPLIT>, grid, dim3(64 * RowsShape<HD>::WAVES), 0, a));
    if (!a.planned || per_head == 1) return IAM_OK;
    const dim3 join((unsigned)a.g.n_kv * (R * (HD / 4) / kJoinThreads), (unsigned)items);
    return per_head > 8 * items ? launch(c, "kv8_attention.join", k_kv8_join<HD, SPLIT, 4>, join, dim3(kJoinThreads * 4), 0, a)
                                : launch(c, "kv8_attention.join", k_kv8_join<HD, SPLIT, 1>, join, dim3(kJoinThreads), 0, a);
}

template <int HD>
static int rows_dim(Ctx* c, const Attn8Args& a, int format)
{
    if (format == IAM_KV8_INT8)
        return a.type == IAM_F32 ? rows_launch<HD, IAM_KV8_INT8, true>(c, a) : rows_launch<HD, IAM_KV8_INT8, false>(c, a);
    return a.type == IAM_F32 ? rows_launch<HD, IAM_KV8_E4M3, true>(c, a) : rows_launch<HD, IAM_KV8_E4M3, false>(c, a);
}

int attn8_rows(Ctx* c, const Attn8Args& a, int head_dim, int format)
{
    if (head_dim == 64) return rows_dim<64>(c, a, format);
    if (head_dim == 128) return rows_dim<128>(c, a, format);
    return rows_dim<256>(c, a, format);
}

}  // namespace iam
