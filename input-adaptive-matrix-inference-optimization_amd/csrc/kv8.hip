// The 8-bit KV cache: writing tokens, reading back what they stand for.
#include "kv8.h"
#include "wave.h"

namespace iam {

constexpr int kAppendThreads = 256;

struct AppendArgs {
    const void* src[2];      // K, V
    uint8_t* tiles[2];
    float* scales[2];
    uint16_t* open[2];
    const int* pos;
    const int* count;
    Kv8Geometry g;
    int tokens;
    size_t stride;           // values between tokens
};

__device__ __forceinline__ float half_value(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

// what a byte of a tile stands for, before its scale
template <int FMT>
__device__ __forceinline__ float number(uint8_t b)
{
    half2v lo, hi;
    widen4<FMT>(b, lo, hi);
    return (float)lo[0];
}

// the 16 values (t, d) of run r of a tile: r = 64 * group + 16 * g + m
template <int HD, bool IS_V>
__device__ __forceinline__ int run_token(int r, int e)
{
    const int g = (r >> 4) & 3, m = r & 15, grp = r >> 6;
    return IS_V ? (e >> 3) * 32 + ((e >> 2) & 1) * 16 + g * 4 + (e & 3) : grp / (HD / 64) * 16 + m;
}
template <int HD, bool IS_V>
__device__ __forceinline__ int run_dim(int r, int e)
{
    const int g = (r >> 4) & 3, m = r & 15, grp = r >> 6;
    return IS_V ? grp * 16 + m : grp % (HD / 64) * 64 + g * 16 + e;
}

// n_new rows from token t0 of the open block on, 8 values at a time
template <typename T, int HD, bool IS_V>
__device__ __forceinline__ void open_rows(uint16_t* open, const T* src, size_t stride, int t0, int n_new)
{
    constexpr int Q = HD / 8;
    typedef Pack<T, 8, (int)sizeof(T)> Eight;
    for (int i = threadIdx.x; i < n_new * Q; i += kAppendThreads) {
        const int t = i / Q, d = i % Q * 8;
        const Eight x = *reinterpret_cast<const Eight*>(src + (size_t)t * stride + d);
        half8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (_Float16)to_f32(x.v[e]);
        if constexpr (IS_V) {
#pragma unroll
            for (int e = 0; e < 8; e++) open[v_place(t0 + t, d + e)] = __builtin_bit_cast(uint16_t, (_Float16)h[e]);
        } else {
            *reinterpret_cast<half8*>(open + k_place<HD>(t0 + t, d)) = h;
        }
    }
}

// Workgroup (unit, KV head, K or V; sequence) takes the unit-th block that the
// call's tokens of the sequence touch.  Its new tokens' rows come in 8 values
// at a time.  A block that they fill: the rows go to LDS as fp16, and each
// thread takes HD / 64 runs of 16 values in the tile's order, the earlier
// tokens' from the open block (which is in that order), or from the tile
// where the sequence went back into it; the largest magnitude of all gives the
// scale, and each run becomes 16 bytes.  A block that stays open gets its new
// tokens in fp16.  Only the first block reads the open block and only the last
// may write it, so unit 0 takes both, one after the other.  4000 tokens of 8 x
// 128 fp16 as e4m3 take 12.5 us, 24.6 MB (5 us at a copy's rate): all
// workgroups run at once, and their loads do not hide the arithmetic, 29
// instructions a value, the exact quotients above all (6 us), nor the 2-byte
// reads of V's rows from LDS.  One token is bound by the launch.
template <typename T, int HD, int FMT, bool IS_V>
__device__ __forceinline__ void append_block(const AppendArgs& a, uint16_t* rows, float* red, int seq, int head, int block,
                                             int p0, int p1)
{
    constexpr int RS = HD + 8;                       // LDS row stride: 16 bytes of padding
    constexpr int NT = kAppendThreads, Q = HD / 8, LOADS = kBlk * Q / NT, RUNS = kBlk * HD / 16 / NT;
    const int tid = threadIdx.x;
    const int t0 = max(p0 - block * kBlk, 0);        // new tokens t0 .. t1 of the block
    const int t1 = min(p1 - block * kBlk, kBlk - 1);
    const bool full = t1 == kBlk - 1;
    const size_t cell = kv8_cell(a.g, seq, block, head);
    uint8_t* tile = a.tiles[IS_V] + cell * (size_t)(kBlk * HD);
    uint16_t* open = a.open[IS_V] + ((size_t)seq * a.g.n_kv + head) * (size_t)(kBlk * HD);
    float* scale_p = a.scales[IS_V] + cell;
    const float was = t0 > 0 ? *scale_p : -1.0f;
    const bool reopened = !(was < 0.0f);             // the earlier tokens are in the tile
    // the call's token at position p is row p - p0; the new rows, 8 values a load
    const T* src = reinterpret_cast<const T*>(a.src[IS_V]) + (size_t)head * HD +
                   ((size_t)seq * a.tokens + (size_t)(block * kBlk + t0 - p0)) * a.stride;
    const int n_new = t1 - t0 + 1;
    auto run_of_tile = [&](int r, _Float16* v) __attribute__((always_inline)) {
        const uint4 w = *reinterpret_cast<const uint4*>(tile + (size_t)r * 16);
        const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            half2v lo, hi;
            widen4<FMT>(wd[i], lo, hi);
            v[4 * i] = (_Float16)((float)lo[0] * was);
            v[4 * i + 1] = (_Float16)((float)lo[1] * was);
            v[4 * i + 2] = (_Float16)((float)hi[0] * was);
            v[4 * i + 3] = (_Float16)((float)hi[1] * was);
        }
    };
    if (!full) {
        if (reopened) {
            // all of the tile's values (those from t0 on are written over, or
            // lie past the sequence's end)
#pragma unroll 1
            for (int r = tid; r < kBlk * HD / 16; r += NT) {
                _Float16 v[16];
                run_of_tile(r, v);
#pragma unroll
                for (int e = 0; e < 16; e++) open[r * 16 + e] = __builtin_bit_cast(uint16_t, v[e]);
            }
        }
        __syncthreads();                             // (every thread has read the scale, too)
        open_rows<T, HD, IS_V>(open, src, a.stride, t0, n_new);
        if (tid == 0) *scale_p = -1.0f;
        return;
    }
    typedef Pack<T, 8, (int)sizeof(T)> Eight;
    half8 got[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; u++) {
        const int i = tid + u * NT, t = i / Q, d = i % Q * 8;
        if (t < n_new) {
            const Eight x = *reinterpret_cast<const Eight*>(src + (size_t)t * a.stride + d);
#pragma unroll
            for (int e = 0; e < 8; e++) got[u][e] = (_Float16)to_f32(x.v[e]);
        }
    }
#pragma unroll
    for (int u = 0; u < LOADS; u++) {
        const int i = tid + u * NT, t = i / Q, d = i % Q * 8;
        if (t < n_new) *reinterpret_cast<half8*>(rows + (t0 + t) * RS + d) = got[u];
    }
    _Float16 v[RUNS][16];
    if (t0 > 0) {
#pragma unroll
        for (int u = 0; u < RUNS; u++) {
            const int r = tid + u * NT;
            if (reopened) {
                run_of_tile(r, v[u]);
            } else {
                const half8 x = *reinterpret_cast<const half8*>(open + r * 16), y = *reinterpret_cast<const half8*>(open + r * 16 + 8);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[u][e] = x[e];
                    v[u][8 + e] = y[e];
                }
            }
        }
    }
    __syncthreads();
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < RUNS; u++) {
        const int r = tid + u * NT;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int t = run_token<HD, IS_V>(r, e);
            if (t >= t0) v[u][e] = __builtin_bit_cast(_Float16, rows[t * RS + run_dim<HD, IS_V>(r, e)]);
            top = fmaxf(top, fabsf((float)v[u][e]));
            bad |= (__builtin_bit_cast(uint16_t, v[u][e]) & 0x7c00) == 0x7c00;
        }
    }
    if (bad) top = INFINITY;
    top = wave_max(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) top = fmaxf(top, red[w]);
    const float scale = top < INFINITY ? __fmul_rn(top, kv8_unit<FMT>()) : NAN;
    const bool some = scale > 0.0f;                  // else the numbers are zeros
    const float r1 = some ? __fdiv_rn(1.0f, scale) : 0.0f;
#pragma unroll
    for (int u = 0; u < RUNS; u++) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++)
            w[e >> 2] |= (some ? narrow<FMT>((float)v[u][e], scale, r1) : kv8_zero<FMT>()) << ((e & 3) * 8);
        *reinterpret_cast<uint4*>(tile + (size_t)(tid + u * NT) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (tid == 0) *scale_p = scale;
}

template <typename T, int HD, int FMT>
__global__ __launch_bounds__(kAppendThreads) void k_kv8_append(AppendArgs a)
{
    __shared__ __align__(16) uint16_t rows[kBlk * (HD + 8)];
    __shared__ float red[kAppendThreads / 64];
    const int seq = blockIdx.y;
    const bool is_v = blockIdx.x & 1;
    const int head = (blockIdx.x >> 1) % a.g.n_kv, unit = (blockIdx.x >> 1) / a.g.n_kv;
    const int p0 = a.pos[seq];
    int n = a.tokens;
    if (a.count) n = min(n, a.count[seq]);
    if (p0 < 0 || p0 >= a.g.max_ctx || n <= 0) return;
    const int p1 = p0 + min(n, a.g.max_ctx - p0) - 1;
    const int first = p0 / kBlk, last = p1 / kBlk;
    const bool stays_open = p1 % kBlk != kBlk - 1;   // the last block
    const int block = first + unit;
    if (block > last || (unit > 0 && block == last && stays_open)) return;
    if (is_v) append_block<T, HD, FMT, true>(a, rows, red, seq, head, block, p0, p1);
    else append_block<T, HD, FMT, false>(a, rows, red, seq, head, block, p0, p1);
    if (unit == 0 && last > first && stays_open) {
        __syncthreads();                             // the first block's reads of the open one are done
        const T* src = reinterpret_cast<const T*>(a.src[is_v]) + (size_t)head * HD +
                       ((size_t)seq * a.tokens + (size_t)(last * kBlk - p0)) * a.stride;
        uint16_t* open = a.open[is_v] + ((size_t)seq * a.g.n_kv + head) * (size_t)(kBlk * HD);
        const int n = p1 - last * kBlk + 1;
        if (is_v) open_rows<T, HD, true>(open, src, a.stride, 0, n);
        else open_rows<T, HD, false>(open, src, a.stride, 0, n);
        if (threadIdx.x == 0) a.scales[is_v][kv8_cell(a.g, seq, last, head)] = -1.0f;
    }
}

struct ReadArgs {
    const uint8_t* tiles[2];
    const float* scales[2];
    const uint16_t* open[2];
    float* out[2];
    const int* pos;
    Kv8Geometry g;
    int tokens;
};

// Many tokens: workgroup (unit, KV head, K or V; sequence) takes the unit-th
// block that the rows touch: its runs into LDS (as fp16, numbers before their
// scale: exact), then out by rows, 8 values a thread.  Bound by the writes.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void k_kv8_read_blocks(ReadArgs a)
{
    constexpr int RS = HD + 8, NT = 256, RUNS = kBlk * HD / 16 / NT, Q = HD / 8;
    __shared__ __align__(16) uint16_t rows[kBlk * RS];
    const int tid = threadIdx.x, seq = blockIdx.y, is_v = blockIdx.x & 1;
    const int head = (blockIdx.x >> 1) % a.g.n_kv, unit = (blockIdx.x >> 1) / a.g.n_kv;
    const long long q0 = a.pos[seq], q1 = q0 + a.tokens;                 // the positions asked for
    const int p0 = (int)max(q0, 0ll), p1 = (int)min(q1, (long long)a.g.max_ctx);   // of them, those there are
    const int block = p0 / kBlk + unit;
    if (p0 >= p1 || block > (p1 - 1) / kBlk) return;
    const size_t cell = kv8_cell(a.g, seq, block, head);
    const float scale = a.scales[is_v][cell];
    const bool is_open = scale < 0.0f;
    auto spread = [&](int r, const _Float16* v) __attribute__((always_inline)) {
        if (is_v) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                rows[run_token<HD, true>(r, e) * RS + run_dim<HD, true>(r, e)] = __builtin_bit_cast(uint16_t, v[e]);
        } else {
            half8 x, y;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = v[e];
                y[e] = v[8 + e];
            }
            uint16_t* to = rows + run_token<HD, false>(r, 0) * RS + run_dim<HD, false>(r, 0);
            *reinterpret_cast<half8*>(to) = x;
            *reinterpret_cast<half8*>(to + 8) = y;
        }
    };
#pragma unroll
    for (int u = 0; u < RUNS; u++) {
        const int r = tid + u * NT;
        _Float16 v[16];
        if (is_open) {
            const half8* o = reinterpret_cast<const half8*>(a.open[is_v] + ((size_t)seq * a.g.n_kv + head) * (size_t)(kBlk * HD) + r * 16);
            const half8 x = o[0], y = o[1];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = x[e];
                v[8 + e] = y[e];
            }
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(a.tiles[is_v] + cell * (size_t)(kBlk * HD) + r * 16);
            const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                half2v lo, hi;
                widen4<FMT>(wd[i], lo, hi);
                v[4 * i] = lo[0];
                v[4 * i + 1] = lo[1];
                v[4 * i + 2] = hi[0];
                v[4 * i + 3] = hi[1];
            }
        }
        spread(r, v);
    }
    __syncthreads();
    const float f = is_open ? 1.0f : scale;
    const int t0 = max(p0 - block * kBlk, 0), n = min(p1 - block * kBlk, kBlk) - t0;
    float* out = a.out[is_v] + ((size_t)seq * a.tokens + (size_t)(block * kBlk + t0 - q0)) * ((size_t)a.g.n_kv * HD) + (size_t)head * HD;
    for (int i = tid; i < n * Q; i += NT) {
        const int t = i / Q, d = i % Q * 8;
        const half8 x = *reinterpret_cast<const half8*>(rows + (t0 + t) * RS + d);
        Pack<float, 8, 4> y;
#pragma unroll
        for (int e = 0; e < 8; e++) y.v[e] = (float)x[e] * f;
        *reinterpret_cast<Pack<float, 8, 4>*>(out + (size_t)t * a.g.n_kv * HD + d) = y;
    }
}

// A few tokens: one thread per value.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void k_kv8_read(ReadArgs a)
{
    const int is_v = blockIdx.z, seq = blockIdx.y;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)a.tokens * a.g.n_kv * HD) return;
    const int d = (int)(i % HD), head = (int)(i / HD % a.g.n_kv), token = (int)(i / HD / a.g.n_kv);
    const long long p = (long long)a.pos[seq] + token;
    if (p < 0 || p >= a.g.max_ctx) return;
    const int block = (int)(p / kBlk), t = (int)(p % kBlk);
    const size_t cell = kv8_cell(a.g, seq, block, head);
    const int at = is_v ? v_place(t, d) : k_place<HD>(t, d);
    const float s = a.scales[is_v][cell];
    const float v = s < 0.0f ? half_value(a.open[is_v][((size_t)seq * a.g.n_kv + head) * (size_t)(kBlk * HD) + at])
                             : number<FMT>(a.tiles[is_v][cell * (size_t)(kBlk * HD) + at]) * s;
    a.out[is_v][((size_t)seq * a.tokens + token) * ((size_t)a.g.n_kv * HD) + (size_t)head * HD + d] = v;
}

__global__ __launch_bounds__(256) void k_kv8_reset(float* __restrict__ k, float* __restrict__ v, size_t n)
{
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) k[i] = v[i] = -1.0f;
}

int kv8_check(Ctx* c, const iam_kv8_cache* k, const char* what)
{
    const std::string w(what);
    size_t numbers, scales, open;
    const int rc = iam_kv8_size(k->n_seq, k->max_ctx, k->n_kv, k->head_dim, &numbers, &scales, &open);
    if (rc != IAM_OK) return rc;
    IAM_REQUIRE(k->format == IAM_KV8_INT8 || k->format == IAM_KV8_E4M3, w + ": unknown cache format");
    const void* part[6] = {k->k, k->v, k->k_scale, k->v_scale, k->k_open, k->v_open};
    const size_t bytes[3] = {numbers, scales, open};
    for (int i = 0; i < 6; i++) {
        IAM_REQUIRE(part[i] && aligned(part[i], 16), w + ": a part of the cache is null or not 16-byte aligned");
        IAM_TRY(check_dev_range(c, part[i], bytes[i / 2], what));
        for (int j = 0; j < i; j++)
            IAM_REQUIRE(!overlaps(part[i], bytes[i / 2], part[j], bytes[j / 2]), w + ": parts of the cache overlap");
    }
    return IAM_OK;
}

bool kv8_overlaps(const iam_kv8_cache* k, const void* p, size_t bytes)
{
    size_t n[3];
    if (iam_kv8_size(k->n_seq, k->max_ctx, k->n_kv, k->head_dim, &n[0], &n[1], &n[2]) != IAM_OK) return true;
    return overlaps(p, bytes, k->k, n[0]) || overlaps(p, bytes, k->v, n[0]) || overlaps(p, bytes, k->k_scale, n[1]) ||
           overlaps(p, bytes, k->v_scale, n[1]) || overlaps(p, bytes, k->k_open, n[2]) || overlaps(p, bytes, k->v_open, n[2]);
}

static Kv8Geometry geometry(const iam_kv8_cache* k) { return {k->n_seq, k->max_ctx, k->n_kv, kv8_blocks(k->max_ctx)}; }

template <typename T, int HD>
static int append_typed(Ctx* c, const AppendArgs& a, int format, dim3 grid)
{
    return format == IAM_KV8_INT8
               ? launch(c, "kv8_append", k_kv8_append<T, HD, IAM_KV8_INT8>, grid, dim3(kAppendThreads), 0, a)
               : launch(c, "kv8_append", k_kv8_append<T, HD, IAM_KV8_E4M3>, grid, dim3(kAppendThreads), 0, a);
}

template <typename T>
static int append_dim(Ctx* c, const AppendArgs& a, const iam_kv8_cache* k, dim3 grid)
{
    if (k->head_dim == 64) return append_typed<T, 64>(c, a, k->format, grid);
    if (k->head_dim == 128) return append_typed<T, 128>(c, a, k->format, grid);
    return append_typed<T, 256>(c, a, k->format, grid);
}

// Tokens from which blocks are read as a whole (8 KV heads of 128, one
// sequence, a launch: by value 4.0 us for 1 and 2 tokens, 4.7 to 5.1 for 4;
// by blocks 4.1 for 8 to 64, and 11 for 4000 where by value took 23)
constexpr int kReadBlocks = 4;

template <int HD>
static int read_dim(Ctx* c, const ReadArgs& a, int format)
{
    if (a.tokens >= kReadBlocks) {
        const int units = std::min((a.tokens - 1 + kBlk - 1) / kBlk + 1, a.g.blocks);
        IAM_REQUIRE((int64_t)units * a.g.n_kv < (1 << 23), "kv8_read: too many tokens at a time");
        const dim3 grid((unsigned)units * a.g.n_kv * 2, (unsigned)a.g.n_seq);
        return format == IAM_KV8_INT8 ? launch(c, "kv8_read", k_kv8_read_blocks<HD, IAM_KV8_INT8>, grid, dim3(256), 0, a)
                                      : launch(c, "kv8_read", k_kv8_read_blocks<HD, IAM_KV8_E4M3>, grid, dim3(256), 0, a);
    }
    const size_t per = (size_t)a.tokens * a.g.n_kv * HD;
    const dim3 grid((unsigned)((per + 255) / 256), (unsigned)a.g.n_seq, 2);
    return format == IAM_KV8_INT8 ? launch(c, "kv8_read", k_kv8_read<HD, IAM_KV8_INT8>, grid, dim3(256), 0, a)
                                  : launch(c, "kv8_read", k_kv8_read<HD, IAM_KV8_E4M3>, grid, dim3(256), 0, a);
}

}  // namespace iam

using namespace iam;

extern "C" {

int iam_kv8_size(int n_seq, int max_ctx, int n_kv, int head_dim, size_t* numbers, size_t* scales, size_t* open)
{
    IAM_REQUIRE(n_seq >= 1 && n_seq <= 65535 && n_kv >= 1 && n_kv <= 512, "kv8: n_seq must be 1 to 65535, n_kv 1 to 512");
    IAM_REQUIRE(max_ctx >= 1 && max_ctx <= (1 << 24), "kv8: max_ctx must be 1 to 2^24");
    IAM_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "kv8: head_dim must be 64, 128 or 256");
    const size_t cells = (size_t)n_seq * kv8_blocks(max_ctx) * n_kv;
    if (numbers) *numbers = cells * kBlk * head_dim;
    if (scales) *scales = cells * sizeof(float);
    if (open) *open = (size_t)n_seq * n_kv * kBlk * head_dim * sizeof(uint16_t);
    return IAM_OK;
}

int iam_kv8_reset(iam_ctx* c, const iam_kv8_cache* k)
{
    if (!c || !k) return fail(IAM_E_INVALID, "kv8_reset: null argument");
    IAM_TRY(kv8_check(c, k, "kv8_reset"));
    DeviceGuard on(c);
    const size_t n = (size_t)k->n_seq * kv8_blocks(k->max_ctx) * k->n_kv;
    return launch(c, "kv8_reset", k_kv8_reset, dim3((unsigned)std::min<size_t>((n + 255) / 256, 4096)), dim3(256), 0,
                  k->k_scale, k->v_scale, n);
}

int iam_kv8_append(iam_ctx* c, const iam_kv8_cache* k, const void* key, const void* value, int type, int n_tokens,
                   size_t stride, const int* pos, const int* count)
{
    if (!c || !k || !key || !value || !pos) return fail(IAM_E_INVALID, "kv8_append: null argument");
    IAM_TRY(kv8_check(c, k, "kv8_append"));
    IAM_REQUIRE(type == IAM_F32 || type == IAM_F16 || type == IAM_BF16, "kv8_append: unknown type");
    IAM_REQUIRE(n_tokens >= 0 && n_tokens <= (1 << 24), "kv8_append: n_tokens must be 0 to 2^24");
    const size_t width = (size_t)k->n_kv * k->head_dim, B = type_bytes(type);
    if (!stride) stride = width;
    IAM_REQUIRE(stride >= width && stride < ((size_t)1 << 31), "kv8_append: the stride must hold a row and be below 2^31");
    IAM_REQUIRE(aligned(key, B) && aligned(value, B) && aligned(pos, 4) && aligned(count, 4),
                "kv8_append: k and v must be aligned to their type");
    if (n_tokens == 0) return IAM_OK;
    const size_t bytes = rows_bytes((size_t)k->n_seq * n_tokens, width, stride, B);
    IAM_TRY(check_dev_range(c, key, bytes, "kv8_append k"));
    IAM_TRY(check_dev_range(c, value, bytes, "kv8_append v"));
    IAM_TRY(check_dev_range(c, pos, (size_t)k->n_seq * 4, "kv8_append pos"));
    if (count) IAM_TRY(check_dev_range(c, count, (size_t)k->n_seq * 4, "kv8_append count"));
    IAM_REQUIRE(!kv8_overlaps(k, key, bytes) && !kv8_overlaps(k, value, bytes) && !kv8_overlaps(k, pos, (size_t)k->n_seq * 4) &&
                    (!count || !kv8_overlaps(k, count, (size_t)k->n_seq * 4)),
                "kv8_append: an input overlaps the cache");
    DeviceGuard on(c);
    AppendArgs a{};
    a.src[0] = key;
    a.src[1] = value;
    a.tiles[0] = k->k;
    a.tiles[1] = k->v;
    a.scales[0] = k->k_scale;
    a.scales[1] = k->v_scale;
    a.open[0] = k->k_open;
    a.open[1] = k->v_open;
    a.pos = pos;
    a.count = count;
    a.g = geometry(k);
    a.tokens = n_tokens;
    a.stride = stride;
    // n tokens touch at most ceil((n - 1) / 64) + 1 blocks
    const int units = std::min((n_tokens - 1 + kBlk - 1) / kBlk + 1, kv8_blocks(k->max_ctx));
    IAM_REQUIRE((int64_t)units * k->n_kv < (1 << 23), "kv8_append: too many tokens at a time");
    const dim3 grid((unsigned)units * k->n_kv * 2, (unsigned)k->n_seq);
    if (type == IAM_F32) return append_dim<float>(c, a, k, grid);
    if (type == IAM_F16) return append_dim<_Float16>(c, a, k, grid);
    return append_dim<__bf16>(c, a, k, grid);
}

int iam_kv8_read(iam_ctx* c, const iam_kv8_cache* k, const int* pos, int n_tokens, float* k_out, float* v_out)
{
    if (!c || !k || !pos || !k_out || !v_out) return fail(IAM_E_INVALID, "kv8_read: null argument");
    IAM_TRY(kv8_check(c, k, "kv8_read"));
    IAM_REQUIRE(n_tokens >= 0 && n_tokens <= (1 << 24), "kv8_read: n_tokens must be 0 to 2^24");
    IAM_REQUIRE(aligned(k_out, 4) && aligned(v_out, 4) && aligned(pos, 4), "kv8_read: pointers must be 4-byte aligned");
    if (n_tokens == 0) return IAM_OK;
    const size_t per = (size_t)n_tokens * k->n_kv * k->head_dim, bytes = per * k->n_seq * 4;
    IAM_TRY(check_dev_range(c, k_out, bytes, "kv8_read k"));
    IAM_TRY(check_dev_range(c, v_out, bytes, "kv8_read v"));
    IAM_TRY(check_dev_range(c, pos, (size_t)k->n_seq * 4, "kv8_read pos"));
    IAM_REQUIRE(!kv8_overlaps(k, k_out, bytes) && !kv8_overlaps(k, v_out, bytes) && !overlaps(k_out, bytes, v_out, bytes) &&
                    !overlaps(pos, (size_t)k->n_seq * 4, k_out, bytes) && !overlaps(pos, (size_t)k->n_seq * 4, v_out, bytes),
                "kv8_read: an output overlaps the cache, the positions or the other output");
    DeviceGuard on(c);
    ReadArgs a{};
    a.tiles[0] = k->k;
    a.tiles[1] = k->v;
    a.scales[0] = k->k_scale;
    a.scales[1] = k->v_scale;
    a.open[0] = k->k_open;
    a.open[1] = k->v_open;
    a.out[0] = k_out;
    a.out[1] = v_out;
    a.pos = pos;
    a.g = geometry(k);
    a.tokens = n_tokens;
    if (k->head_dim == 64) return read_dim<64>(c, a, k->format);
    if (k->head_dim == 128) return read_dim<128>(c, a, k->format);
    return read_dim<256>(c, a, k->format);
}

}  // extern "C"
