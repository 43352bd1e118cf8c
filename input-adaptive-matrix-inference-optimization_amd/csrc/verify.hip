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

struct VerifyArgs {
    const void* target;
    const void* draft;       // may be null
    size_t t_stride, d_stride;
    int d_type;
    int seqs, n, vocab;
    double inv_t, inv_d;     // 1 / temperature; 0: greedy
    const int* tokens;
    const int* count;        // may be null
    const float* uniform;
    int* out;
    int* accepted;
    double* stat;            // [seqs][2 n + 1][2]: largest logit and sum of exponentials (NaN: no distribution)
};

__device__ __forceinline__ double logit_of(const void* p, int type, size_t at)
{
    if (type == IAM_F32) return (double)reinterpret_cast<const float*>(p)[at];
    if (type == IAM_F16) return (double)(float)reinterpret_cast<const _Float16*>(p)[at];
    return (double)(float)reinterpret_cast<const __bf16*>(p)[at];
}

// The largest value and its first place, over the workgroup (NaN counts as +inf)
struct Best {
    double m;
    int at;
    __device__ __forceinline__ void take(double v, int i)
    {
        if (v > m || (v == m && i < at)) {
            m = v;
            at = i;
        }
    }
};
__device__ __forceinline__ Best block_best(Best b, Best* red)
{
    for (int d = 1; d < 64; d *= 2) {
        const double m = __shfl_xor(b.m, d);
        const int at = __shfl_xor(b.at, d);
        b.take(m, at);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = b;
    __syncthreads();
    b = red[0];
    for (int w = 1; w < kVerWaves; w++) b.take(red[w].m, red[w].at);
    return b;
}

// A workgroup takes a row of logits: what its softmax is made of, or (greedy)
// where its largest value is.
__global__ __launch_bounds__(kVerThreads) void k_verify_rows(VerifyArgs a, int type)
{
    __shared__ Best red[kVerWaves];
    __shared__ double sums[kVerWaves];
    const int rows = 2 * a.n + 1, s = blockIdx.x / rows, r = blockIdx.x - s * rows, tid = threadIdx.x;
    const bool is_draft = r > a.n;
    if (is_draft && (!a.draft || a.inv_t == 0.0)) return;
    const int dt = is_draft ? a.d_type : type;
    const void* x = is_draft ? a.draft : a.target;
    const size_t base = is_draft ? ((size_t)s * a.n + (r - a.n - 1)) * a.d_stride : ((size_t)s * (a.n + 1) + r) * a.t_stride;
    Best b{-INFINITY, 0x7fffffff};
    for (int i = tid; i < a.vocab; i += kVerThreads) {
        const double v = logit_of(x, dt, base + i);
        b.take(v != v ? (double)INFINITY : v, i);
    }
    b = block_best(b, red);
    const bool none = !(fabs(b.m) < (double)INFINITY);
    double* stat = a.stat + 2 * (size_t)blockIdx.x;
    if (a.inv_t == 0.0) {
        if (tid == 0) stat[0] = none ? -1.0 : (double)b.at;
        return;
    }
    double z = 0.0;
    if (!none)
        for (int i = tid; i < a.vocab; i += kVerThreads)
            z += exp((logit_of(x, dt, base + i) - b.m) * (is_draft ? a.inv_d : a.inv_t));
    z = wave_sum(z);
    if ((tid & 63) == 0) sums[tid >> 6] = z;
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
        for (int w = 0; w < kVerWaves; w++) z += sums[w];
        stat[0] = b.m;
        stat[1] = none ? NAN : z;
    }
}

// A workgroup takes a sequence: which tokens are kept, and the one that follows.
__global__ __launch_bounds__(kVerThreads) void k_verify_pick(VerifyArgs a, int type)
{
    __shared__ double part[kVerThreads + 1];
    __shared__ int picked;
    const int s = blockIdx.x, tid = threadIdx.x;
    const int n = a.count ? min(max(a.count[s], 0), a.n) : a.n;
    const double* stat = a.stat + 2 * (size_t)s * (2 * a.n + 1);
    const int* tokens = a.tokens + (size_t)s * a.n;
    const bool greedy = a.inv_t == 0.0;
    int kept = 0;
    for (; kept < n; kept++) {
        const int t = tokens[kept];
        if (greedy) {
            if (stat[2 * kept] != (double)t) break;
            continue;
        }
        if (t < 0 || t >= a.vocab) break;
        const double p = exp((logit_of(a.target, type, ((size_t)s * (a.n + 1) + kept) * a.t_stride + t) - stat[2 * kept]) * a.inv_t) / stat[2 * kept + 1];
        double q = 1.0;
        if (a.draft) {
            const double* d = stat + 2 * (a.n + 1 + kept);
            q = exp((logit_of(a.draft, a.d_type, ((size_t)s * a.n + kept) * a.d_stride + t) - d[0]) * a.inv_d) / d[1];
        }
        if (!((double)a.uniform[(size_t)s * (a.n + 1) + kept] * q < p)) break;
    }
    int* out = a.out + (size_t)s * (a.n + 1);
    int follow = -1;
    if (greedy) {
        follow = (int)stat[2 * kept];
    } else if (stat[2 * kept + 1] == stat[2 * kept + 1]) {
        const double m = stat[2 * kept], iz = 1.0 / stat[2 * kept + 1];
        const size_t prow = ((size_t)s * (a.n + 1) + kept) * a.t_stride, drow = ((size_t)s * a.n + kept) * a.d_stride;
        const int gone = kept < n ? tokens[kept] : -1;
        const double* d = stat + 2 * (a.n + 1 + kept);
        bool less = kept < n && gone >= 0 && gone < a.vocab && !(a.draft && d[1] != d[1]);
        const double dm = less && a.draft ? d[0] : 0.0, diz = less && a.draft ? 1.0 / d[1] : 0.0;
        auto weight = [&](int i) {
            double w = exp((logit_of(a.target, type, prow + i) - m) * a.inv_t) * iz;
            if (less) {
                if (a.draft) w = fmax(w - exp((logit_of(a.draft, a.d_type, drow + i) - dm) * a.inv_d) * diz, 0.0);
                else if (i == gone) w = 0.0;
            }
            return w;
        };
        const int per = (a.vocab + kVerThreads - 1) / kVerThreads, i0 = min(a.vocab, tid * per), i1 = min(a.vocab, i0 + per);
        for (;;) {
            double w = 0.0;
            for (int i = i0; i < i1; i++) w += weight(i);
            __syncthreads();
            part[tid] = w;
            __syncthreads();
            if (tid == 0) {
                double c = 0.0;
                for (int i = 0; i < kVerThreads; i++) {
                    const double v = part[i];
                    part[i] = c;
                    c += v;
                }
                part[kVerThreads] = c;
                picked = -1;
            }
            __syncthreads();
            if (part[kVerThreads] > 0.0 || !less) break;
            less = false;   // nowhere positive: p alone
        }
        const double want = (double)a.uniform[(size_t)s * (a.n + 1) + a.n] * part[kVerThreads];
        // the slice in which the sum passes it; without one (by rounding) the last token of any weight
        const bool mine = part[tid] <= want && part[tid + 1] > want;
        if (mine) {
            double c = part[tid];
            int last = -1;
            for (int i = i0; i < i1; i++) {
                const double w = weight(i);
                c += w;
                if (w > 0.0) last = i;
                if (c > want) break;
            }
            picked = last;
        }
        __syncthreads();
        if (picked < 0 && tid == 0)
            for (int i = a.vocab - 1; i >= 0 && picked < 0; i--)
                if (weight(i) > 0.0) picked = i;
        __syncthreads();
        follow = picked;
    }
    for (int i = tid; i <= a.n; i += kVerThreads) out[i] = i < kept ? tokens[i] : i == kept ? follow : -1;
    if (tid == 0) a.accepted[s] = kept;
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
    IAM_TRY(ensure_verify_scratch(c, S * (2 * n + 1) * 2, 0));
    const VerifyArgs a{target, draft, t_stride, d_stride, d_type, seqs, n, vocab, greedy ? 0.0 : 1.0 / temperature,
                       draft ? 1.0 / draft_temperature : 0.0, tokens, count, uniform, out, accepted, c->ver_part};
    const dim3 grid((unsigned)(S * (2 * n + 1)));
    IAM_TRY(launch(c, "verify_rows", k_verify_rows, grid, dim3(kVerThreads), 0, a, t_type));
    return launch(c, "verify_pick", k_verify_pick, dim3((unsigned)seqs), dim3(kVerThreads), 0, a, t_type);
}
