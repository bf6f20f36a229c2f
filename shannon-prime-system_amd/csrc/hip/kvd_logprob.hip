// kvd_logprob.hip -- of each row of logits: log probabilities of given tokens,
// entropy, and the largest logits' tokens.
//
// With y = scale x, M = max y, c = the number of y equal to M:
//   r = c - 1 + sum_{y < M} e^(y - M)        (softmax's sum less its largest term, 1)
//   lse = M + log1p(r),  log p_t = (y_t - M) - log1p(r),
//   H = log1p(r) - sum_{y < M} e^(y - M) (y - M) / (1 + r).
// r is kept without the 1, which f32 sums would round small remainders away on: a
// row that is sure of its token has an entropy of the remainder's size.
//
// k_lp_part reads a row once, a segment of it per workgroup, held in registers: its
// maximum, its r and sum of e^d d, and its n_top largest as sorted keys.  k_lp_merge
// joins a row's segments:
//   r = (segments at M) - 1 + sum_{m_s = M} r_s + sum_{m_s < M} e^(m_s - M) (1 + r_s),
// and so on.  The floor is the row's bytes: 64 rows of 262144 are 67 MB, 14 us, which
// k_lp_part takes without alternatives.
//
// The n_top largest of a workgroup: the n_top-th largest of its threads' maxima is a
// bound from below, found by bisection with ballots; it leaves few candidates (about
// 25 of 8192 at 20), which are ranked by counting.  More than the list holds (many equal
// logits) are searched by rounds, from memory: keys kept for that would fill the
// registers, and 64 of them let 8 workgroups share a unit.  64 rows of 262144, 20
// alternatives: k_lp_part 20.1 us, k_lp_merge 6.6 (28.8 and 7.8 with a bound of
// each wave's own, 32 steps and 82 registers).  The rest above the bytes is the bound's and the
// ranking's latency, once for each workgroup.
#include "kvd_op.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

constexpr int LP_THREADS = 256, LP_WAVES = LP_THREADS / 64;
constexpr int LP_LIST = 1024;                    // candidates of a workgroup
constexpr int LP_SEGS = 128;                     // segments of a row at most
constexpr int LP_LONG = 32, LP_SHORT = 8;        // logits per thread

typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t ORDER_MIN = 0x007FFFFF;       // -infinity's

// The order of alternatives as an unsigned number, NaN above all, one zero; 0 is below
// any logit.  The lower token first among equals.
__device__ __forceinline__ uint32_t lp_order(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t order) { return __uint_as_float(order >> 31 ? order ^ 0x80000000u : ~order); }
__device__ __forceinline__ uint64_t lp_key(uint32_t order, int t) { return order ? (uint64_t)order << 32 | (uint32_t)~t : 0; }

template <typename T, typename Op> __device__ __forceinline__ T lp_block(T v, T *red, Op op) {
    #pragma unroll
    for (int o = 32; o; o >>= 1) v = op(v, (T)__shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    #pragma unroll
    for (int w = 1; w < LP_WAVES; w++) v = op(v, red[w]);
    return v;
}

// A bound T >= 1 on the workgroup's k-th largest order from below: the k-th largest of
// the threads' largest, s.lane, its lower half cleared (16 steps for 32, and few more candidates).
struct LpSelect {
    uint64_t list[LP_LIST + 4], red[LP_WAVES];
    uint32_t lane[LP_THREADS];
    int count;
};
__device__ __forceinline__ uint32_t lp_bound(const uint32_t (&q)[LP_WAVES], int k) {
    uint32_t T = 0;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
        int c = 0;
        #pragma unroll
        for (int w = 0; w < LP_WAVES; w++) c += __popcll(__ballot(q[w] >= (T | bit)));
        if (c >= k) T |= bit;
    }
    return T ? T : 1u;
}
// The k largest of the workgroup's keys, descending, to dst[0..k) (0 where there are
// fewer), from the list of those above a bound (s.count of them) or, where that
// overflowed, by rounds over key(i) of i < size, from memory.
template <typename Key> __device__ __forceinline__ void lp_rank(LpSelect &s, int k, int size, Key key, uint64_t *dst) {
    const int n = s.count;
    if (n <= LP_LIST) {
        for (int i = threadIdx.x; i < n; i += LP_THREADS) {
            const uint64_t x = s.list[i];
            int rank = 0;
            for (int j = 0; j < n; j += 4)
                #pragma unroll
                for (int u = 0; u < 4; u++) rank += j + u < n && s.list[j + u] > x;
            if (rank < k) dst[rank] = x;
        }
        for (int i = n + threadIdx.x; i < k; i += LP_THREADS) dst[i] = 0;
        return;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < k; i++) {
        uint64_t best = 0;
        for (int j = threadIdx.x; j < size; j += LP_THREADS) {
            const uint64_t x = key(j);
            if (x < last && x > best) best = x;
        }
        __syncthreads();
        last = lp_block(best, s.red, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (threadIdx.x == 0) dst[i] = last;
    }
}

// A segment's part of its row: M, r, sum of e^d d; nan != 0: it holds a NaN.
struct LpPart { float m, r, e1, nan; };

// grid (segments, rows); keys [row][segment][n_top]
template <int N>
__global__ __launch_bounds__(LP_THREADS) void k_lp_part(sp_hipkv_logprob_args a, LpPart *part, uint64_t *keys) {
    __shared__ float red[4][LP_WAVES];
    __shared__ LpSelect sel;
    const int row = blockIdx.y, t0 = blockIdx.x * N * LP_THREADS + threadIdx.x * 4;
    const float *x = a.logits + row * a.stride;
    float v[N];
    #pragma unroll
    for (int k = 0; k < N / 4; k++) {
        const int t = t0 + k * 4 * LP_THREADS;
        v4u f = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (t + 4 <= a.vocab) f = *(const v4u *)(x + t);
        else if (t < a.vocab) {                  // absent: below every logit
            f[0] = x[t];
            if (t + 1 < a.vocab) f[1] = x[t + 1];
            if (t + 2 < a.vocab) f[2] = x[t + 2];
        }
        #pragma unroll
        for (int e = 0; e < 4; e++) v[4 * k + e] = f[e];
    }
    // the threads' largest, in order, serve the maximum (scaling keeps the order) and the bound
    float big = -INFINITY, nan = 0.0f;
    #pragma unroll
    for (int e = 0; e < N; e++) {
        big = fmaxf(big, v[e]);
        nan = v[e] != v[e] ? 1.0f : nan;
    }
    sel.lane[threadIdx.x] = t0 < a.vocab ? lp_order(nan != 0.0f ? NAN : big) : 0;
    if (threadIdx.x == 0) sel.count = 0;
    __syncthreads();
    uint32_t q[LP_WAVES];
    #pragma unroll
    for (int w = 0; w < LP_WAVES; w++) q[w] = sel.lane[64 * w + (threadIdx.x & 63)];
    const uint32_t top = (uint32_t)wave_allmax_i((int)(max(max(q[0], q[1]), max(q[2], q[3])) ^ 0x80000000u)) ^ 0x80000000u;
    const float m = lp_value(top) * a.scale;
    float r = 0.0f, e1 = 0.0f, same = 0.0f;
    #pragma unroll
    for (int e = 0; e < N; e++) {
        const float d = fmaxf(v[e] * a.scale - m, -200.0f);      // e^-200 is 0
        const float w = d < 0.0f ? __builtin_amdgcn_exp2f(d * 1.44269504088896341f) : 0.0f;
        r += w; e1 += w * d;
        same += d == 0.0f ? 1.0f : 0.0f;
    }
    #pragma unroll
    for (int o = 32; o; o >>= 1) {
        r += __shfl_xor(r, o, 64); e1 += __shfl_xor(e1, o, 64);
        same += __shfl_xor(same, o, 64); nan = fmaxf(nan, __shfl_xor(nan, o, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        const int w = threadIdx.x >> 6;
        red[0][w] = r; red[1][w] = e1; red[2][w] = nan; red[3][w] = same;      // r without the count, which would swallow it
    }
    if (a.n_top) {
        const uint32_t T = lp_bound(q, a.n_top);
        int lim = LP_THREADS;
        if (T <= ORDER_MIN) {
            // Fewer than n_top threads have a logit above -infinity (a masked vocabulary).
            // Of the others the lowest tokens count: those of each thread's first four up to the
            // ninth thread that has none, 36 or more.
            int c = 0;
            #pragma unroll
            for (int w = 0; w < LP_WAVES; w++) {
                uint64_t none = __ballot(q[w] == ORDER_MIN);
                for (; none; none &= none - 1)
                    if (++c == 9) lim = 64 * w + __builtin_ctzll(none);
            }
        }
        if (__any(sel.lane[threadIdx.x] >= T)) {
            const float least = T <= ORDER_MIN ? -INFINITY : lp_value(T);
            #pragma unroll
            for (int e = 0; e < N; e++)
                if (!(v[e] < least) && (v[e] != -INFINITY || lim == LP_THREADS || (e < 4 && (int)threadIdx.x <= lim))) {
                    const int t = t0 + (e / 4) * 4 * LP_THREADS + e % 4;
                    if (t >= a.vocab) continue;
                    const int at = atomicAdd(&sel.count, 1);
                    if (at < LP_LIST) sel.list[at] = lp_key(lp_order(v[e]), t);
                }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float rs = 0.0f, sm = 0.0f, es = 0.0f, ns = 0.0f;
        #pragma unroll
        for (int w = 0; w < LP_WAVES; w++) {
            rs += red[0][w]; es += red[1][w]; ns = fmaxf(ns, red[2][w]); sm += red[3][w];
        }
        part[(size_t)row * gridDim.x + blockIdx.x] = {m, rs + (sm - 1.0f), es, ns};
    }
    if (a.n_top) {
        const int first = blockIdx.x * N * LP_THREADS;
        lp_rank(sel, a.n_top, min(N * LP_THREADS, a.vocab - first), [&](int i) { return lp_key(lp_order(x[first + i]), first + i); },
                keys + ((size_t)row * gridDim.x + blockIdx.x) * a.n_top);
    }
}

// one workgroup per row
__global__ __launch_bounds__(LP_THREADS) void k_lp_merge(sp_hipkv_logprob_args a, int segs, const LpPart *part, const uint64_t *keys) {
    __shared__ float redf[LP_WAVES];
    __shared__ double redd[3][LP_WAVES];
    __shared__ LpSelect sel;
    __shared__ uint64_t top[32];
    const int row = blockIdx.x, have = segs * a.n_top;
    const float *x = a.logits + row * a.stride;
    const bool mine = (int)threadIdx.x < segs;
    constexpr int N = LP_SEGS * 32 / LP_THREADS;
    LpPart p = {-INFINITY, 0.0f, 0.0f, 0.0f};
    if (mine) p = part[(size_t)row * segs + threadIdx.x];
    uint64_t k[N];
    uint32_t big = 0;
    #pragma unroll
    for (int e = 0; e < N; e++) {
        const int i = e * LP_THREADS + (int)threadIdx.x;
        k[e] = i < have ? keys[(size_t)row * have + i] : 0;
        big = max(big, (uint32_t)(k[e] >> 32));
    }
    // given tokens' logits, on their way while the sums are joined
    const int gt = (int)threadIdx.x < a.n_given ? a.given[(size_t)row * a.n_given + threadIdx.x] : -1;
    const float gx = gt >= 0 && gt < a.vocab ? x[gt] : NAN;
    sel.lane[threadIdx.x] = big;
    if (threadIdx.x == 0) sel.count = 0;
    const float M = lp_block(p.m, redf, [](float u, float w) { return fmaxf(u, w); });
    // NaN as a count in the same sum
    const bool live = mine && p.m > -INFINITY && M < INFINITY;
    const double f = live ? exp((double)p.m - (double)M) : 0.0;
    const bool at = live && p.m == M;
    double s[3] = {live ? (at ? (double)p.r : f * (1.0 + (double)p.r)) : 0.0,
                   live ? f * ((double)p.e1 + ((double)p.m - (double)M) * (1.0 + (double)p.r)) : 0.0,
                   (at ? 1.0 : 0.0) + (p.nan != 0.0f ? 65536.0 : 0.0)};
    #pragma unroll
    for (int i = 0; i < 3; i++) {
        #pragma unroll
        for (int o = 32; o; o >>= 1) s[i] += __shfl_xor(s[i], o, 64);
        if ((threadIdx.x & 63) == 0) redd[i][threadIdx.x >> 6] = s[i];
    }
    if (a.n_top) {
        uint32_t q[LP_WAVES];
        #pragma unroll
        for (int w = 0; w < LP_WAVES; w++) q[w] = sel.lane[64 * w + (threadIdx.x & 63)];
        const uint32_t T = lp_bound(q, a.n_top);
        #pragma unroll
        for (int e = 0; e < N; e++)
            if ((uint32_t)(k[e] >> 32) >= T) {
                const int i = atomicAdd(&sel.count, 1);
                if (i < LP_LIST) sel.list[i] = k[e];
            }
    }
    __syncthreads();
    if (a.n_top) lp_rank(sel, a.n_top, have, [&](int i) { return keys[(size_t)row * have + i]; }, top);
    #pragma unroll
    for (int i = 0; i < 3; i++) s[i] = (redd[i][0] + redd[i][1]) + (redd[i][2] + redd[i][3]);
    const bool nan = s[2] >= 65536.0, odd = nan || M == INFINITY || M == -INFINITY;
    const double r = s[0] + (s[2] - 1.0), e1 = s[1], l1 = log1p(r);
    const float lr = odd ? NAN : (float)l1;
    if (threadIdx.x == 0) {
        if (a.lse) a.lse[row] = nan ? NAN : odd ? M : (float)((double)M + l1);
        if (a.entropy) a.entropy[row] = odd ? NAN : (float)(l1 - e1 / (1.0 + r));
    }
    if ((int)threadIdx.x < a.n_given) a.given_logprob[(size_t)row * a.n_given + threadIdx.x] = gx * a.scale - M - lr;
    if (!a.n_top) return;
    __syncthreads();
    if ((int)threadIdx.x < a.n_top) {
        const int t = (int)~(uint32_t)top[threadIdx.x];
        const float v = lp_value((uint32_t)(top[threadIdx.x] >> 32));
        a.top_ids[(size_t)row * a.n_top + threadIdx.x] = t;
        if (a.top_logprob) a.top_logprob[(size_t)row * a.n_top + threadIdx.x] = v * a.scale - M - lr;
    }
}

// Segments of 2048 logits where that is what it takes to use the device, else of 8192
// (one row of 151936: 75 workgroups for 19).
struct LpPlan { int per, segs; int64_t parts; };       // parts: room for this many rows or fewer
LpPlan lp_plan(const sp_hipkv_logprob_args &a) {
    const int longs = (a.vocab + LP_LONG * LP_THREADS - 1) / (LP_LONG * LP_THREADS);
    const int shorts = (a.vocab + LP_SHORT * LP_THREADS - 1) / (LP_SHORT * LP_THREADS);
    const int64_t few = shorts <= LP_SEGS ? std::min(a.n_rows, 511 / longs) * (int64_t)shorts : 0, many = (int64_t)a.n_rows * longs;
    if (shorts <= LP_SEGS && many < 512) return {LP_SHORT, shorts, few};
    return {LP_LONG, longs, std::max(few, many)};
}
size_t lp_part_bytes(const LpPlan &p) { return (size_t)p.parts * sizeof(LpPart); }

int logprob_check(const char *who, const sp_hipkv_logprob_args *a) {
    OP_NEED(a, "null arguments");
    OP_NEED(a->n_rows >= 0 && a->n_rows <= 65535, "n_rows outside [0, 65535]");
    OP_NEED(a->vocab >= 1 && a->vocab <= LP_SEGS * LP_LONG * LP_THREADS, "vocab outside [1, 2^20]");
    OP_NEED(a->n_given >= 0 && a->n_given <= 64, "n_given outside [0, 64]");
    OP_NEED(a->n_top >= 0 && a->n_top <= 32 && a->n_top <= a->vocab, "n_top outside [0, 32] or above vocab");
    return 0;
}
int logprob_check_arrays(const char *who, const sp_hipkv_logprob_args *a, size_t need) {
    OP_NEED(a->scale > 0.0f && std::isfinite(a->scale), "scale is not positive and finite");
    OP_NEED(a->stride >= a->vocab || a->n_rows == 1, "stride is below vocab");
    OP_NEED(a->logits && (!a->n_given || (a->given && a->given_logprob)) && (!a->n_top || a->top_ids), "null array");
    OP_NEED(aligned(a->logits, 4), "misaligned logits");
    OP_NEED(!need || (a->work && a->work_bytes >= need && aligned(a->work, 16)), "work is missing, too small or not 16-byte aligned");
    return 0;
}

}  // namespace

hipError_t launch_logprob(const sp_hipkv_logprob_args &a, hipStream_t s) {
    const LpPlan p = lp_plan(a);
    LpPart *part = (LpPart *)a.work;
    uint64_t *keys = (uint64_t *)((uint8_t *)a.work + lp_part_bytes(p));
    const dim3 grid(p.segs, a.n_rows), wg(LP_THREADS);
    const hipError_t e = op_launch(p.per == LP_LONG ? k_lp_part<LP_LONG> : k_lp_part<LP_SHORT>, grid, wg, s, a, part, keys);
    return e != hipSuccess ? e : op_launch(k_lp_merge, dim3(a.n_rows), wg, s, a, p.segs, part, keys);
}

}  // namespace kvd

extern "C" int sp_hipkv_token_logprobs_work(const sp_hipkv_logprob_args *a, size_t *bytes) {
    using namespace kvd;
    const char *who = "sp_hipkv_token_logprobs_work";
    if (logprob_check(who, a)) return 1;
    OP_NEED(bytes, "null bytes");
    const LpPlan p = lp_plan(*a);
    *bytes = lp_part_bytes(p) + (size_t)p.parts * a->n_top * sizeof(uint64_t);
    return 0;
}

extern "C" int sp_hipkv_token_logprobs(const sp_hipkv_logprob_args *a, void *stream) {
    using namespace kvd;
    const char *who = "sp_hipkv_token_logprobs";
    if (logprob_check(who, a)) return 1;
    if (!a->n_rows) return 0;
    size_t need = 0;
    if (sp_hipkv_token_logprobs_work(a, &need) || logprob_check_arrays(who, a, need)) return 1;
    OpDevice dev((hipStream_t)stream);
    return op_done(who, dev.err != hipSuccess ? dev.err : launch_logprob(*a, (hipStream_t)stream));
}
