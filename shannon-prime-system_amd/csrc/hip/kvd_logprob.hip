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
// One workgroup per row, which it reads once for M, once for the sums and once for
// each alternative (the largest key below the last one's).
#include "kvd_op.h"
#include "kvd_vec.h"

namespace kvd {

namespace {

constexpr int LP_THREADS = 256;

// The order of alternatives as an unsigned key, NaN above all, one zero; the lower
// token first among equals.
__device__ __forceinline__ uint32_t lp_order(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_key(float x, int t) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~t; }

template <typename T, typename Op> __device__ T lp_block(T v, T *red, Op op) {
    for (int o = 32; o; o >>= 1) v = op(v, (T)__shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < LP_THREADS / 64; w++) v = op(v, red[w]);
    return v;
}

__global__ __launch_bounds__(LP_THREADS) void k_logprob_row(sp_hipkv_logprob_args a) {
    __shared__ uint64_t red8[LP_THREADS / 64];
    __shared__ float red4[LP_THREADS / 64];
    const int row = blockIdx.x;
    const float *x = a.logits + row * a.stride;
    float m = -INFINITY, bad = 0.0f;
    for (int t = threadIdx.x; t < a.vocab; t += LP_THREADS) {
        const float y = x[t] * a.scale;
        if (y != y) bad = 1.0f;
        m = fmaxf(m, y);
    }
    m = lp_block(m, red4, [](float p, float q) { return fmaxf(p, q); });
    bad = lp_block(bad, red4, [](float p, float q) { return fmaxf(p, q); });
    float r = 0.0f, e1 = 0.0f, same = 0.0f;
    for (int t = threadIdx.x; t < a.vocab; t += LP_THREADS) {
        const float d = x[t] * a.scale - m;
        if (d == 0.0f) same += 1.0f;
        else if (d > -INFINITY) { const float e = expf(d); r += e; e1 += e * d; }
    }
    auto add = [](float p, float q) { return p + q; };
    same = lp_block(same, red4, add);
    r = lp_block(r, red4, add) + (same - 1.0f);
    e1 = lp_block(e1, red4, add);
    const bool nan = bad != 0.0f, odd = nan || m == INFINITY || m == -INFINITY;
    const float lr = odd ? NAN : log1pf(r);
    if (threadIdx.x == 0) {
        if (a.lse) a.lse[row] = nan ? NAN : odd ? m : m + lr;
        if (a.entropy) a.entropy[row] = odd ? NAN : lr - e1 / (1.0f + r);
    }
    for (int i = threadIdx.x; i < a.n_given; i += LP_THREADS) {
        const int t = a.given[(size_t)row * a.n_given + i];
        a.given_logprob[(size_t)row * a.n_given + i] = t < 0 || t >= a.vocab ? NAN : x[t] * a.scale - m - lr;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < a.n_top; i++) {
        uint64_t best = 0;
        for (int t = threadIdx.x; t < a.vocab; t += LP_THREADS) {
            const uint64_t k = lp_key(x[t], t);
            if (k < last && k > best) best = k;
        }
        last = lp_block(best, red8, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (threadIdx.x == 0) {
            const int t = (int)~(uint32_t)last;
            a.top_ids[(size_t)row * a.n_top + i] = t;
            if (a.top_logprob) a.top_logprob[(size_t)row * a.n_top + i] = x[t] * a.scale - m - lr;
        }
    }
}

int logprob_check(const char *who, const sp_hipkv_logprob_args *a) {
    OP_NEED(a, "null arguments");
    OP_NEED(a->n_rows >= 0 && a->n_rows <= 65535, "n_rows outside [0, 65535]");
    OP_NEED(a->vocab >= 1 && a->vocab <= 1 << 24, "vocab outside [1, 2^24]");
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

void launch_logprob(const sp_hipkv_logprob_args &a, hipStream_t s) {
    hipLaunchKernelGGL(k_logprob_row, dim3(a.n_rows), dim3(LP_THREADS), 0, s, a);
}

}  // namespace kvd

extern "C" int sp_hipkv_token_logprobs_work(const sp_hipkv_logprob_args *a, size_t *bytes) {
    using namespace kvd;
    const char *who = "sp_hipkv_token_logprobs_work";
    if (logprob_check(who, a)) return 1;
    OP_NEED(bytes, "null bytes");
    *bytes = 0;
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
    if (dev.err == hipSuccess) launch_logprob(*a, (hipStream_t)stream);
    return op_done(who, dev);
}
