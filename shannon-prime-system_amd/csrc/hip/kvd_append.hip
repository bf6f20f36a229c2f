// kvd_append.hip -- appending tokens to the paged cache: norm and rotation of q and k,
// K and V rows into their pages.
//
// A workgroup takes one head (of q, k or v) of the tokens that fall into one page, a wave the
// 16 positions of a block in four rounds of four: lane (i, l) of round r has position
// 4 r + i and the pairs l PP .. (l + 1) PP of its head, PP = head_dim / 32, so that a head's
// row is read and written whole by 16 lanes, and a block's largest magnitude and scale stay in
// a wave.  V codes lie by columns (their byte order is the matrix products'): they
// pass LDS, from where a thread writes the 16 bytes of a column that it owns.
//
// Everything is computed in 64 bits: the angle of position p is p freq, off by 2^-53 of
// itself (in 32 bits it would be off by 0.008 at position 131072), and a code is the rounded
// quotient itself, not that of a rounded value.  Sine and cosine are their Taylor series
// behind a reduction by multiples of pi / 2; f64 runs at the rate of f32 here.
#include "kvd_serve.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

// sin and cos of x, |x| below 2^30: x = n pi / 2 + r, |r| <= pi / 4 (a little more where n rounds),
// series to r^15 / 15! and r^16 / 16!, whose next terms are below 2^-54
__device__ __forceinline__ void turn(double x, double &c, double &s) {
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, x);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double a = -1.0 / 1307674368000.0, b = 1.0 / 20922789888000.0;
    a = fma(a, z, 1.0 / 6227020800.0);  b = fma(b, z, -1.0 / 87178291200.0);
    a = fma(a, z, -1.0 / 39916800.0);   b = fma(b, z, 1.0 / 479001600.0);
    a = fma(a, z, 1.0 / 362880.0);      b = fma(b, z, -1.0 / 3628800.0);
    a = fma(a, z, -1.0 / 5040.0);       b = fma(b, z, 1.0 / 40320.0);
    a = fma(a, z, 1.0 / 120.0);         b = fma(b, z, -1.0 / 720.0);
    a = fma(a, z, -1.0 / 6.0);          b = fma(b, z, 1.0 / 24.0);
                                        b = fma(b, z, -0.5);
    a = fma(a * z, r, r);               b = fma(b, z, 1.0);
    const int q = (int)n;
    const double u = q & 1 ? b : a, v = q & 1 ? a : b;
    s = q & 2 ? -u : u;
    c = (q + 1) & 2 ? -v : v;
}

// y as an f32 whose rounding to bf16 is that of y: to the odd of its two neighbours
__device__ __forceinline__ float odd_float(double y) {
    const float f = (float)y;
    uint32_t u = __float_as_uint(f);
    const double d = (double)f;
    if (d != y && fabsf(f) < INFINITY) {
        u -= fabs(d) > fabs(y);                                           // towards zero
        u |= 1;
    }
    return __uint_as_float(u);
}

// The exponent of a block's scale: the least e, from -126 on, with big <= 127 2^e; INT32_MAX if
// f32 has none
__device__ __forceinline__ int scale_exp(double big) {
    const uint64_t u = __builtin_bit_cast(uint64_t, big);
    const int e = (int)(u >> 52 & 2047) - 1022;                           // big = m 2^e, m in [1/2, 1)
    if (e > 128) return INT32_MAX;
    return max((u & 0xFFFFFFFFFFFFFull) <= 63ull << 46 ? e - 7 : e - 6, -126);
}
// A block's scale from what it needs and, where it holds earlier positions, what it has
__device__ __forceinline__ float block_scale(int e, bool older, float was) {
    const float s = e == INT32_MAX ? NAN : __uint_as_float((uint32_t)(e + 127) << 23);
    return older && !(was < s) && s == s ? was : s;
}
__device__ __forceinline__ int code_of(double y, double inv) {
    const double r = rint(y * inv);
    return r == r ? (int)fmin(fmax(r, -127.0), 127.0) : 0;
}
// a stored code at another scale
__device__ __forceinline__ uint32_t recode(uint32_t code, float ratio) {
    const float x = (float)(int8_t)code * ratio;
    return (uint32_t)(x == x ? (int)rintf(x) : 0) & 255;
}

template <typename T, int ROWS, int HD>
__global__ __launch_bounds__(256) void k_append(sp_hipkv_append_args a, int seq_pages) {
    constexpr int PP = HD / 32, H2 = HD / 2;
    constexpr bool B8 = ROWS == SP_HIPKV_ROWS_BLOCK8;
    constexpr int COL = PAGE + 16;                                        // bytes of a column of V codes in LDS
    __shared__ __align__(16) uint8_t s_code[B8 ? HD * COL : 16];
    __shared__ float s_ratio;
    // this workgroup's sequence and page
    const int slot = blockIdx.y;
    int s, j;
    if (seq_pages) { s = slot / seq_pages; j = slot - s * seq_pages; }
    else { s = unit_seq(a.start, a.n_seqs, slot, 1, PAGE, 2); j = slot - (int)unit_base(a.start, s, 1, PAGE, 2); }
    const int t0 = max(gmem(a.start)[s], 0), first = min(max(gmem(a.cached)[s], 0), a.max_positions);
    const int n = min(min(gmem(a.start)[s + 1], a.n_tokens) - t0, min(a.max_tokens, a.max_positions - first)), end = first + n;
    const int lp = first / PAGE + j;
    if (n <= 0 || j < 0 || lp > (end - 1) / PAGE) return;
    // q, k or v, and its head
    int h = blockIdx.x, kind = 0;
    const int nq = a.q_out ? a.n_heads : 0;
    if (h >= nq) { h -= nq; kind = 1; }
    if (kind == 1 && h >= a.n_kv_heads) { h -= a.n_kv_heads; kind = 2; }
    const bool stored = kind && !(a.ring_pages && lp + a.ring_pages <= (end - 1) / PAGE);
    if (!stored && !(kind == 0 || (kind == 1 && a.k_out))) return;
    const int lane = threadIdx.x & 63, u = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane >> 4, l = lane & 15;
    const int b0 = lp * PAGE + BLOCK8 * u;
    const bool some = b0 < end && b0 + BLOCK8 > first, cols = B8 && kind == 2;
    if (!some && !cols) return;
    uint8_t *page = stored ? (uint8_t *)gmem(gmem(a.tables)[s])[a.ring_pages ? lp % a.ring_pages : lp] : nullptr;
    float *scale_at = B8 && stored ? (float *)(page + (size_t)2 * a.n_kv_heads * PAGE * HD) + ((kind - 1) * a.n_kv_heads + h) * PAGE_BLOCKS + u : nullptr;
    auto live = [&](int r) { const int p = b0 + 4 * r + i; return p >= first && p < end; };
    auto round_live = [&](int r) { return b0 + 4 * r < end && b0 + 4 * r + 4 > first; };
    const T *src = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
    const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
    float x[4][2][PP];
    #pragma unroll
    for (int r = 0; r < 4; r++)
        if (live(r)) {
            const T *row = src + (size_t)(t0 + b0 + 4 * r + i - first) * stride + (size_t)h * HD + l * PP;
            load_values(row, x[r][0]);
            load_values(row + H2, x[r][1]);
        }
    const bool older = B8 && some && stored && first > b0;                // positions of the block from earlier calls
    if (kind == 2) {
        if constexpr (!B8) {
            #pragma unroll
            for (int r = 0; r < 4; r++)
                if (live(r)) {
                    float *row = (float *)page + ((size_t)(a.n_kv_heads + h) * PAGE + BLOCK8 * u + 4 * r + i) * HD + l * PP;
                    store_values(row, x[r][0]);
                    store_values(row + H2, x[r][1]);
                }
        } else {
            if (threadIdx.x == 0) s_ratio = 1.0f;
            __syncthreads();
            if (some) {
                uint32_t big = 0;                                         // as bits: NaN is above infinity
                #pragma unroll
                for (int r = 0; r < 4; r++)
                    if (live(r)) {
                        #pragma unroll
                        for (int k = 0; k < PP; k++) big = max(big, max(__float_as_uint(x[r][0][k]) & 0x7FFFFFFFu, __float_as_uint(x[r][1][k]) & 0x7FFFFFFFu));
                    }
                big = (uint32_t)wave_allmax_i((int)big);
                const float was = older ? *scale_at : 0.0f;
                const float sc = block_scale(scale_exp((double)__uint_as_float(big)), older, was);
                const double inv = 1.0 / (double)sc;
                if (lane == 0) {
                    *scale_at = sc;
                    if (older) s_ratio = was / sc;
                }
                #pragma unroll
                for (int r = 0; r < 4; r++)
                    if (live(r)) {
                        #pragma unroll
                        for (int k = 0; k < PP; k++) {
                            uint8_t *col = s_code + (l * PP + k) * COL + 16 * r + 4 * u + i;
                            col[0] = (uint8_t)code_of((double)x[r][0][k], inv);
                            col[H2 * COL] = (uint8_t)code_of((double)x[r][1][k], inv);
                        }
                    }
            }
            __syncthreads();
            const float ratio = s_ratio;                                  // of the codes that the first block has already
            const int p0 = lp * PAGE, old0 = first / BLOCK8 * BLOCK8;
            for (int id = threadIdx.x; id < HD * 4; id += 256) {
                const int d = id >> 2, g = id & 3;
                v4u w = *(const v4u *)(s_code + d * COL + 16 * g);
                KVD_GLOBAL v4u *dst = gmem((v4u *)(page + ((size_t)a.n_kv_heads + h) * PAGE * HD + (size_t)d * PAGE + 16 * g));
                uint32_t fresh = 0, again = 0;                            // bytes to write, bytes to round again
                #pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int p = p0 + (k >> 2) * 16 + 4 * g + (k & 3);
                    fresh |= (uint32_t)(p >= first && p < end) << k;
                    again |= (uint32_t)(p >= old0 && p < first && ratio != 1.0f) << k;
                }
                if (!(fresh | again)) continue;
                if (fresh != 0xFFFF) {
                    const v4u o = *dst;
                    #pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const int sh = 8 * (k & 3);
                        uint32_t b = o[k >> 2] >> sh & 255;
                        if (again >> k & 1) b = recode(b, ratio);
                        if (!(fresh >> k & 1)) w[k >> 2] = (w[k >> 2] & ~(255u << sh)) | b << sh;
                    }
                }
                *dst = w;
            }
        }
        return;
    }
    // q or k: norm, rotation
    double y[4][2][PP];
    double f[PP];
    float w[2][PP];
    const float *nw = kind ? a.k_norm : a.q_norm;
    if (a.freq) {
        #pragma unroll
        for (int k = 0; k < PP; k++) f[k] = gmem(a.freq)[l * PP + k];
    }
    if (nw) {
        #pragma unroll
        for (int k = 0; k < PP; k++) { w[0][k] = gmem(nw)[l * PP + k]; w[1][k] = gmem(nw)[H2 + l * PP + k]; }
    }
    double big = 0.0;
    #pragma unroll
    for (int r = 0; r < 4; r++) {
        if (!round_live(r)) continue;
        #pragma unroll
        for (int k = 0; k < PP; k++) { y[r][0][k] = (double)x[r][0][k]; y[r][1][k] = (double)x[r][1][k]; }
        if (nw) {
            double ss = 0.0;
            #pragma unroll
            for (int k = 0; k < PP; k++) ss = fma(y[r][0][k], y[r][0][k], fma(y[r][1][k], y[r][1][k], ss));
            #pragma unroll
            for (int o = 1; o < 16; o <<= 1) ss += __shfl_xor(ss, o, 64);
            const double m = 1.0 / sqrt(ss * (1.0 / HD) + (double)a.eps);
            #pragma unroll
            for (int k = 0; k < PP; k++) { y[r][0][k] = y[r][0][k] * m * (double)w[0][k]; y[r][1][k] = y[r][1][k] * m * (double)w[1][k]; }
        }
        if (a.freq) {
            const double p = (double)(b0 + 4 * r + i);
            #pragma unroll
            for (int k = 0; k < PP; k++) {
                double c, sn;
                turn(p * f[k], c, sn);
                const double x0 = y[r][0][k], x1 = y[r][1][k];
                y[r][0][k] = fma(x0, c, -(x1 * sn));
                y[r][1][k] = fma(x0, sn, x1 * c);
            }
        }
        if (B8 && live(r)) {
            #pragma unroll
            for (int k = 0; k < PP; k++)
                #pragma unroll
                for (int e = 0; e < 2; e++) {                              // NaN and infinities as infinity
                    const double v = fabs(y[r][e][k]);
                    big = v < INFINITY ? fmax(big, v) : INFINITY;
                }
        }
        void *back = kind ? a.k_out : a.q_out;
        if (back && live(r)) {
            T *row = (T *)back + (size_t)(t0 + b0 + 4 * r + i - first) * (kind ? a.k_out_stride : a.q_out_stride) + (size_t)h * HD + l * PP;
            float z[2][PP];
            #pragma unroll
            for (int k = 0; k < PP; k++)
                #pragma unroll
                for (int e = 0; e < 2; e++) z[e][k] = sizeof(T) == 4 ? (float)y[r][e][k] : odd_float(y[r][e][k]);
            store_values(row, z[0]);
            store_values(row + H2, z[1]);
        }
        if (!B8 && stored && live(r)) {
            float *row = (float *)page + ((size_t)h * PAGE + BLOCK8 * u + 4 * r + i) * HD + l * PP;
            float z[2][PP];
            #pragma unroll
            for (int k = 0; k < PP; k++) { z[0][k] = (float)y[r][0][k]; z[1][k] = (float)y[r][1][k]; }
            store_values(row, z[0]);
            store_values(row + H2, z[1]);
        }
    }
    if (!B8 || !stored) return;
    big = bcast63(wave_to63(big, 0.0, [](double p, double q) { return fmax(p, q); }));
    const float was = older ? *scale_at : 0.0f;
    const float sc = block_scale(scale_exp(big), older, was), ratio = was / sc;
    const double inv = 1.0 / (double)sc;
    if (lane == 0) *scale_at = sc;
    #pragma unroll
    for (int r = 0; r < 4; r++) {
        const int p = b0 + 4 * r + i;
        const bool again = older && p < first && ratio != 1.0f;
        if (!live(r) && !again) continue;
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            uint8_t *row = page + ((size_t)h * PAGE + BLOCK8 * u + 4 * r + i) * HD + l * PP + e * H2;
            uint32_t c[(PP + 3) / 4];
            if (again) {
                #pragma unroll
                for (int k = 0; k < PP; k++) {
                    const uint32_t b = recode(gmem(row)[k], ratio);
                    c[k / 4] = k % 4 ? c[k / 4] | b << 8 * (k % 4) : b;
                }
            } else {
                #pragma unroll
                for (int k = 0; k < PP; k++) {
                    const uint32_t b = (uint32_t)code_of(y[r][e][k], inv) & 255;
                    c[k / 4] = k % 4 ? c[k / 4] | b << 8 * (k % 4) : b;
                }
            }
            if constexpr (PP == 2) *gmem((uint16_t *)row) = (uint16_t)c[0];
            else if constexpr (PP == 4) *gmem((uint32_t *)row) = c[0];
            else *gmem((v2u *)row) = (v2u){c[0], c[1]};
        }
    }
}

// Pages that a call's tokens may fall into: with few tokens a sequence every sequence's most,
// else by the packed tokens (a page and its neighbour more for each sequence).
struct AppendPlan { int slots, seq_pages; };
AppendPlan append_plan(const sp_hipkv_append_args &a) {
    const int64_t most = ((int64_t)a.max_tokens + PAGE - 2) / PAGE + 1, packed = (int64_t)a.n_tokens / PAGE + 2 * a.n_seqs;
    return most * a.n_seqs <= packed ? AppendPlan{(int)(most * a.n_seqs), (int)most} : AppendPlan{(int)packed, 0};
}

int append_check(const sp_hipkv_append_args *a) {
    const char *who = "sp_hipkv_append";
    if (serve_check(who, a)) return 1;
    OP_NEED(a->rows == SP_HIPKV_ROWS_F32 || a->rows == SP_HIPKV_ROWS_BLOCK8, "rows is neither f32 nor 8-bit blocks");
    OP_NEED(a->max_positions >= 0 && a->max_positions <= 1 << 20, "max_positions outside [0, 2^20]");
    OP_NEED(a->max_tokens <= 1 << 20, "max_tokens above 2^20");
    OP_NEED(a->ring_pages >= 0, "negative ring_pages");
    OP_NEED(std::isfinite(a->eps) && a->eps >= 0, "eps is negative or not finite");
    if (!a->n_tokens) return 0;
    OP_NEED(a->start && a->cached && a->tables, "null array");
    OP_NEED(aligned(a->tables, 8) && aligned(a->freq, 8), "misaligned array");
    OP_NEED(!a->q_out || a->q, "q_out without q");
    if (serve_rows(who, a, a->k, a->k_stride, a->n_kv_heads) || serve_rows(who, a, a->v, a->v_stride, a->n_kv_heads)) return 1;
    if (a->k_out && serve_rows(who, a, a->k_out, a->k_out_stride, a->n_kv_heads)) return 1;
    if (a->q_out && (serve_rows(who, a, a->q, a->q_stride, a->n_heads) || serve_rows(who, a, a->q_out, a->q_out_stride, a->n_heads))) return 1;
    OP_NEED(a->q_out != a->q || a->q_out_stride == a->q_stride, "q_out is q with another stride");
    OP_NEED(a->k_out != a->k || a->k_out_stride == a->k_stride, "k_out is k with another stride");
    return 0;
}

template <typename T, int ROWS> hipError_t append_go(const sp_hipkv_append_args &a, hipStream_t s) {
    const AppendPlan p = append_plan(a);
    const dim3 grid((a.q_out ? a.n_heads : 0) + 2 * a.n_kv_heads, p.slots);
    return op_launch(a.head_dim == 256 ? k_append<T, ROWS, 256> : a.head_dim == 128 ? k_append<T, ROWS, 128> : k_append<T, ROWS, 64>,
                     grid, dim3(256), s, a, p.seq_pages);
}

}  // namespace

hipError_t launch_append(const sp_hipkv_append_args &a, hipStream_t s) {
    if (a.rows == SP_HIPKV_ROWS_F32) return a.type == SP_HIPKV_F32 ? append_go<float, SP_HIPKV_ROWS_F32>(a, s) : append_go<Bf16, SP_HIPKV_ROWS_F32>(a, s);
    return a.type == SP_HIPKV_F32 ? append_go<float, SP_HIPKV_ROWS_BLOCK8>(a, s) : append_go<Bf16, SP_HIPKV_ROWS_BLOCK8>(a, s);
}

}  // namespace kvd

extern "C" size_t sp_hipkv_block8_page_bytes(int32_t n_kv_heads, int32_t head_dim) {
    if (n_kv_heads <= 0 || n_kv_heads > 4096 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
    return kvd::block8_bytes(n_kv_heads, head_dim);
}

extern "C" int sp_hipkv_append(const sp_hipkv_append_args *a, void *stream) {
    using namespace kvd;
    if (append_check(a)) return 1;
    if (!a->n_tokens) return 0;
    OpDevice dev((hipStream_t)stream);
    return op_done("sp_hipkv_append", dev.err != hipSuccess ? dev.err : launch_append(*a, (hipStream_t)stream));
}
