// kvd_append.hip -- appending tokens to the paged cache: norm and rotation of q and k,
// K and V rows into their pages.
//
// A wave takes the 16 positions of a block, or half of them, in rounds of four, of one head of q, k
// or v: lane (i, l) of round r has position 4 r + i and the pairs l PP .. (l + 1) PP of a head, PP =
// head_dim / 32, so that a row is read and written whole by 16 lanes, and a block's largest
// magnitude and scale stay in a wave.  V codes lie by columns (their byte order is the
// matrix products'): they pass LDS, from where a thread writes the bytes of a column that it owns.
//
// Everything is computed in 64 bits: the angle of position p is p freq, off by 2^-53 of
// itself (in 32 bits it would be off by 0.008 at position 131072), and a code is the rounded
// quotient itself, not that of a rounded value.  f64 runs at the rate of f32 here.  Sine and
// cosine are Taylor series behind a reduction by multiples of pi / 2, for four positions and for a
// step of four; the others' follow by turning.  Of long appends a workgroup takes one block of four q or k heads,
// whose sines it forms once, in LDS; of short ones each wave forms its own (the step's by parts in its four rows of
// lanes, none for single tokens).
//
// 4096 tokens of 32 and 8 heads of 128 in bf16 take 34.7 us (36.4 with sines a head), 20.8 at the rate of a
// large copy.  Without norm and rotation they take 30 to 32: waves load, compute and store by turns, and what
// counts is how many rows are on their way.  (K's values formed again behind the scale, for fewer registers: 58 us for
// 64, 3900 tokens of 16 and 8 heads of 256, but 36 here and 14.5 for 11.8, four prompts of 200; for 256 dims and long
// appends alone it is left.)  16
// and 8 heads of 256 in f32 to f32 rows, which need no scale first, run at 88 % of a copy's rate.
#include "kvd_serve.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

typedef double v2d __attribute__((ext_vector_type(2)));

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

// the sum over the 16 lanes of a row
__device__ __forceinline__ double row_sum(double x) {
    auto step = [&](auto ctrl) { x += __builtin_bit_cast(double, dpp64<decltype(ctrl)::value, 0xF>(__builtin_bit_cast(uint64_t, x), 0)); };
    step(std::integral_constant<int, 0xB1>{});                            // quad_perm 1,0,3,2
    step(std::integral_constant<int, 0x4E>{});                            // quad_perm 2,3,0,1
    step(std::integral_constant<int, 0x141>{});                           // row_half_mirror
    step(std::integral_constant<int, 0x140>{});                           // row_mirror
    return x;
}
// 1 / sqrt(x): the instruction's estimate (2^-24 or better), then Newton's y + y (1 - x y^2) / 2 twice: 3/8 e^2 each; 0 of
// infinity, where Newton's step is 0 x inf
__device__ __forceinline__ double inv_sqrt(double x) {
    double y = __builtin_amdgcn_rsq(x);
    #pragma unroll
    for (int i = 0; i < 2; i++) y = fma(y * 0.5, fma(-(x * y), y, 1.0), y);
    return x == INFINITY ? 0.0 : y;
}

// y[] as f32, or as f32 whose rounding to bf16 is that of y: only where the nearest f32 lies half way between
// two bf16 does the second rounding need the side that y is on
template <typename T, int N> __device__ __forceinline__ void rounded(const double (&y)[N], float (&z)[N]) {
    bool tie = false;
    #pragma unroll
    for (int k = 0; k < N; k++) {
        z[k] = (float)y[k];
        tie |= sizeof(T) == 2 && (__float_as_uint(z[k]) & 0xFFFF) == 0x8000;
    }
    if (sizeof(T) == 2 && __builtin_expect(__any(tie), 0)) {
        #pragma unroll
        for (int k = 0; k < N; k++) {
            const uint32_t u = __float_as_uint(z[k]);
            if ((u & 0xFFFF) == 0x8000) z[k] = __uint_as_float(u + (fabs(y[k]) > fabs((double)z[k])) - (fabs(y[k]) < fabs((double)z[k])));
        }
    }
}

// The exponent of a block's scale: the least e, from -126 on, with big <= 127 2^e; INT32_MAX if
// f32 has none, or big is none
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
// Codes, in the low byte: adding 3 2^51 (2^22) leaves the nearest integer in the low bits, ties to even
__device__ __forceinline__ uint32_t code_of(double y, double inv) { return (uint32_t)__builtin_bit_cast(uint64_t, fma(y, inv, 6755399441055744.0)); }
__device__ __forceinline__ uint32_t code_of(float y, float inv) { return __float_as_uint(fmaf(y, inv, 12582912.0f)); }
// a stored code at another scale
__device__ __forceinline__ uint32_t recode(uint32_t code, float ratio) { return code_of((float)(int8_t)code, ratio) & 255; }

// Waves that share a block, two rounds each: of 8-bit rows of 256 dims one alone holds 64 values of 64 bits a lane
// until the block's scale is known (3900 tokens of 16 and 8 heads 76 us for 71, 20 prompts of 40 30.3 for 27.9; of
// 128 dims, each wave with sines of its own, 36.5 us for 44, 4096 tokens of 32 and 8 heads)
constexpr int block_waves(int rows, int hd) { return rows == SP_HIPKV_ROWS_BLOCK8 && hd == 256 ? 2 : 1; }

// q and k heads by workgroups of HG
template <int HG> __host__ __device__ constexpr int append_qk(const sp_hipkv_append_args &a) {
    return ((a.q_out ? a.n_heads : 0) + a.n_kv_heads + HG - 1) / HG * HG;
}

// NB: 4, a page, or 1.
template <typename T, int ROWS, int HD, int NB>
__global__ __launch_bounds__(64 * NB * block_waves(ROWS, HD), 2) void k_append(sp_hipkv_append_args a, int seq_units) {
    constexpr int PP = HD / 32, H2 = HD / 2, UNIT = BLOCK8 * NB, WB = block_waves(ROWS, HD), NR = 4 / WB, NT = 64 * NB * WB;
    constexpr bool B8 = ROWS == SP_HIPKV_ROWS_BLOCK8;
    constexpr int COL = 16 * NB + 16;                                     // bytes of a column of V codes in LDS
    constexpr int HG = NB > 1 ? 4 : 1;                                    // heads of q and k of a workgroup
    constexpr int CODES = B8 ? HD * COL : 16, SINES = NB > 1 ? 16 * H2 * 16 : 16;
    __shared__ __align__(16) uint8_t s_code[CODES > SINES ? CODES : SINES];
    __shared__ float s_ratio;
    __shared__ double s_big[NB * WB];
    // this workgroup's sequence and unit of positions
    const int slot = blockIdx.y;
    UnitSeq seq;
    int j;
    if (seq_units) {
        seq.s = slot / seq_units;
        j = slot - seq.s * seq_units;
        seq.start = gmem(a.start)[seq.s]; seq.end = gmem(a.start)[seq.s + 1];
    } else {
        seq = unit_seq(a.start, a.n_seqs, slot, 1, UNIT, 2);
        j = slot - (int)unit_base(seq.start, seq.s, 1, UNIT, 2);
    }
    const int s = seq.s;
    const void *const *table = gmem(a.tables)[s];
    const int t0 = max(seq.start, 0), first = min(max(gmem(a.cached)[s], 0), a.max_positions);
    const int n = min(min(seq.end, a.n_tokens) - t0, min(a.max_tokens, a.max_positions - first)), end = first + n;
    const int p0 = (first / UNIT + j) * UNIT, lp = p0 / PAGE;
    if (n <= 0 || j < 0 || p0 >= end) return;
    // q, k or v, and its head: of V a head's NB blocks, of q and k one block of HG heads, which share its sines
    const int nq = a.q_out ? a.n_heads : 0, qk = append_qk<HG>(a), x0 = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane >> 4, l = lane & 15;
    int h = x0 - qk, kind = 2, blk = wave / WB;
    if (x0 < qk) {
        if constexpr (HG > 1) { h = x0 / HG * HG + blk; blk = x0 % HG; }
        else h = x0;
        kind = h >= nq;
        if (kind) h -= nq;
    }
    const bool stored = kind && h < a.n_kv_heads && !(a.ring_pages && lp + a.ring_pages <= (end - 1) / PAGE);
    if (kind == 2 && !stored) return;
    const int b0 = p0 + BLOCK8 * blk, r0 = wave % WB * NR, u = b0 / BLOCK8 % PAGE_BLOCKS;
    const bool some = b0 < end && b0 + BLOCK8 > first;
    if (!some && !(B8 && kind == 2)) return;                              // (of q and k all waves, of f32 rows of V without more barriers)
    const bool mine = kind == 0 || stored || (a.k_out && h < a.n_kv_heads);
    if (HG == 1 && !mine) return;
    uint8_t *page = stored ? (uint8_t *)gmem(table)[a.ring_pages ? lp % a.ring_pages : lp] : nullptr;
    auto live = [&](int r) { const int p = b0 + 4 * (r0 + r) + i; return (HG == 1 || mine) && p >= first && p < end; };
    auto round_live = [&](int r) { return b0 + 4 * (r0 + r) < end && b0 + 4 * (r0 + r) + 4 > first; };
    const bool older = B8 && some && stored && first > b0;                // positions of the block from earlier calls
    auto row_of = [&](auto *p, int64_t stride, int r, int head) __attribute__((always_inline)) {
        return p + (size_t)(t0 + b0 + 4 * (r0 + r) + i - first) * stride + (size_t)head * HD + l * PP;
    };
    auto put = [&](auto *row, const float (&z)[2 * PP]) __attribute__((always_inline)) {
        float z0[PP], z1[PP];
        #pragma unroll
        for (int k = 0; k < PP; k++) { z0[k] = z[k]; z1[k] = z[PP + k]; }
        store_values(row, z0);
        store_values(row + H2, z1);
    };
    const T *src = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
    const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
    float x[NR][2][PP] = {};
    #pragma unroll
    for (int r = 0; r < NR; r++)
        if (live(r)) {
            const T *row = row_of(src, stride, r, h);
            load_values(row, x[r][0]);
            load_values(row + H2, x[r][1]);
        }
    if (kind == 2) {
        if constexpr (!B8) {
            #pragma unroll
            for (int r = 0; r < NR; r++)
                if (live(r)) {
                    float *row = (float *)page + ((size_t)(a.n_kv_heads + h) * PAGE + BLOCK8 * u + 4 * (r0 + r) + i) * HD + l * PP;
                    store_values(row, x[r][0]);
                    store_values(row + H2, x[r][1]);
                }
        } else {
            float *scale_at = (float *)(page + (size_t)2 * a.n_kv_heads * PAGE * HD) + (a.n_kv_heads + h) * PAGE_BLOCKS + u;
            if (threadIdx.x == 0) s_ratio = 1.0f;
            if (NT > 64) __syncthreads();
            uint32_t big = 0;                                         // as bits: NaN is above infinity
            #pragma unroll
            for (int r = 0; r < NR; r++)
                if (live(r)) {
                    #pragma unroll
                    for (int k = 0; k < PP; k++) big = max(big, max(__float_as_uint(x[r][0][k]) & 0x7FFFFFFFu, __float_as_uint(x[r][1][k]) & 0x7FFFFFFFu));
                }
            big = (uint32_t)wave_allmax_i((int)big);
            const float was = older ? *scale_at : 0.0f;
            if constexpr (WB > 1) {
                if (lane == 0) ((uint32_t *)s_big)[wave] = big;
                __syncthreads();
                big = max(big, ((uint32_t *)s_big)[wave ^ 1]);
            }
            if (some) {
                const float sc = block_scale(scale_exp((double)__uint_as_float(big)), older, was), inv = 1.0f / sc;
                if (lane == 0 && r0 == 0) {
                    *scale_at = sc;
                    if (older) s_ratio = was / sc;
                }
                #pragma unroll
                for (int r = 0; r < NR; r++)
                    if (live(r)) {
                        #pragma unroll
                        for (int k = 0; k < PP; k++) {
                            uint8_t *col = s_code + (l * PP + k) * COL + 4 * NB * (r0 + r) + 4 * (wave / WB) + i;
                            col[0] = (uint8_t)code_of(x[r][0][k], inv);
                            col[H2 * COL] = (uint8_t)code_of(x[r][1][k], inv);
                        }
                    }
            }
            __syncthreads();
            const float ratio = s_ratio;                              // of the codes that the first block has already
            const int old0 = first / BLOCK8 * BLOCK8;
            // NB words of four positions each, 4 g .. of NB neighbouring blocks
            for (int id = threadIdx.x; id < HD * 4; id += NT) {
                const int d = id >> 2, g = id & 3;
                uint32_t w[NB];
                const uint32_t *from = (const uint32_t *)(s_code + d * COL + 4 * NB * g);
                KVD_GLOBAL uint32_t *dst = gmem((uint32_t *)(page + ((size_t)a.n_kv_heads + h) * PAGE * HD + (size_t)d * PAGE + 16 * g + (NB == 1 ? 4 * u : 0)));
                uint32_t fresh = 0, again = 0;                        // bytes to write, bytes to round again
                #pragma unroll
                for (int k = 0; k < 4 * NB; k++) {
                    const int p = p0 + (k >> 2) * 16 + 4 * g + (k & 3);
                    fresh |= (uint32_t)(p >= first && p < end) << k;
                    again |= (uint32_t)(p >= old0 && p < first && ratio != 1.0f) << k;
                }
                if (!(fresh | again)) continue;
                #pragma unroll
                for (int k = 0; k < NB; k++) w[k] = from[k];
                if (fresh != (1u << 4 * NB) - 1) {
                    uint32_t o[NB];
                    #pragma unroll
                    for (int k = 0; k < NB; k++) o[k] = dst[k];
                    #pragma unroll
                    for (int k = 0; k < 4 * NB; k++) {
                        const int sh = 8 * (k & 3);
                        uint32_t b = o[k >> 2] >> sh & 255;
                        if (again >> k & 1) b = recode(b, ratio);
                        if (!(fresh >> k & 1)) w[k >> 2] = (w[k >> 2] & ~(255u << sh)) | b << sh;
                    }
                }
                if constexpr (NB == 4) *(KVD_GLOBAL v4u *)dst = (v4u){w[0], w[1], w[2], w[3]};
                else dst[0] = w[0];
            }
        }
        return;
    }
    // q or k: norm and rotation
    const float *nw = kind ? a.k_norm : a.q_norm;
    float w[2][PP];
    double c[PP], sn[PP], cs[PP], ss[PP], y[B8 ? NR : 1][2 * PP];         // 8-bit rows wait for their block's scale
    if (nw) {
        #pragma unroll
        for (int k = 0; k < PP; k++) { w[0][k] = gmem(nw)[l * PP + k]; w[1][k] = gmem(nw)[H2 + l * PP + k]; }
    }
    // the first round with tokens, from whose sines the others' are turned
    const int rounds0 = max((first - b0) / 4 - r0, 0);
    v2d *s_sin = (v2d *)s_code;                                            // [position][pair % PP][pair / PP]: a row of lanes reads 256 bytes
    if (a.freq) {
        if constexpr (HG > 1) {
            for (int id = threadIdx.x; id < 4 * H2; id += NT) {
                const int pair = id % H2, at = id / H2 * H2 + pair % PP * 16 + pair / PP;
                const double f = gmem(a.freq)[pair];
                double c0, s0, c4, s4;
                turn((double)(b0 + id / H2) * f, c0, s0);
                turn(4.0 * f, c4, s4);
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    s_sin[at + 4 * r * H2] = (v2d){c0, s0};
                    const double t = fma(c0, c4, -(s0 * s4));
                    s0 = fma(c0, s4, s0 * c4);
                    c0 = t;
                }
            }
            __syncthreads();
        } else {
            #pragma unroll
            for (int k = 0; k < PP; k++) turn((double)(b0 + 4 * (r0 + rounds0) + i) * gmem(a.freq)[l * PP + k], c[k], sn[k]);
            if (rounds0 + 1 < NR && round_live(rounds0 + 1)) {            // the step's are the same in all four rows: each forms a part
                constexpr int PART = PP > 4 ? PP / 4 : 1, ROWS_OF = PP / PART;
                double cp[PART], sp[PART];
                #pragma unroll
                for (int k = 0; k < PART; k++) turn(4.0 * gmem(a.freq)[l * PP + i % ROWS_OF * PART + k], cp[k], sp[k]);
                #pragma unroll
                for (int k = 0; k < PP; k++) {
                    cs[k] = __shfl(cp[k % PART], k / PART * 16 + l, 64);
                    ss[k] = __shfl(sp[k % PART], k / PART * 16 + l, 64);
                }
            }
        }
    }
    T *back = (T *)(kind ? a.k_out : a.q_out);
    const int64_t back_stride = kind ? a.k_out_stride : a.q_out_stride;
    double big = 0.0, none = 0.0;                                          // none: NaN if some value is not finite
    #pragma unroll
    for (int r = 0; r < NR; r++) {
        double (&v)[2 * PP] = y[B8 ? r : 0];
        if (HG == 1 && r > rounds0 && a.freq) {
            #pragma unroll
            for (int k = 0; k < PP; k++) {
                const double t = fma(c[k], cs[k], -(sn[k] * ss[k]));
                sn[k] = fma(c[k], ss[k], sn[k] * cs[k]);
                c[k] = t;
            }
        }
        if ((NB == 1 || WB > 1) && !round_live(r)) continue;
        if (HG > 1 && a.freq) {
            #pragma unroll
            for (int k = 0; k < PP; k++) {
                const v2d z = s_sin[(4 * (r0 + r) + i) * H2 + k * 16 + l];
                c[k] = z[0]; sn[k] = z[1];
            }
        }
        #pragma unroll
        for (int k = 0; k < PP; k++) { v[k] = (double)x[r][0][k]; v[PP + k] = (double)x[r][1][k]; }
        if (nw) {
            double q = 0.0;
            #pragma unroll
            for (int k = 0; k < 2 * PP; k++) q = fma(v[k], v[k], q);
            const double m = inv_sqrt(row_sum(q) * (1.0 / HD) + (double)a.eps);
            #pragma unroll
            for (int k = 0; k < PP; k++) { v[k] *= m * (double)w[0][k]; v[PP + k] *= m * (double)w[1][k]; }
        }
        if (a.freq) {
            #pragma unroll
            for (int k = 0; k < PP; k++) {
                const double x0 = v[k], x1 = v[PP + k];
                v[k] = fma(x0, c[k], -(x1 * sn[k]));
                v[PP + k] = fma(x0, sn[k], x1 * c[k]);
            }
        }
        if (!live(r)) continue;
        float z[2 * PP];
        if (back) {
            rounded<T>(v, z);
            put(row_of(back, back_stride, r, h), z);
        }
        if constexpr (B8) {
            #pragma unroll
            for (int k = 0; k < 2 * PP; k++) { big = fmax(big, fabs(v[k])); none = fma(v[k], 0.0, none); }
        } else if (stored) {
            rounded<float>(v, z);
            put((float *)page + ((size_t)h * PAGE + BLOCK8 * u + 4 * (r0 + r) + i) * HD + l * PP, z);
        }
    }
    if constexpr (B8) {
        big = none == none ? big : INFINITY;
        big = bcast63(wave_to63(big, 0.0, [](double p, double q) { return fmax(p, q); }));
        float *scale_at = (float *)(page + (size_t)2 * a.n_kv_heads * PAGE * HD) + h * PAGE_BLOCKS + u;
        const float was = stored && older ? *scale_at : 0.0f;
        if constexpr (WB > 1) {                                            // (all waves, those of q too)
            if (lane == 0) s_big[wave] = big;
            __syncthreads();
            big = fmax(big, s_big[wave ^ 1]);
        }
        if (!stored) return;
        const float sc = block_scale(scale_exp(big), older, was), ratio = was / sc;
        const double inv = 1.0 / (double)sc;
        if (lane == 0 && r0 == 0) *scale_at = sc;
        #pragma unroll
        for (int r = 0; r < NR; r++) {
            const bool again = older && b0 + 4 * (r0 + r) + i < first && ratio != 1.0f;
            if (!live(r) && !again) continue;
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                uint8_t *row = page + ((size_t)h * PAGE + BLOCK8 * u + 4 * (r0 + r) + i) * HD + l * PP + e * H2;
                uint32_t b[(PP + 3) / 4];
                #pragma unroll
                for (int k = 0; k < PP; k++) {
                    const uint32_t code = again ? recode(gmem(row)[k], ratio) : code_of(y[r][e * PP + k], inv) & 255;
                    b[k / 4] = k % 4 ? b[k / 4] | code << 8 * (k % 4) : code;
                }
                if constexpr (PP == 2) *gmem((uint16_t *)row) = (uint16_t)b[0];
                else if constexpr (PP == 4) *gmem((uint32_t *)row) = b[0];
                else *gmem((v2u *)row) = (v2u){b[0], b[1]};
            }
        }
    }
}

// Units of positions that a call's tokens may fall into: with few tokens a sequence every sequence's
// most, else by the packed tokens (a unit and its neighbour more for each sequence).
int64_t append_slots(const sp_hipkv_append_args &a, int unit, int *seq_units) {
    const int64_t most = ((int64_t)a.max_tokens + unit - 2) / unit + 1, packed = (int64_t)a.n_tokens / unit + 2 * a.n_seqs;
    *seq_units = most * a.n_seqs <= packed ? (int)most : 0;
    return *seq_units ? most * a.n_seqs : packed;
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

template <typename T, int ROWS, int NB> hipError_t append_go(const sp_hipkv_append_args &a, hipStream_t s) {
    int seq_units = 0;
    const int64_t slots = append_slots(a, BLOCK8 * NB, &seq_units);
    return op_launch(a.head_dim == 256 ? k_append<T, ROWS, 256, NB> : a.head_dim == 128 ? k_append<T, ROWS, 128, NB> : k_append<T, ROWS, 64, NB>,
                     dim3(append_qk<NB>(a) + a.n_kv_heads, (uint32_t)slots), dim3(64 * NB * block_waves(ROWS, a.head_dim)), s, a, seq_units);
}
template <typename T, int ROWS> hipError_t append_rows(const sp_hipkv_append_args &a, hipStream_t s) {
    return a.max_tokens <= BLOCK8 ? append_go<T, ROWS, 1>(a, s) : append_go<T, ROWS, 4>(a, s);
}

}  // namespace

hipError_t launch_append(const sp_hipkv_append_args &a, hipStream_t s) {
    if (a.rows == SP_HIPKV_ROWS_F32) return a.type == SP_HIPKV_F32 ? append_rows<float, SP_HIPKV_ROWS_F32>(a, s) : append_rows<Bf16, SP_HIPKV_ROWS_F32>(a, s);
    return a.type == SP_HIPKV_F32 ? append_rows<float, SP_HIPKV_ROWS_BLOCK8>(a, s) : append_rows<Bf16, SP_HIPKV_ROWS_BLOCK8>(a, s);
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
