// kvd_prompt.hip -- attention of whole prompts: packed sequences, causal, grouped heads.
//
// The q heads of a kv head share its K and V: the rows of one kv head are r = token G + q
// head of the group, 32 to a matrix tile, QT tiles to a wave, 4 waves to a workgroup, which walk the
// K and V tiles of their rows' span in step, with a running maximum and sum.
//
// Both products are made transposed: S^T = K Q^T (K the A operand, from LDS; Q the B
// operand, in registers), then O^T += V^T P^T.  A lane then holds scores, weights,
// maximum, sum and output of one row, l % 32, shared with lane l ^ 32: no reduction but one
// exchange of halves, and the weights go from one product to the next in registers: the
// 16 scores of a 32 x 32 tile are keys 8 (i / 4) + 4 half + i % 4, and the second product takes its
// keys in that order, V^T fragments coming from row-major LDS by transposing reads.
//
// bf16: weights are rounded to bf16 before the second product, an error of the size of the
// output's own rounding (sqrt 2 of it together); the sum adds them unrounded.
// f32: K, V, q and weights as three bf16 pieces, six products each (kvd_pieces.h).
//
// The running maximum only moves when a score exceeds it by 2^16 in the exponent: weights
// stay below 2^16, nothing is lost below sums of 2^128 (v of 2^90 over 2^20 tokens), and most tiles leave the
// output unscaled.  With 2^8, scores of a standard deviation of 4.5 had some row of 32 move in every
// eighth tile of 8192 tokens, 90 us of 640.
//
// A key that a row does not attend has weight 0, which a V value that is not finite would turn
// into NaN: tiles that some row does not attend whole are staged with zeros in place of such
// values, and rows that attend them get them afterwards.
#include "kvd_serve.h"
#include "kvd_pass.h"
#include <algorithm>

namespace kvd {

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds4s;
constexpr float LOG2E_F = 1.44269504088896341f;

constexpr float SLACK = 16.0f;                                           // exponent (base 2) that a weight may reach

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

template <typename T, int HD> struct PromptShape {
    static constexpr int NP = sizeof(T) == 4 ? 3 : 1, BN = NP == 3 ? 32 : 64;
    static constexpr int QT = 1, BM = 128 * QT;
    static constexpr int WPS = NP == 3 && HD == 256 ? 1 : HD == 256 ? 1 : 2;             // waves a SIMD
};

// eight staged values: f32 as they are, bf16 as bits
template <typename T> struct Chunk;
template <> struct Chunk<float> { v4f a, b; };
template <> struct Chunk<Bf16> { v4u a; };
__device__ __forceinline__ void chunk_load(Chunk<float> &c, const float *p) { c.a = *gmem((const v4f *)p); c.b = *gmem((const v4f *)(p + 4)); }
__device__ __forceinline__ void chunk_load(Chunk<Bf16> &c, const Bf16 *p) { c.a = *gmem((const v4u *)p); }
__device__ __forceinline__ void chunk_zero(Chunk<float> &c) { c.a = c.b = (v4f){0, 0, 0, 0}; }
__device__ __forceinline__ void chunk_zero(Chunk<Bf16> &c) { c.a = (v4u){0, 0, 0, 0}; }
// zeros in place of values that are not finite; whether there were any
__device__ __forceinline__ bool chunk_clean(Chunk<float> &c) {
    bool bad = false;
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        const bool x = !pieces_hold(c.a[k]), y = !pieces_hold(c.b[k]);
        bad |= x | y;
        c.a[k] = x ? 0.0f : c.a[k]; c.b[k] = y ? 0.0f : c.b[k];
    }
    return bad;
}
__device__ __forceinline__ bool bf16_finite(uint32_t u) { return (u & 0x7F80) != 0x7F80; }
__device__ __forceinline__ bool chunk_clean(Chunk<Bf16> &c) {
    bool bad = false;
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        const bool x = !bf16_finite(c.a[k]), y = !bf16_finite(c.a[k] >> 16);
        bad |= x | y;
        c.a[k] &= (x ? 0xFFFF0000u : ~0u) & (y ? 0xFFFFu : ~0u);
    }
    return bad;
}
__device__ __forceinline__ void chunk_pieces(const Chunk<float> &c, bf8 (&p)[3]) {
    const Pieces x = pieces_of([&](int k) { return k < 4 ? c.a[k & 3] : c.b[k & 3]; });
    p[0] = x.p[0]; p[1] = x.p[1]; p[2] = x.p[2];
}
__device__ __forceinline__ void chunk_pieces(const Chunk<Bf16> &c, bf8 (&p)[1]) { p[0] = __builtin_bit_cast(bf8, c.a); }

template <typename T, int HD>
__global__ __launch_bounds__(256, (PromptShape<T, HD>::WPS)) void k_prompt(sp_hipkv_prompt_args a, int slots) {
    using P = PromptShape<T, HD>;
    constexpr int NP = P::NP, BN = P::BN, QT = P::QT, BM = P::BM, KT = BN / 32, DT = HD / 32, C8 = HD / 8, NC = BN * C8 / 256;
    constexpr int NMUL = NP == 3 ? 6 : 1;
    __shared__ __align__(1024) bf8 s_k[NP * BN * C8], s_v[NP * BN * C8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int G = a.n_heads / a.n_kv_heads, h = blockIdx.x % a.n_kv_heads;
    // the longest spans first: a sequence's last rows before its first
    const int slot = slots - 1 - blockIdx.x / a.n_kv_heads;
    const int s = unit_seq(a.start, a.n_seqs, slot, G, BM, 1);
    const int t0 = max(gmem(a.start)[s], 0), n = min(min(gmem(a.start)[s + 1], a.n_tokens) - t0, a.max_tokens);
    const int64_t j = slot - unit_base(a.start, s, G, BM, 1);
    if (n <= 0 || j < 0 || j * BM >= (int64_t)n * G) return;
    const int R = n * G, r0 = (int)j * BM, wr0 = r0 + wave * 32 * QT;
    // tokens of the workgroup and of this wave, and the keys that they attend
    const int W = a.window ? a.window : INT32_MAX;
    const int first = r0 / G, last = (min(r0 + BM, R) - 1) / G, w_first = min(wr0, R - 1) / G, w_last = (min(wr0 + 32 * QT, R) - 1) / G;
    const int k0 = max(first - W + 1, 0) / BN, k1 = last / BN + 1;
    // scale <= 0 goes into q's sign (or makes q zero), so that larger scores have larger weights
    const float sgn = a.scale > 0 ? 1.0f : a.scale < 0 ? -1.0f : 0.0f, c = a.scale == 0 ? LOG2E_F : fabsf(a.scale) * LOG2E_F, slack = SLACK / c;
    int tok[QT];
    bf8 Q[QT][HD / 16][NP];
    #pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = min(wr0 + t * 32 + l32, R - 1);
        tok[t] = r / G;
        const T *q = (const T *)a.q + (size_t)(t0 + tok[t]) * a.q_stride + (size_t)(h * G + r % G) * HD + 8 * half;
        #pragma unroll
        for (int k = 0; k < HD / 16; k++) {
            float x[8];
            load_values(q + 16 * k, x);
            Chunk<float> f = {{x[0] * sgn, x[1] * sgn, x[2] * sgn, x[3] * sgn}, {x[4] * sgn, x[5] * sgn, x[6] * sgn, x[7] * sgn}};
            if constexpr (NP == 3) chunk_pieces(f, Q[t][k]);
            else {
                Chunk<Bf16> b = {{bf16x2(f.a[0], f.a[1]), bf16x2(f.a[2], f.a[3]), bf16x2(f.b[0], f.b[1]), bf16x2(f.b[2], f.b[3])}};
                chunk_pieces(b, Q[t][k]);
            }
        }
    }
    // A row's 16-byte chunks lie in an order that spreads a column of K over the banks, and
    // the 64-byte runs of four rows of V
    auto k_at = [](int row, int ch) { return row * C8 + (HD == 64 ? ch ^ (row >> 1 & 7) : ch ^ (row & 15)); };
    auto v_at = [](int row, int ch) { return row * C8 + (HD == 64 ? ch ^ (row >> 1 & 1) << 2 : ch ^ (row & 3) << 2); };
    const T *kp = (const T *)a.k + (size_t)t0 * a.k_stride + (size_t)h * HD, *vp = (const T *)a.v + (size_t)t0 * a.v_stride + (size_t)h * HD;
    Chunk<T> ck[NC], cv[NC];
    auto load = [&](int tile) {
        #pragma unroll
        for (int k = 0; k < NC; k++) {
            const int id = threadIdx.x + 256 * k, row = tile * BN + id / C8, ch = id % C8;
            if (row < n) {
                chunk_load(ck[k], kp + (size_t)row * a.k_stride + 8 * ch);
                chunk_load(cv[k], vp + (size_t)row * a.v_stride + 8 * ch);
            } else { chunk_zero(ck[k]); chunk_zero(cv[k]); }
        }
    };
    auto put = [&](bool clean) {
        bool bad = false;
        #pragma unroll
        for (int k = 0; k < NC; k++) {
            const int id = threadIdx.x + 256 * k, row = id / C8, ch = id % C8;
            bf8 p[NP];
            chunk_pieces(ck[k], p);
            #pragma unroll
            for (int e = 0; e < NP; e++) s_k[e * BN * C8 + k_at(row, ch)] = p[e];
            if (clean) bad |= chunk_clean(cv[k]);
            chunk_pieces(cv[k], p);
            #pragma unroll
            for (int e = 0; e < NP; e++) s_v[e * BN * C8 + v_at(row, ch)] = p[e];
        }
        return bad;
    };
    v16f O[QT][DT];
    float m[QT], l[QT];
    #pragma unroll
    for (int t = 0; t < QT; t++) {
        m[t] = -INFINITY; l[t] = 0.0f;
        #pragma unroll
        for (int d = 0; d < DT; d++)
            #pragma unroll
            for (int i = 0; i < 16; i++) O[t][d][i] = 0.0f;
    }
    // this lane's address for the transposing reads: row (l % 16) / 4 of four, 4 columns of 16
    const int v_row = 4 * half + (lane & 15) / 4, v_col = 16 * (lane >> 4 & 1) + 4 * (lane & 3);
    load(k0);
    for (int tile = k0; tile < k1; tile++) {
        const int key0 = tile * BN;
        const bool ragged = key0 + BN - 1 > first || key0 < last - W + 1;               // some row does not attend it whole
        const bool flag = put(ragged);
        bool odd = false;
        if (ragged) odd = __syncthreads_or(flag); else __syncthreads();
        if (tile + 1 < k1) load(tile + 1);
        if (wr0 < R && key0 <= w_last && key0 + BN > w_first - W + 1) {
            const bool w_ragged = key0 + BN - 1 > w_first || key0 < w_last - W + 1;
            v16f S[QT][KT];
            #pragma unroll
            for (int t = 0; t < QT; t++)
                #pragma unroll
                for (int u = 0; u < KT; u++)
                    #pragma unroll
                    for (int i = 0; i < 16; i++) S[t][u][i] = 0.0f;
            #pragma unroll
            for (int k = 0; k < HD / 16; k++)
                #pragma unroll
                for (int u = 0; u < KT; u++) {
                    bf8 A[NP];
                    #pragma unroll
                    for (int e = 0; e < NP; e++) A[e] = s_k[e * BN * C8 + k_at(u * 32 + l32, 2 * k + half)];
                    #pragma unroll
                    for (int t = 0; t < QT; t++)
                        #pragma unroll
                        for (int x = 6 - NMUL; x < 6; x++) S[t][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[MUL_A[x]], Q[t][k][MUL_B[x]], S[t][u], 0, 0, 0);
                }
            bf8 Pw[QT][KT][2][NP];
            #pragma unroll
            for (int t = 0; t < QT; t++) {
                if (w_ragged) {
                    #pragma unroll
                    for (int u = 0; u < KT; u++)
                        #pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int key = key0 + u * 32 + 8 * (i / 4) + 4 * half + i % 4;
                            S[t][u][i] = key <= tok[t] && key > tok[t] - W ? S[t][u][i] : -INFINITY;
                        }
                }
                float mx = S[t][0][0];
                #pragma unroll
                for (int u = 0; u < KT; u++)
                    #pragma unroll
                    for (int i = 0; i < 16; i++) mx = fmaxf(mx, S[t][u][i]);
                if (__any(mx > m[t] + slack)) {
                    mx = fmaxf(mx, other_half(mx));
                    const float mn = fmaxf(m[t], mx), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m[t] - mn) * c);
                    m[t] = mn;
                    l[t] *= al;
                    #pragma unroll
                    for (int d = 0; d < DT; d++)
                        #pragma unroll
                        for (int i = 0; i < 16; i++) O[t][d][i] *= al;
                }
                const float nm = m[t] == -INFINITY ? 0.0f : -m[t] * c;
                #pragma unroll
                for (int u = 0; u < KT; u++)
                    #pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float w[8];
                        #pragma unroll
                        for (int i = 0; i < 8; i++) {
                            w[i] = __builtin_amdgcn_exp2f(fmaf(S[t][u][8 * e + i], c, nm));
                            l[t] += w[i];
                        }
                        if constexpr (NP == 3) {
                            const Pieces x = pieces_of([&](int k) { return w[k]; });
                            Pw[t][u][e][0] = x.p[0]; Pw[t][u][e][1] = x.p[1]; Pw[t][u][e][2] = x.p[2];
                        } else Pw[t][u][e][0] = __builtin_bit_cast(bf8, (v4u){bf16x2(w[0], w[1]), bf16x2(w[2], w[3]), bf16x2(w[4], w[5]), bf16x2(w[6], w[7])});
                    }
            }
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int u = 0; u < KT; u++)
                    #pragma unroll
                    for (int e = 0; e < 2; e++) {
                        bf8 A[NP];
                        #pragma unroll
                        for (int x = 0; x < NP; x++) {
                            v4s y[2];
                            #pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const int row = u * 32 + 16 * e + 8 * z + v_row, col = d * 32 + v_col;
                                y[z] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)((uint8_t *)(s_v + x * BN * C8 + v_at(row, col / 8)) + col % 8 * 2));
                            }
                            typedef short v8s __attribute__((ext_vector_type(8)));
                            A[x] = __builtin_bit_cast(bf8, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
                        }
                        #pragma unroll
                        for (int t = 0; t < QT; t++)
                            #pragma unroll
                            for (int x = 6 - NMUL; x < 6; x++) O[t][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[MUL_A[x]], Pw[t][u][e][MUL_B[x]], O[t][d], 0, 0, 0);
                    }
            if (odd) {                                                      // V values that were left out, for the rows that attend them
                #pragma unroll 1
                for (int key = key0; key < min(key0 + BN, n); key++) {
                    const T *row = vp + (size_t)key * a.v_stride + 4 * half;
                    #pragma unroll
                    for (int d = 0; d < DT; d++)
                        #pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float x[4];
                            load_values(row + d * 32 + 2 * i, x);
                            #pragma unroll
                            for (int t = 0; t < QT; t++)
                                #pragma unroll
                                for (int y = 0; y < 4; y++) O[t][d][i + y] += key <= tok[t] && key > tok[t] - W && !pieces_hold(x[y]) ? x[y] * INFINITY : 0.0f;
                        }
                }
            }
        }
        __syncthreads();
    }
    #pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = wr0 + t * 32 + l32;
        const float inv = 1.0f / (l[t] + other_half(l[t]));
        if (r >= R) continue;
        T *o = (T *)a.out + (size_t)(t0 + tok[t]) * a.out_stride + (size_t)(h * G + r % G) * HD + 4 * half;
        #pragma unroll
        for (int d = 0; d < DT; d++)
            #pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float x[4];
                #pragma unroll
                for (int y = 0; y < 4; y++) x[y] = O[t][d][i + y] * inv;
                store_values(o + d * 32 + 2 * i, x);
            }
    }
}

// ---------------------------------------------------------------- bf16
// K and V come through LDS by direct loads, two tiles deep, with one barrier a tile.
template <int HD, int NW>
__global__ __launch_bounds__(64 * NW, HD == 256 ? 1 : 2) void k_prompt16(sp_hipkv_prompt_args a, int slots) {
    constexpr int BN = HD == 256 ? 32 : 64, BM = 32 * NW, KT = BN / 32, KS = HD / 16, DT = HD / 32, C8 = HD / 8, TB = BN * HD * 2;      // bytes of a tile
    __shared__ __align__(1024) uint8_t lds[4 * TB];                       // K of even and odd tiles, then V
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int G = a.n_heads / a.n_kv_heads, h = blockIdx.x % a.n_kv_heads;
    // the longest spans first: a sequence's last rows before its first
    const int slot = slots - 1 - blockIdx.x / a.n_kv_heads;
    const int s = unit_seq(a.start, a.n_seqs, slot, G, BM, 1);
    const int t0 = max(gmem(a.start)[s], 0), n = min(min(gmem(a.start)[s + 1], a.n_tokens) - t0, a.max_tokens);
    const int64_t j = slot - unit_base(a.start, s, G, BM, 1);
    if (n <= 0 || j < 0 || j * BM >= (int64_t)n * G) return;
    const int R = n * G, r0 = (int)j * BM, wr0 = r0 + wave * 32;
    const int W = a.window ? a.window : INT32_MAX;
    const int first = r0 / G, last = (min(r0 + BM, R) - 1) / G, w_first = min(wr0, R - 1) / G, w_last = (min(wr0 + 32, R) - 1) / G;
    const int k0 = max(first - W + 1, 0) / BN, k1 = last / BN + 1;
    const float sgn = a.scale > 0 ? 1.0f : a.scale < 0 ? -1.0f : 0.0f, c = a.scale == 0 ? LOG2E_F : fabsf(a.scale) * LOG2E_F, slack = SLACK / c;
    const Bf16 *kp = (const Bf16 *)a.k + (size_t)t0 * a.k_stride + (size_t)h * HD, *vp = (const Bf16 *)a.v + (size_t)t0 * a.v_stride + (size_t)h * HD;
    // Direct loads fill LDS in order; a lane takes the 16-byte chunk whose place that is: chunks of a K
    // row lie in an order that spreads a column over the banks, 64-byte runs of V that of four rows
    constexpr int RPI = 512 / HD, NI = TB / 1024 / NW;                         // rows of one load, loads of a wave for a tile
    auto k_swz = [](int row) { return HD == 64 ? row >> 1 & 7 : row & 15; };
    auto v_swz = [](int row) { return HD == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; };
    int ko[NI], vo[NI];
    #pragma unroll
    for (int i = 0; i < NI; i++) {
        const int row = (wave * NI + i) * RPI + lane / C8, ch = lane % C8;
        ko[i] = (row * (int)a.k_stride + 8 * (ch ^ k_swz(row))) * 2;
        vo[i] = (row * (int)a.v_stride + 8 * (ch ^ v_swz(row))) * 2;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)lds + wave * NI * 1024;
    auto load = [&](const Bf16 *p, int64_t stride, const int (&off)[NI], int tile, int to) {
        const int rows = min(n - tile * BN, BN);
        const v4i rs = rsrc_of(p + (int64_t)tile * BN * stride, rows > 0 ? (uint32_t)((rows - 1) * (int)stride + HD) * 2 : 0);
        #pragma unroll
        for (int i = 0; i < NI; i++) dma16(lds0 + to * TB + i * 1024, off[i], rs);
    };
    load(kp, a.k_stride, ko, k0, 0);
    load(vp, a.v_stride, vo, k0, 2);
    const int row = min(wr0 + l32, R - 1), tok = row / G;
    bf8 Q[KS];
    {
        const Bf16 *q = (const Bf16 *)a.q + (size_t)(t0 + tok) * a.q_stride + (size_t)(h * G + row % G) * HD + 8 * half;
        #pragma unroll
        for (int k = 0; k < KS; k++) {
            float x[8];
            load_values(q + 16 * k, x);
            Q[k] = __builtin_bit_cast(bf8, (v4u){bf16x2(x[0] * sgn, x[1] * sgn), bf16x2(x[2] * sgn, x[3] * sgn), bf16x2(x[4] * sgn, x[5] * sgn), bf16x2(x[6] * sgn, x[7] * sgn)});
        }
    }
    v16f O[DT];
    const v16f zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    #pragma unroll
    for (int d = 0; d < DT; d++) O[d] = zero;
    float m = -INFINITY, l = 0.0f;
    // this lane's places in a tile: of K by dims, of V (row (l % 16) / 4 of four, 4 columns of 16, for the
    // transposing reads) by columns
    int k_at[KS], v_at[DT];
    #pragma unroll
    for (int k = 0; k < KS; k++) k_at[k] = (l32 * C8 + ((2 * k + half) ^ k_swz(l32))) * 16;
    #pragma unroll
    for (int d = 0; d < DT; d++) {
        const int r = 4 * half + (lane & 15) / 4, col = d * 32 + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
        v_at[d] = (r * C8 + ((col / 8) ^ v_swz(r))) * 16 + col % 8 * 2;
    }
    // V values that were left out of a tile, for the rows that attend them
    auto add_odd = [&](int key0) __attribute__((always_inline)) {
        #pragma unroll 1
        for (int key = key0; key < min(key0 + BN, n); key++) {
            const Bf16 *vrow = vp + (size_t)key * a.v_stride + 4 * half;
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float x[4];
                    load_values(vrow + d * 32 + 2 * i, x);
                    #pragma unroll
                    for (int y = 0; y < 4; y++) O[d][i + y] += key <= tok && key > tok - W && !pieces_hold(x[y]) ? x[y] * INFINITY : 0.0f;
                }
        }
    };
    // zeros in LDS in place of V values that are not finite; whether this thread found one
    auto clean = [&](uint8_t *lds) __attribute__((always_inline)) {
        bool bad = false;
        #pragma unroll
        for (int i = 0; i < NI; i++) {
            Chunk<Bf16> x = {((v4u *)lds)[threadIdx.x + 64 * NW * i]};
            if (chunk_clean(x)) { bad = true; ((v4u *)lds)[threadIdx.x + 64 * NW * i] = x.a; }
        }
        return bad;
    };
    auto work = [&](int tile, auto part) __attribute__((always_inline)) {
        constexpr int BUF = part.value;
        const bool ragged = tile * BN + BN - 1 > first || tile * BN < last - W + 1;        // some row does not attend it whole
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        bool odd = false;
        if (ragged) odd = __syncthreads_or(clean(lds + (2 + BUF) * TB));
        if (tile + 1 < k1) {
            load(kp, a.k_stride, ko, tile + 1, 1 - BUF);
            load(vp, a.v_stride, vo, tile + 1, 3 - BUF);
        }
        if (tile * BN > w_last || tile * BN + BN <= w_first - W + 1) return;               // no row of this wave attends any
        // fragments are read 8 products ahead, the first of V beside the last of K
        constexpr int NF = 8, NKF = KT * KS, NVF = KT * 2 * DT;
        v16f S[KT];
        bf8 F[NF];
        auto read_k = [&](int x) { return *(const bf8 *)(lds + k_at[x % KS] + BUF * TB + x / KS * 32 * HD * 2); };
        auto read_v = [&](int x) {
            typedef short v8s __attribute__((ext_vector_type(8)));
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)(lds + v_at[x % DT] + (2 + BUF) * TB + 16 * (x / DT) * HD * 2));
            const v4s z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)(lds + v_at[x % DT] + (2 + BUF) * TB + (16 * (x / DT) + 8) * HD * 2));
            return __builtin_bit_cast(bf8, __builtin_shufflevector(y, z, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        #pragma unroll
        for (int x = 0; x < NF; x++) F[x] = read_k(x);
        __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
        #pragma unroll
        for (int x = 0; x < NKF; x++) {
            S[x / KS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F[x % NF], Q[x % KS], x % KS ? S[x / KS] : zero, 0, 0, 0);
            F[x % NF] = x + NF < NKF ? read_k(x + NF) : read_v(x + NF - NKF);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (x + NF < NKF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        if (tile * BN + BN - 1 > w_first || tile * BN < w_last - W + 1) {
            #pragma unroll
            for (int u = 0; u < KT; u++)
                #pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = tile * BN + u * 32 + 8 * (i / 4) + 4 * half + i % 4;
                    S[u][i] = key <= tok && key > tok - W ? S[u][i] : -INFINITY;
                }
        }
        float mx = S[0][0];
        #pragma unroll
        for (int u = 0; u < KT; u++)
            #pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, S[u][i]);
        if (__builtin_expect(__any(mx > m + slack), 0)) {
            mx = fmaxf(mx, other_half(mx));
            const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            l *= al;
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int i = 0; i < 16; i++) O[d][i] *= al;
        }
        const float nm = m == -INFINITY ? 0.0f : -m * c;
        bf8 P[KT][2];
        #pragma unroll
        for (int u = 0; u < KT; u++)
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                float w[8];
                #pragma unroll
                for (int i = 0; i < 8; i++) {
                    w[i] = __builtin_amdgcn_exp2f(fmaf(S[u][8 * e + i], c, nm));
                    l += w[i];
                }
                P[u][e] = __builtin_bit_cast(bf8, (v4u){bf16x2(w[0], w[1]), bf16x2(w[2], w[3]), bf16x2(w[4], w[5]), bf16x2(w[6], w[7])});
            }
        #pragma unroll
        for (int x = 0; x < NVF; x++) {
            O[x % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F[x % NF], P[x / DT / 2][x / DT % 2], O[x % DT], 0, 0, 0);
            if (x + NF < NVF) F[x % NF] = read_v(x + NF);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (x + NF < NVF) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        if (odd) add_odd(tile * BN);
    };
    for (int tile = k0; tile < k1; tile += 2) {
        work(tile, std::integral_constant<int, 0>{});
        if (tile + 1 < k1) work(tile + 1, std::integral_constant<int, 1>{});
    }
    const int r = wr0 + l32;
    const float inv = 1.0f / (l + other_half(l));
    if (r >= R) return;
    Bf16 *o = (Bf16 *)a.out + (size_t)(t0 + tok) * a.out_stride + (size_t)(h * G + r % G) * HD + 4 * half;
    #pragma unroll
    for (int d = 0; d < DT; d++)
        #pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
            #pragma unroll
            for (int y = 0; y < 4; y++) x[y] = O[d][i + y] * inv;
            store_values(o + d * 32 + 2 * i, x);
        }
}

int prompt_check(const sp_hipkv_prompt_args *a) {
    const char *who = "sp_hipkv_prompt_attention";
    if (serve_check(who, a)) return 1;
    OP_NEED(a->window >= 0, "negative window");
    OP_NEED(std::isfinite(a->scale), "scale is not finite");
    if (!a->n_tokens) return 0;
    OP_NEED(a->start, "null array");
    return serve_rows(who, a, a->q, a->q_stride, a->n_heads) || serve_rows(who, a, a->k, a->k_stride, a->n_kv_heads) ||
           serve_rows(who, a, a->v, a->v_stride, a->n_kv_heads) || serve_rows(who, a, a->out, a->out_stride, a->n_heads);
}

template <typename T, int HD> hipError_t prompt_go(const sp_hipkv_prompt_args &a, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        constexpr int NW = 4;
        const int slots = (int)((int64_t)a.n_tokens * (a.n_heads / a.n_kv_heads) / (32 * NW)) + a.n_seqs;
        return op_launch(k_prompt16<HD, NW>, dim3((uint32_t)((int64_t)slots * a.n_kv_heads)), dim3(64 * NW), s, a, slots);
    }
    const int slots = (int)((int64_t)a.n_tokens * (a.n_heads / a.n_kv_heads) / PromptShape<T, HD>::BM) + a.n_seqs;
    return op_launch(k_prompt<T, HD>, dim3((uint32_t)((int64_t)slots * a.n_kv_heads)), dim3(256), s, a, slots);
}
template <typename T> hipError_t prompt_type(const sp_hipkv_prompt_args &a, hipStream_t s) {
    return a.head_dim == 256 ? prompt_go<T, 256>(a, s) : a.head_dim == 128 ? prompt_go<T, 128>(a, s) : prompt_go<T, 64>(a, s);
}

}  // namespace

hipError_t launch_prompt(const sp_hipkv_prompt_args &a, hipStream_t s) {
    return a.type == SP_HIPKV_F32 ? prompt_type<float>(a, s) : prompt_type<Bf16>(a, s);
}

}  // namespace kvd

extern "C" int sp_hipkv_prompt_attention(const sp_hipkv_prompt_args *a, void *stream) {
    using namespace kvd;
    if (prompt_check(a)) return 1;
    if (!a->n_tokens) return 0;
    OpDevice dev((hipStream_t)stream);
    return op_done("sp_hipkv_prompt_attention", dev.err != hipSuccess ? dev.err : launch_prompt(*a, (hipStream_t)stream));
}
