// kvd_prompt.hip -- attention of whole prompts: packed sequences, causal, grouped heads.
//
// The q heads of a kv head share its K and V: the rows of one kv head are r = token G + q
// head of the group, 32 to a wave, a matrix tile.  The waves of a workgroup walk the K and V tiles of their
// rows' span in step, with a running maximum and sum.
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
// f32: K, V, q and weights as two f16 numbers each, three products (below).
//
// The running maximum only moves when a score exceeds it by 2^16 (f32: 2^8, f16 numbers end
// sooner) in the exponent: weights stay below 2^16, nothing is lost below sums of 2^128 (v of 2^90 over 2^20 tokens), and most tiles leave the
// output unscaled.  With 2^8, scores of a standard deviation of 4.5 had some row of 32 move in every
// eighth tile of 8192 tokens, 90 us of 640.
//
// A key that a row does not attend has weight 0, which a V value that is not finite would turn
// into NaN: tiles that some row does not attend whole are staged with zeros in place of such
// values, and rows that attend them get them afterwards.
#include "kvd_serve.h"
#include "kvd_pass.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds4s;
constexpr float LOG2E_F = 1.44269504088896341f;

constexpr float SLACK = 16.0f;                                           // exponent (base 2) that a weight may reach
// Whether the largest score of a tile moves a row's maximum m.  The slack is infinite where scores weigh next to
// nothing; the first score moves a maximum of -inf then too, as -inf + inf is no number.
__device__ __forceinline__ bool moves(float mx, float m, float slack) { return !(mx <= m + slack); }

// waves that share a row's dims
constexpr int prompt_split(int hd) { return hd == 256 ? 2 : 1; }

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

__device__ __forceinline__ bool bf16_finite(uint32_t u) { return (u & 0x7F80) != 0x7F80; }
// zeros in place of values that are not finite; whether there were any
__device__ __forceinline__ bool chunk_clean(v4u &c) {
    bool bad = false;
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        const bool x = !bf16_finite(c[k]), y = !bf16_finite(c[k] >> 16);
        bad |= x | y;
        c[k] &= (x ? 0xFFFF0000u : ~0u) & (y ? 0xFFFFu : ~0u);
    }
    return bad;
}
__device__ __forceinline__ bool finite32(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// Joins the outputs of the KS parts of RG row groups (maxima m, sums l, exponents by c): of the tiles of 32
// columns each part's wave sums up every KS-th and hands its rows' quotients to put(column tile, index, 4
// values).  Its own share of them stays in registers, the other parts' pass LDS, 4 KiB a tile and wave.
constexpr int join_bytes(int rg, int ks, int dt) { return rg * (ks - 1) * dt * 4096; }
template <int RG, int KS, int DT, typename Put>
__device__ __forceinline__ void join_parts(v16f (&O)[DT], float m, float l, float c, uint8_t *lds, v2f (*s_ml)[32], int wave, int lane, Put &&put) {
    v4f *x = (v4f *)lds;
    const int rg = wave % RG, part = wave / RG;
    auto at = [&](int d, int k, int i) { return (((d * (KS - 1) + k - (k > d % KS)) * RG + rg) * 4 + i) * 64 + lane; };
    auto own = [&](int d, int i) { return (v4f){O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]}; };
    if (lane < 32) s_ml[wave][lane] = (v2f){m, l};
    __syncthreads();                                                       // K and V are read
    #pragma unroll
    for (int d = 0; d < DT; d++)
        if (d % KS != part) {
            #pragma unroll
            for (int i = 0; i < 4; i++) x[at(d, part, i)] = own(d, i);
        }
    __syncthreads();
    float M = -INFINITY, L = 0.0f, f[KS];
    #pragma unroll
    for (int k = 0; k < KS; k++) M = fmaxf(M, s_ml[k * RG + rg][lane & 31][0]);
    #pragma unroll
    for (int k = 0; k < KS; k++) {
        const v2f ml = s_ml[k * RG + rg][lane & 31];
        f[k] = ml[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml[0] - M) * c);
        L += ml[1] == 0.0f ? 0.0f : f[k] * ml[1];                          // NaN sums stay, empty ones add nothing
    }
    const float inv = 1.0f / L;
    #pragma unroll
    for (int d = 0; d < DT; d++)
        if (d % KS == part) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                v4f y = {0, 0, 0, 0};
                #pragma unroll
                for (int k = 0; k < KS; k++) y += (k == d % KS ? own(d, i) : x[at(d, k, i)]) * f[k];
                const float z[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
                put(d, 4 * i, z);
            }
        }
}

// ---------------------------------------------------------------- bf16
// K and V come through LDS by direct loads, two tiles deep, with one barrier a tile.  A workgroup's waves
// are RG row groups of 32 times KS parts of a tile's keys, 32 KT of them each; the parts are joined at the
// end through LDS.  KS > 1 is for calls with too few rows to fill the device, where the way along the keys is what
// takes the time.
//
// Dims of 256 are shared by two waves, as in f32 (below), who hand each other their parts of the scores
// where the tile's K lay: 2000 tokens of 16 heads of 256 take 79 us, 88 with one wave for all
// dims, which leaves one wave a SIMD.
template <int HD, int RG, int KS, int KT>
__global__ __launch_bounds__(64 * RG * KS * prompt_split(HD), 2) void k_prompt16(sp_hipkv_prompt_args a, int slots) {
    constexpr int SP = prompt_split(HD), NW = RG * KS * SP, BN = 32 * KT * KS, BM = 32 * RG, NS = HD / SP / 16, DT = HD / SP / 32, C8 = HD / 8, TB = BN * HD * 2;      // bytes of a tile
    __shared__ __align__(1024) uint8_t lds[4 * TB];                       // K of even and odd tiles, then V
    __shared__ v2f s_ml[KS > 1 ? NW : 1][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int G = a.n_heads / a.n_kv_heads, h = blockIdx.x % a.n_kv_heads;
    // the longest spans first: a sequence's last rows before its first
    const int slot = slots - 1 - blockIdx.x / a.n_kv_heads;
    const UnitSeq seq = unit_seq(a.start, a.n_seqs, slot, G, BM, 1);
    const int t0 = max(seq.start, 0), n = min(min(seq.end, a.n_tokens) - t0, a.max_tokens);
    const int64_t j = slot - unit_base(seq.start, seq.s, G, BM, 1);
    if (n <= 0 || j < 0 || j * BM >= (int64_t)n * G) return;
    const int R = n * G, r0 = (int)j * BM, wr0 = r0 + wave % RG * 32;
    const int part = wave / RG % KS, dim0 = wave / (RG * KS) * (HD / SP);                 // this wave's keys of a tile, and dims
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
    bf8 Q[NS];
    {
        const Bf16 *q = (const Bf16 *)a.q + (size_t)(t0 + tok) * a.q_stride + (size_t)(h * G + row % G) * HD + dim0 + 8 * half;
        #pragma unroll
        for (int k = 0; k < NS; k++) {
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
    int k_at[NS], v_at[DT];
    #pragma unroll
    for (int k = 0; k < NS; k++) k_at[k] = ((part * 32 * KT + l32) * C8 + ((dim0 / 8 + 2 * k + half) ^ k_swz(l32))) * 16;
    #pragma unroll
    for (int d = 0; d < DT; d++) {
        const int r = 4 * half + (lane & 15) / 4, col = dim0 + d * 32 + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
        v_at[d] = ((part * 32 * KT + r) * C8 + ((col / 8) ^ v_swz(r))) * 16 + col % 8 * 2;
    }
    // V values that were left out of a tile, for the rows that attend them
    auto add_odd = [&](int key0) __attribute__((always_inline)) {
        #pragma unroll 1
        for (int key = key0; key < min(key0 + 32 * KT, n); key++) {
            const Bf16 *vrow = vp + (size_t)key * a.v_stride + dim0 + 4 * half;
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float x[4];
                    load_values(vrow + d * 32 + 2 * i, x);
                    #pragma unroll
                    for (int y = 0; y < 4; y++) O[d][i + y] += key <= tok && key > tok - W && !finite32(x[y]) ? x[y] * INFINITY : 0.0f;
                }
        }
    };
    // zeros in LDS in place of V values that are not finite; whether this thread found one
    auto clean = [&](uint8_t *lds) __attribute__((always_inline)) {
        bool bad = false;
        #pragma unroll
        for (int i = 0; i < NI; i++) {
            v4u x = ((v4u *)lds)[threadIdx.x + 64 * NW * i];
            if (chunk_clean(x)) { bad = true; ((v4u *)lds)[threadIdx.x + 64 * NW * i] = x; }
        }
        return bad;
    };
    auto work = [&](int tile, auto buf) __attribute__((always_inline)) {
        constexpr int BUF = buf.value;
        const bool ragged = tile * BN + BN - 1 > first || tile * BN < last - W + 1;        // some row does not attend it whole
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        bool odd = false;
        if (ragged) odd = __syncthreads_or(clean(lds + (2 + BUF) * TB));
        if (tile + 1 < k1) {
            load(kp, a.k_stride, ko, tile + 1, 1 - BUF);
            load(vp, a.v_stride, vo, tile + 1, 3 - BUF);
        }
        const int key0 = tile * BN + part * 32 * KT;                                       // this wave's keys
        const bool idle = key0 > w_last || key0 + 32 * KT <= w_first - W + 1;              // none that a row of it attends
        if (SP == 1 && idle) return;
        // fragments are read up to 8 products ahead, the first of V beside the last of K
        constexpr int NKF = KT * NS, NVF = KT * 2 * DT, NF = NKF < 8 ? NKF : 8;
        static_assert(NF <= NVF, "the first NF fragments of V");
        v16f S[KT];
        bf8 F[NF];
        auto read_k = [&](int x) { return *(const bf8 *)(lds + k_at[x % NS] + BUF * TB + x / NS * 32 * HD * 2); };
        auto read_v = [&](int x) {
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)(lds + v_at[x % DT] + (2 + BUF) * TB + 16 * (x / DT) * HD * 2));
            const v4s z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)(lds + v_at[x % DT] + (2 + BUF) * TB + (16 * (x / DT) + 8) * HD * 2));
            return __builtin_bit_cast(bf8, __builtin_shufflevector(y, z, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        #pragma unroll
        for (int x = 0; x < NF; x++) F[x] = read_k(x);
        __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
        #pragma unroll
        for (int x = 0; x < NKF; x++) {
            S[x / NS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F[x % NF], Q[x % NS], x % NS ? S[x / NS] : zero, 0, 0, 0);
            F[x % NF] = x + NF < NKF ? read_k(x + NF) : read_v(x + NF - NKF);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (x + NF < NKF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        if constexpr (SP == 2) {                                           // both waves' parts of the scores, in the tile's K
            static_assert(KT * KS == 1 && NW * 4096 <= TB, "a tile of 32 keys, whose K the waves' parts fit");
            __syncthreads();
            v4f *x = (v4f *)(lds + BUF * TB);
            #pragma unroll
            for (int i = 0; i < 4; i++) x[(wave * 4 + i) * 64 + lane] = (v4f){S[0][4 * i], S[0][4 * i + 1], S[0][4 * i + 2], S[0][4 * i + 3]};
            __syncthreads();
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const v4f y = x[((wave ^ RG) * 4 + i) * 64 + lane];
                #pragma unroll
                for (int e = 0; e < 4; e++) S[0][4 * i + e] += y[e];
            }
            if (idle) return;
        }
        if (key0 + 32 * KT - 1 > w_first || key0 < w_last - W + 1) {
            #pragma unroll
            for (int u = 0; u < KT; u++)
                #pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = key0 + u * 32 + 8 * (i / 4) + 4 * half + i % 4;
                    S[u][i] = key <= tok && key > tok - W ? S[u][i] : -INFINITY;
                }
        }
        float mx = S[0][0];
        #pragma unroll
        for (int u = 0; u < KT; u++)
            #pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, S[u][i]);
        if (__builtin_expect(__any(moves(mx, m, slack)), 0)) {
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
        if (odd) add_odd(key0);
    };
    for (int tile = k0; tile < k1; tile += 2) {
        work(tile, std::integral_constant<int, 0>{});
        if (tile + 1 < k1) work(tile + 1, std::integral_constant<int, 1>{});
    }
    l += other_half(l);
    const int r = wr0 + l32;
    Bf16 *o = (Bf16 *)a.out + (size_t)(t0 + r / G) * a.out_stride + (size_t)(h * G + r % G) * HD + dim0 + 4 * half;
    if constexpr (KS == 1) {
        // Rows pass LDS, so that a store instruction writes whole rows and not 8 bytes of each of 32 (nine sequences of
        // 64 to 1000 tokens of 32 and 8 heads of 128: 62 us for 64.5)
        const float inv = 1.0f / l;
        constexpr int CW = HD / SP / 8;                                    // 16-byte chunks of a row of this wave's
        static_assert(NW * 32 * CW * 16 <= 4 * TB, "the waves' rows");
        uint8_t *own = lds + wave * 32 * CW * 16;
        __syncthreads();                                                   // K and V are read
        #pragma unroll
        for (int d = 0; d < DT; d++)
            #pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(v2u *)(own + (l32 * CW + ((4 * d + i / 4) ^ (l32 & (CW - 1)))) * 16 + 8 * half) = (v2u){bf16x2(O[d][i] * inv, O[d][i + 1] * inv), bf16x2(O[d][i + 2] * inv, O[d][i + 3] * inv)};
        __builtin_amdgcn_wave_barrier();
        #pragma unroll
        for (int i = 0; i < CW / 2; i++) {
            const int y = (i * 64 + lane) / CW, ch = lane % CW, to = wr0 + y;
            const v4u x = *(const v4u *)(own + (y * CW + (ch ^ (y & (CW - 1)))) * 16);
            if (to < R) *gmem((v4u *)((Bf16 *)a.out + (size_t)(t0 + to / G) * a.out_stride + (size_t)(h * G + to % G) * HD + dim0 + 8 * ch)) = x;
        }
    } else {
        static_assert(join_bytes(RG, KS, DT) <= 4 * TB, "the parts' outputs");
        join_parts<RG, KS, DT>(O, m, l, c, lds, s_ml, wave, lane, [&](int d, int i, const float (&x)[4]) {
            if (r < R) store_values(o + d * 32 + 2 * i, x);
        });
    }
}

// ---------------------------------------------------------------- f32
// An f32 as two f16: h, its rounding, and l, that of what is left, of values times the power of two
// that brings their row's largest to 2^14 .. 2^15: x = h + l but for 2^-22 of itself, or 2^-39 of the largest.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
struct Halves { h8 h, l; };
template <typename X> __device__ __forceinline__ Halves halves_of(X &&x) {                 // of x(0) .. x(7)
    v4u h, l;
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        const float a = x(2 * k), b = x(2 * k + 1);
        const h2 y = __builtin_convertvector((v2f){a, b}, h2);
        h[k] = __builtin_bit_cast(uint32_t, y);
        // a - h as one instruction each (the compiler takes two)
        float c, d;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(c) : "v"(h[k]), "v"(a));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h[k]), "v"(b));
        l[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){c, d}, h2));
    }
    return {__builtin_bit_cast(h8, h), __builtin_bit_cast(h8, l)};
}
// of a row's largest magnitude the exponent e (`least` at least), and of that the factor 2^(141 - e) and its inverse
__device__ __forceinline__ uint32_t row_exp(float big, uint32_t least = 16) { return min(max(__float_as_uint(big) >> 23, least), 254u); }
__device__ __forceinline__ float row_up(uint32_t e) { return __uint_as_float((268u - e) << 23); }
__device__ __forceinline__ float row_down(uint32_t e) { return __uint_as_float((e - 14u) << 23); }
// the largest over N = 8, 16 or 32 neighbouring lanes, of numbers that are not negative (as bits: one instruction a step)
template <int N> __device__ __forceinline__ float lanes_max(float y) {
    uint32_t x = __float_as_uint(y);
    auto step = [&](auto ctrl) { x = max(x, dpp32<decltype(ctrl)::value, 0xF>(x, 0)); };
    step(std::integral_constant<int, 0xB1>{});                            // quad_perm 1,0,3,2
    step(std::integral_constant<int, 0x4E>{});                            // quad_perm 2,3,0,1
    step(std::integral_constant<int, 0x141>{});                           // row_half_mirror
    if constexpr (N > 8) step(std::integral_constant<int, 0x140>{});      // row_mirror
    if constexpr (N > 16) {
        const v2u z = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(x, x, false, false));
        x = max(z[0], z[1]);
    }
    return __uint_as_float(x);
}
__device__ __forceinline__ float abs_max(const v4f &a, const v4f &b) {
    return fmaxf(fmaxf(fmaxf(fabsf(a[0]), fabsf(a[1])), fmaxf(fabsf(a[2]), fabsf(a[3]))), fmaxf(fmaxf(fabsf(b[0]), fabsf(b[1])), fmaxf(fabsf(b[2]), fabsf(b[3]))));
}
__device__ __forceinline__ v16f mfma_halves(const Halves &a, const Halves &b, v16f c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.l, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}

// A tile of 32 KS keys comes into LDS as it is, by direct loads, while the one before is worked on, and is
// taken apart by all threads: rows of K and of V each by a factor of their own, whose inverses join the
// scores and the weights.  The weights so become numbers of V's range, of which f16 pairs hold 2^-32 of the
// largest that a row of q has met: each has a factor 2^ge of its own for them, which (as the scores'
// maximum does) moves when they leave the range that it leaves them, with the output.  One factor for
// all rows would let a large V that one row attends, or none, take the others' bits.
//
// Dims of 256 are shared by two waves, each 128 of the scores' products and of the output's columns,
// who hand each other their parts of the scores through LDS, where K lay as it came (the next K is
// sent for after that): one wave with all of them needs over 256 registers, so that a SIMD has no other
// to work while it waits (2047 tokens of 16 and 8 heads with a window of 1024: 200 us; so 178, 167
// at the rate of a library's f32 product, 62 at a third of the bf16 one's).  Two waves a SIMD leave 256 registers: nine are
// spilled here and where 128 dims are in two parts, seven where they are in one.
template <int HD, int RG, int KS>
__global__ __launch_bounds__(64 * RG * KS * prompt_split(HD), 2) void k_prompt32(sp_hipkv_prompt_args a, int slots) {
    constexpr int SPLIT = prompt_split(HD), NW = RG * KS * SPLIT, BN = 32 * KS, BM = 32 * RG, NS = HD / SPLIT / 16, DT = HD / SPLIT / 32, C8 = HD / 8, RAW = BN * HD * 4, PIECE = BN * HD * 2, NC = BN * C8 / (64 * NW);
    constexpr float SLACK32 = 8.0f;                                       // weights times 2^7 are f16 numbers
    __shared__ __align__(1024) uint8_t raw[2 * RAW + 4 * PIECE];          // K, V; K's h and l, V's h and l
    __shared__ __align__(16) float s_kf[BN], s_vf[BN];
    __shared__ v2f s_ml[KS > 1 ? NW : 1][32];
    uint8_t *lds = raw + 2 * RAW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int G = a.n_heads / a.n_kv_heads, h = blockIdx.x % a.n_kv_heads;
    // the longest spans first: a sequence's last rows before its first
    const int slot = slots - 1 - blockIdx.x / a.n_kv_heads;
    const UnitSeq seq = unit_seq(a.start, a.n_seqs, slot, G, BM, 1);
    const int t0 = max(seq.start, 0), n = min(min(seq.end, a.n_tokens) - t0, a.max_tokens);
    const int64_t j = slot - unit_base(seq.start, seq.s, G, BM, 1);
    if (n <= 0 || j < 0 || j * BM >= (int64_t)n * G) return;
    const int R = n * G, r0 = (int)j * BM, wr0 = r0 + wave % RG * 32;
    const int part = wave / RG % KS, dim0 = wave / (RG * KS) * (HD / SPLIT);              // this wave's keys of a tile, and dims
    const int W = a.window ? a.window : INT32_MAX;
    const int first = r0 / G, last = (min(r0 + BM, R) - 1) / G, w_first = min(wr0, R - 1) / G, w_last = (min(wr0 + 32, R) - 1) / G;
    const int k0 = max(first - W + 1, 0) / BN, k1 = last / BN + 1;
    const float *kp = (const float *)a.k + (size_t)t0 * a.k_stride + (size_t)h * HD, *vp = (const float *)a.v + (size_t)t0 * a.v_stride + (size_t)h * HD;
    constexpr int NI = RAW / 1024 / NW;                                   // loads of a wave for a tile
    int ko[NI], vo[NI];
    #pragma unroll
    for (int i = 0; i < NI; i++) {
        // of a row first the even 16 bytes, then the odd: a thread's 32 bytes are then read without bank conflicts
        const int at = (wave * NI + i) * 64 + lane, r = at / (2 * C8), p = at % (2 * C8), unit = p < C8 ? 2 * p : 2 * (p - C8) + 1;
        ko[i] = (r * (int)a.k_stride + 4 * unit) * 4;
        vo[i] = (r * (int)a.v_stride + 4 * unit) * 4;
    }
    const uint32_t raw0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)raw + wave * NI * 1024;
    auto load = [&](const float *p, int64_t stride, const int (&off)[NI], int tile, int to) __attribute__((always_inline)) {
        const int rows = min(n - tile * BN, BN);
        const v4i rs = rsrc_of(p + (int64_t)tile * BN * stride, rows > 0 ? (uint32_t)((rows - 1) * (int)stride + HD) * 4 : 0);
        #pragma unroll
        for (int i = 0; i < NI; i++) dma16(raw0 + to + i * 1024, off[i], rs);
    };
    load(kp, a.k_stride, ko, k0, 0);
    load(vp, a.v_stride, vo, k0, RAW);
    // q's halves; its factor joins that of the scores, c >= 0 (scale <= 0 goes into q's sign, or makes q zero)
    const float sgn = a.scale > 0 ? 1.0f : a.scale < 0 ? -1.0f : 0.0f;
    const int row = min(wr0 + l32, R - 1), tok = row / G;
    Halves Q[NS];
    float c;
    {
        const float *q = (const float *)a.q + (size_t)(t0 + tok) * a.q_stride + (size_t)(h * G + row % G) * HD + dim0 + 8 * half;
        float x[NS][8];
        float big = 0.0f;                                                  // (a NaN makes its own way into the scores)
        #pragma unroll
        for (int k = 0; k < NS; k++) load_values(q + 16 * k, x[k]);
        #pragma unroll
        for (int k = 0; k < NS; k++)
            #pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[k][i]));
        big = fmaxf(big, other_half(big));
        if constexpr (SPLIT == 2) {                                        // one factor for both parts of a row
            ((float *)lds)[wave * 32 + l32] = big;
            __syncthreads();
            big = fmaxf(big, ((float *)lds)[(wave ^ RG * KS) * 32 + l32]);
            __syncthreads();
        }
        // (the least exponent keeps c from vanishing, which would make NaN of a masked score, -inf x 0: c is 2^-126 or more, of a
        // scale that is no normal number 2^-148; what a row of q so loses is below 2^-142 |k| in a score)
        const uint32_t e = row_exp(big, max(142 - (int)(__float_as_uint(a.scale) >> 23 & 255), 16));
        const float up = sgn * row_up(e);
        c = (a.scale == 0 ? LOG2E_F : fabsf(a.scale) * LOG2E_F) * row_down(e);
        #pragma unroll
        for (int k = 0; k < NS; k++) Q[k] = halves_of([&](int i) { return x[k][i] * up; });
    }
    const float slack = SLACK32 / c;
    v16f O[DT];
    const v16f zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    #pragma unroll
    for (int d = 0; d < DT; d++) O[d] = zero;
    float m = -INFINITY, l = 0.0f;
    float tm = 0.0f;                                                       // the largest weight times factor of V so far
    int ge = 126;                                                          // O is relative to 2^-ge
    // A row's 16-byte chunks lie in an order that spreads a column of K over the banks, and
    // the 64-byte runs of four rows of V
    auto k_swz = [](int r) { return HD == 64 ? r >> 1 & 7 : r & 15; };
    auto v_swz = [](int r) { return HD == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2; };
    int k_at[NS], v_at[DT];
    #pragma unroll
    for (int k = 0; k < NS; k++) k_at[k] = ((part * 32 + l32) * C8 + ((dim0 / 8 + 2 * k + half) ^ k_swz(l32))) * 16;
    #pragma unroll
    for (int d = 0; d < DT; d++) {
        const int r = 4 * half + (lane & 15) / 4, col = dim0 + d * 32 + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
        v_at[d] = ((part * 32 + r) * C8 + ((col / 8) ^ v_swz(r))) * 16 + col % 8 * 2;
    }
    for (int tile = k0; tile < k1; tile++) {
        const bool ragged = tile * BN + BN - 1 > first || tile * BN < last - W + 1;        // some row does not attend it whole
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        bool bad = false;
        #pragma unroll
        for (int i = 0; i < NC; i++) {
            const int id = threadIdx.x + 64 * NW * i, r = id / C8, ch = id % C8;
            const v4f *at = (const v4f *)raw + r * 2 * C8 + ch;
            const v4f x0 = at[0], x1 = at[C8];
            v4f y0 = at[RAW / 16], y1 = at[RAW / 16 + C8];
            float kb = abs_max(x0, x1), vb = abs_max(y0, y1);
            if (ragged || __any(!(vb < INFINITY))) {                         // a row of V has the factor of its finite values
                vb = 0.0f;
                #pragma unroll
                for (int k = 0; k < 4; k++) {
                    const bool f0 = finite32(y0[k]), f1 = finite32(y1[k]);
                    vb = fmaxf(vb, fmaxf(f0 ? fabsf(y0[k]) : 0.0f, f1 ? fabsf(y1[k]) : 0.0f));
                    if (ragged) {
                        bad |= !f0 | !f1;
                        y0[k] = f0 ? y0[k] : 0.0f; y1[k] = f1 ? y1[k] : 0.0f;
                    }
                }
            }
            const uint32_t ke = row_exp(lanes_max<C8>(kb)), ve = row_exp(lanes_max<C8>(vb));
            const float ku = row_up(ke), vu = row_up(ve);
            if (ch == 0) { s_kf[r] = row_down(ke); s_vf[r] = __uint_as_float((ve - 15) << 23); }       // (2^(ve - 142), half of what V was divided by)
            // (an infinity in K becomes h = inf, l = NaN)
            const Halves K = halves_of([&](int k) { return (k < 4 ? x0[k & 3] : x1[k & 3]) * ku; });
            const Halves V = halves_of([&](int k) { return (k < 4 ? y0[k & 3] : y1[k & 3]) * vu; });
            h8 *kd = (h8 *)lds + r * C8 + (ch ^ k_swz(r)), *vd = (h8 *)(lds + 2 * PIECE) + r * C8 + (ch ^ v_swz(r));
            kd[0] = K.h; kd[PIECE / 16] = K.l;
            vd[0] = V.h; vd[PIECE / 16] = V.l;
        }
        bool odd = false;
        if (ragged) odd = __syncthreads_or(bad); else __syncthreads();
        if (tile + 1 < k1) {
            if (SPLIT == 1) load(kp, a.k_stride, ko, tile + 1, 0);
            load(vp, a.v_stride, vo, tile + 1, RAW);
        }
        const int key0 = tile * BN + part * 32;                            // this wave's keys
        const bool idle = key0 > w_last || key0 + 32 <= w_first - W + 1;   // none that a row of it attends
        // fragments are read NF products ahead, the first of V beside the last of K
        constexpr int NF = SPLIT == 2 && NW == 4 ? 6 : 4, NVF = 2 * DT;
        constexpr bool AHEAD = SPLIT == 1 || NW == 4;                      // (two waves a SIMD, each with sums of 128 dims, have no registers for V's first)
        Halves F[NF];
        auto read_k = [&](int x) { return Halves{*(const h8 *)(lds + k_at[x]), *(const h8 *)(lds + k_at[x] + PIECE)}; };
        auto read_v = [&](int x) {
            h8 V[2];
            #pragma unroll
            for (int z = 0; z < 2; z++) {
                const uint8_t *at = lds + v_at[x % DT] + (2 + z) * PIECE + 16 * (x / DT) * HD * 2;
                const v4s p = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)at), q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4s *)(at + 8 * HD * 2));
                V[z] = __builtin_bit_cast(h8, __builtin_shufflevector(p, q, 0, 1, 2, 3, 4, 5, 6, 7));
            }
            return Halves{V[0], V[1]};
        };
        v16f S = zero;
        if (!idle) {
            #pragma unroll
            for (int x = 0; x < NF; x++) F[x] = read_k(x);
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NF, 0);
            #pragma unroll
            for (int x = 0; x < NS; x++) {
                S = mfma_halves(F[x % NF], Q[x], S);
                if (x + NF < NS) F[x % NF] = read_k(x + NF); else if (AHEAD) F[x % NF] = read_v(x + NF - NS);
                __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
                if (x + NF < NS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); else if (AHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            }
        }
        if constexpr (SPLIT == 2) {
            float *x = (float *)raw + wave * 1024 + lane * 4;
            #pragma unroll
            for (int i = 0; i < 16; i += 4) *(v4f *)(x + i * 64) = (v4f){S[i], S[i + 1], S[i + 2], S[i + 3]};
            __syncthreads();
            const float *y = (const float *)raw + (wave ^ RG * KS) * 1024 + lane * 4;
            #pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const v4f z = *(const v4f *)(y + i * 64);
                #pragma unroll
                for (int k = 0; k < 4; k++) S[i + k] += z[k];
            }
            __syncthreads();
            if (tile + 1 < k1) load(kp, a.k_stride, ko, tile + 1, 0);
        }
        if (idle) continue;
        // this lane's keys: 8 (i / 4) + 4 half + i % 4
        #pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const v4f x = *(const v4f *)(s_kf + part * 32 + 2 * i + 4 * half);
            #pragma unroll
            for (int k = 0; k < 4; k++) S[i + k] *= x[k];
        }
        if (key0 + 31 > w_first || key0 < w_last - W + 1) {
            asm volatile("");                                              // a branch: whole tiles do without this
            #pragma unroll
            for (int i = 0; i < 16; i++) {
                const int key = key0 + 8 * (i / 4) + 4 * half + i % 4;
                S[i] = key <= tok && key > tok - W ? S[i] : -INFINITY;
            }
        }
        float mx = S[0];
        #pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, S[i]);
        float al = 1.0f, mt = 0.0f;
        const bool moved = __any(moves(mx, m, slack));
        if (__builtin_expect(moved, 0)) {
            mx = fmaxf(mx, other_half(mx));
            const float mn = fmaxf(m, mx);
            al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            l *= al;
        }
        const float nm = m == -INFINITY ? 0.0f : -m * c;
        #pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const v4f x = *(const v4f *)(s_vf + part * 32 + 2 * i + 4 * half);
            #pragma unroll
            for (int k = 0; k < 4; k++) {
                const float w = __builtin_amdgcn_exp2f(fmaf(S[i + k], c, nm));
                l += w;
                S[i + k] = w * x[k];
                mt = fmaxf(mt, S[i + k]);
            }
        }
        if (__builtin_expect(moved || __any(ldexpf(mt, ge) > 32768.0f), 0)) {
            tm = fmaxf(tm * al, mt);
            tm = fmaxf(tm, other_half(tm));
            const int to = 134 - min(max((int)(__float_as_uint(tm) >> 23), 8), 254);
            const float f = ldexpf(al, to - ge);
            ge = to;
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int i = 0; i < 16; i++) O[d][i] *= f;
        }
        #pragma unroll
        for (int i = 0; i < 16; i++) S[i] = ldexpf(S[i], ge);
        Halves P[2];
        #pragma unroll
        for (int e = 0; e < 2; e++) P[e] = halves_of([&](int k) { return S[8 * e + k]; });
        if (!AHEAD) {
            #pragma unroll
            for (int x = 0; x < NF; x++) F[(NS + x) % NF] = read_v(x);
        }
        #pragma unroll
        for (int x = 0; x < NVF; x++) {
            O[x % DT] = mfma_halves(F[(NS + x) % NF], P[x / DT], O[x % DT]);
            if (x + NF < NVF) F[(NS + x) % NF] = read_v(x + NF);
            __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
            if (x + NF < NVF) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        }
        if (odd) {                                                          // V values that were left out, for the rows that attend them
            #pragma unroll 1
            for (int key = key0; key < min(key0 + 32, n); key++) {
                const float *vrow = vp + (size_t)key * a.v_stride + dim0 + 4 * half;
                #pragma unroll
                for (int d = 0; d < DT; d++)
                    #pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float x[4];
                        load_values(vrow + d * 32 + 2 * i, x);
                        #pragma unroll
                        for (int y = 0; y < 4; y++) O[d][i + y] += key <= tok && key > tok - W && !finite32(x[y]) ? x[y] * INFINITY : 0.0f;
                    }
            }
        }
    }
    l += other_half(l);
    const int r = wr0 + l32;
    float *o = (float *)a.out + (size_t)(t0 + r / G) * a.out_stride + (size_t)(h * G + r % G) * HD + dim0 + 4 * half;
    if constexpr (KS == 1) {
        const float inv = 1.0f / l;
        if (r >= R) return;
        #pragma unroll
        for (int d = 0; d < DT; d++)
            #pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float x[4];
                #pragma unroll
                for (int y = 0; y < 4; y++) x[y] = ldexpf(O[d][i + y] * inv, 1 - ge);
                store_values(o + d * 32 + 2 * i, x);
            }
    } else {
        #pragma unroll
        for (int d = 0; d < DT; d++)
            #pragma unroll
            for (int i = 0; i < 16; i++) O[d][i] = ldexpf(O[d][i], 1 - ge);                 // each part has its own
        static_assert(join_bytes(RG, KS, DT) <= 2 * RAW + 4 * PIECE, "the parts' outputs");
        join_parts<RG, KS, DT>(O, m, l, c, raw, s_ml, wave, lane, [&](int d, int i, const float (&x)[4]) {
            if (r < R) store_values(o + d * 32 + 2 * i, x);
        });
    }
}

// Units of `rows` rows that a call's rows may fall into, each a workgroup for every kv head
int64_t prompt_slots(const sp_hipkv_prompt_args &a, int rows) { return (int64_t)a.n_tokens * (a.n_heads / a.n_kv_heads) / rows + a.n_seqs; }

// sizes; the pointers are not looked at
int prompt_check(const char *who, const sp_hipkv_prompt_args *a) {
    if (serve_check(who, a)) return 1;
    OP_NEED(a->window >= 0, "negative window");
    OP_NEED(std::isfinite(a->scale), "scale is not finite");
    OP_NEED(!a->n_tokens || prompt_slots(*a, 64) * a->n_kv_heads < 1 << 23, "too many sequences, heads and tokens for one launch");      // (of 512 threads, 2^32 in all)
    return 0;
}
int prompt_check_arrays(const char *who, const sp_hipkv_prompt_args *a) {
    OP_NEED(a->start, "null array");
    return serve_rows(who, a, a->q, a->q_stride, a->n_heads) || serve_rows(who, a, a->k, a->k_stride, a->n_kv_heads) ||
           serve_rows(who, a, a->v, a->v_stride, a->n_kv_heads) || serve_rows(who, a, a->out, a->out_stride, a->n_heads);
}

// The form that a call takes: row groups of 32, parts of a tile's keys, tiles of 32 keys a part (f32: 1)
struct PromptForm { int rg, ks, kt; };
template <typename T, int HD> PromptForm prompt_form(const sp_hipkv_prompt_args &a) {
    // A window well below the longest prompt: all spans are much the same, and what counts is how often the
    // units are filled.  Waves that share keys, one workgroup of eight a unit, then pay in one round only, and for
    // spans that are worth sharing; `span` is the longest.
    const bool even = a.window && 3 * (int64_t)a.window < 2 * (int64_t)a.max_tokens;
    const int span = even ? a.window : a.max_tokens;
    if constexpr (sizeof(T) == 4) {
        // Up to some workgroups a unit it is the way along the keys that takes the time, and a workgroup of eight
        // waves walks 64 keys (dims of 64: 128) in the time that four take for 32.  One sequence of n tokens,
        // 16 and 8 heads of 128: 18.1 us for 18.9 at n = 130, 65 for 88 at 1000, 118 for 163 at 2000; 32 and 8
        // heads: 151 for 176 at 2000 (504 workgroups), 772 for 726 at 5000.  Dims of 64: 32 and 8 heads 11.9 for 11.9 at 130, 42 for 52 at 1000 (504), 123 for 99 at 2000.  Six of 50 to 400 tokens: 33 for 39.5
        // (216), 46.6 for 45.9 (384).  In windows of 64, 128, 256 of 500 tokens of 16 and 8 heads 19.0, 22.4, 29.5 for 20.6, 25.8, 36.1 (64),
        // of 1500 of 32 and 8 38.8, 46.3, 59.3 for 27.8, 34.6, 47.2 (376), dims of 64, of 500 13.5, 14.0, 17.1 for 11.3, 14.2, 20.0 (256), of
        // 1000 25.3, 26.4, 31.9 for 12.1, 15.2, 20.9 (504).
        if constexpr (HD < 256) {
            constexpr int KS = HD == 128 ? 2 : 4, RG = 8 / KS;
            const int64_t units = prompt_slots(a, 32 * RG) * a.n_kv_heads;
            if (a.max_tokens >= 128 && span >= 32 * KS && units <= (even ? 256 : 512)) return {RG, KS, 1};
        }
        // Dims of 256: a unit holds one workgroup, and with no more than one for each the longest span is what counts,
        // which 64 rows walk faster than 128 (one wave a SIMD has registers for more fragments ahead): 16 and 8 heads
        // 121 us for 146 at 1000 tokens, 260 for 283 at 2047 (256 units of 128 rows), 455 for 365 at 2600.  Of even spans
        // it is the sum that counts from half as many on: a window of 1024 of 1400 tokens 130 for 160, of 1788 204 for 163.
        if constexpr (HD == 256) {
            if ((int64_t)a.n_tokens * a.n_heads / 128 <= (even ? 128 : 256)) return {2, 1, 1};
        }
        return {4, 1, 1};
    }
    else if constexpr (HD == 256) return {2, 1, 1};
    else {
        // A unit holds two workgroups of four waves: with fewer rows than half of them take, the keys of 64 rows
        // are shared by four waves each, a workgroup of eight a unit.  One sequence of 16 and 8 heads of 128: 13.0
        // us for 15.3 at 500 tokens, 21.7 for 27.4 at 1200; 32 and 8 heads: 13.5 for 15.8 at 500, 22.8, too many,
        // for 21.9 at 800; 130 tokens, too few keys: 9.2 for 8.6.  Windows of 128, 256 of 500 tokens of 32 and 8 heads 12.1, 13.4 for
        // 11.7, 13.9 (256 workgroups); 256, 512 of 1200 of 16 and 8 21.6, 21.0 for 14.1, 18.6 (304).
        if (span >= 192 && prompt_slots(a, 64) * a.n_kv_heads <= (even ? 256 : 304)) return {2, 4, 1};
        // With fewer than all take, the keys of 128 rows by two: 16 and 8 heads 50.5 for 58.1 at 2800 tokens, 60.0 for 68.4 at
        // 3300, 103 for 100.9 at 4500; 32 and 8 26.1 for 29.2 at 1200, 48.6 for 48.0 at 2000.  Short sequences' last tiles
        // cost more (six of 50 to 400 tokens 13.7 for 13.2), and dims of 64 gain nothing (19.8 for 19.7 at 1200).
        // Windows of 256, 512, 1024 of 2000 tokens of 16 and 8 heads 15.8, 19.3, 26.3 for 14.9, 19.5, 27.6 (256 workgroups), of 2800
        // 28.0, 34.9, 42.1 for 19.6, 26.0, 31.0 (352).
        if constexpr (HD == 128)
            if (a.n_tokens >= (int64_t)800 * a.n_seqs && span >= 512 && prompt_slots(a, 128) * a.n_kv_heads <= (even ? 256 : 432)) return {4, 2, 1};
        // Two rounds of workgroups of 256 rows, or many: K and V are fetched half as often.  32 and 8 heads 143 us for 151
        // at 4000 tokens (504 of them), 505 for 520 at 8192 (1032), but 256 for 253 at 5500 (696); 16 and 8 257 for
        // 281 at 8192 (520), 148 for 137 at 5500 (352).  Not of even spans: a window of 1024 78.6 for 76.7 at 4000, 159.7 for 153.4 at 8192.
        if constexpr (HD == 128) {
            const int64_t units = prompt_slots(a, 256) * a.n_kv_heads;
            if (!even && a.n_tokens >= (int64_t)2000 * a.n_seqs && units >= 432 && (units <= 528 || units >= 864)) return {8, 1, 2};
        }
        return {4, 1, 2};
    }
}
template <typename T, int HD> hipError_t prompt_go(const sp_hipkv_prompt_args &a, hipStream_t s) {
    const PromptForm f = prompt_form<T, HD>(a);
    const int64_t slots = prompt_slots(a, 32 * f.rg);
    const dim3 grid((uint32_t)(slots * a.n_kv_heads)), wg(64 * f.rg * f.ks * prompt_split(HD));
    auto run = [&](auto k) { return op_launch(k, grid, wg, s, a, (int)slots); };
    if constexpr (sizeof(T) == 4) {
        if constexpr (HD == 256) return f.rg == 2 ? run(k_prompt32<HD, 2, 1>) : run(k_prompt32<HD, 4, 1>);
        else return f.ks > 1 ? run(k_prompt32<HD, HD == 128 ? 4 : 2, HD == 128 ? 2 : 4>) : run(k_prompt32<HD, 4, 1>);
    }
    else if constexpr (HD == 256) return run(k_prompt16<HD, 2, 1, 1>);
    else {
        if (f.ks == 4) return run(k_prompt16<HD, 2, 4, 1>);
        if constexpr (HD == 128) {
            if (f.ks == 2) return run(k_prompt16<HD, 4, 2, 1>);
            if (f.rg == 8) return run(k_prompt16<HD, 8, 1, 2>);
        }
        return run(k_prompt16<HD, 4, 1, 2>);
    }
}
// f(value type, std::integral_constant of the head dim) for the call's
template <typename F> auto prompt_pick(const sp_hipkv_prompt_args &a, F &&f) {
    auto dim = [&](auto t) {
        return a.head_dim == 256 ? f(t, std::integral_constant<int, 256>{}) : a.head_dim == 128 ? f(t, std::integral_constant<int, 128>{}) : f(t, std::integral_constant<int, 64>{});
    };
    return a.type == SP_HIPKV_F32 ? dim(float{}) : dim(Bf16{});
}

}  // namespace

hipError_t launch_prompt(const sp_hipkv_prompt_args &a, hipStream_t s) {
    return prompt_pick(a, [&](auto t, auto hd) { return prompt_go<decltype(t), hd.value>(a, s); });
}

}  // namespace kvd

extern "C" int sp_hipkv_prompt_attention_plan(const sp_hipkv_prompt_args *a, int32_t plan[4]) {
    using namespace kvd;
    const char *who = "sp_hipkv_prompt_attention_plan";
    if (prompt_check(who, a)) return 1;
    OP_NEED(plan, "null plan");
    prompt_pick(*a, [&](auto t, auto hd) {
        const PromptForm f = prompt_form<decltype(t), hd.value>(*a);
        plan[0] = 32 * f.rg; plan[1] = 32 * f.ks * f.kt; plan[2] = f.ks; plan[3] = f.rg * f.ks * prompt_split(hd.value);
        return 0;
    });
    return 0;
}

extern "C" int sp_hipkv_prompt_attention(const sp_hipkv_prompt_args *a, void *stream) {
    using namespace kvd;
    const char *who = "sp_hipkv_prompt_attention";
    if (prompt_check(who, a)) return 1;
    if (!a->n_tokens) return 0;
    if (prompt_check_arrays(who, a)) return 1;
    OpDevice dev((hipStream_t)stream);
    return op_done(who, dev.err != hipSuccess ? dev.err : launch_prompt(*a, (hipStream_t)stream));
}
