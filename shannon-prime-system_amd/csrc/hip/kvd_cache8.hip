// kvd_cache8.hip -- attention of new tokens over the 8-bit paged cache.
//
// The q heads of a kv head share its K and V: the rows of one kv head are r = token G + q
// head of the group, 16 of them, a matrix tile, to a workgroup.  Its waves take the pages of a
// range (a split) in turn, each with a running maximum, sum and output of its own; they meet
// in LDS at the end, the splits in k_cache_merge.
//
// Codes go to the int8 matrix cores as they lie in memory.  q is taken to integers of 23 bits and
// a sign (127 2^16 for the row's largest value) and these to three digits to base 256, from -128
// on, so a score is three exact integer products; so are then the weights of a page, each times
// its V block's scale (127 2^16 for the row's largest).  (bf16 values: 15 bits, two digits.)  With 22 bits above a power of two outputs
// were off by 1.4e-6 where f32 products are by 0.7e-6.  Digits joined: d2 2^16 + (d1 2^8 + d0), the bracket in int32 (256 dims of
// 2^14 fit), the rest in f32.
//
// Scores are made transposed (K the A operand): lane (g, l) then has row l and the
// positions 16 u + 4 g + i of a page, u, i < 4, which as k slots 16 g + 4 u + i are its share of the
// second product's A operand.  V's bytes lie in that order in a column (include/sp_hipkv.h), so
// nothing is transposed or moved between lanes, and a wave's loads are whole columns.
#include "kvd_serve.h"
#include "kvd_pass.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

constexpr float LOG2E_F = 1.44269504088896341f;
constexpr int CACHE_PAGES = 256, CACHE_WAVES = 4;                       // pages of a split at most; waves of a workgroup
// Digits of q and the weights: three, and for bf16 values, which are off by 2^-9 themselves, two (15
// bits: a third fewer products, three instructions for five to join them; a q value below 2^-7 of its row's
// largest so loses bits that it has, 2^-16 of the largest); the largest magnitude that they hold, with room for carries.
template <typename T> constexpr int DIG = sizeof(T) == 4 ? 3 : 2;
template <typename T> constexpr float DIGITS = sizeof(T) == 4 ? 127 * 65536 : 127 * 256;
// the number that products with digits 0, 1, .. make up
__device__ __forceinline__ float joined(int a, int b) { return (float)(b * 256 + a); }
__device__ __forceinline__ float joined(int a, int b, int c) { return fmaf((float)c, 65536.0f, (float)(b * 256 + a)); }

// the bytes b of four words, b = 0 .. ND - 1: p[b]
template <int ND> __device__ __forceinline__ void byte_planes(const uint32_t (&t)[4], uint32_t (&p)[ND]) {
    const uint32_t a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400), b = __builtin_amdgcn_perm(t[3], t[2], 0x05010400);
    p[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
    p[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    if constexpr (ND == 3) p[2] = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0602) | __builtin_amdgcn_perm(t[3], t[2], 0x06020C0C);
}

__device__ __forceinline__ const uint8_t *uniform(const uint8_t *x) {
    const uint64_t p = (uint64_t)x;
    return (const uint8_t *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)p));
}

// the largest of lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float rows_max(float x) {
    const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <typename T, int HD>
__global__ __launch_bounds__(64 * CACHE_WAVES, HD == 256 ? 1 : 2) void k_cache(sp_hipkv_cache_args a, int groups, int nsplit, int pages) {
    static_assert(HD / 64 <= CACHE_WAVES, "a wave for every 64 dims of q");
    constexpr int ND = DIG<T>, KS = HD / 64, CT = HD / 16, NW = CACHE_WAVES, NT = 64 * NW, UB = HD == 256 ? 2 : 4;
    __shared__ v4i s_q[KS * ND][64];
    __shared__ uint32_t s_big[KS][16];
    __shared__ __align__(16) float s_o[NW][16][HD];
    __shared__ float s_m[NW][16], s_l[NW][16], s_M[16], s_L[16];
    __shared__ const uint8_t *s_page[CACHE_PAGES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads;
    int id = blockIdx.x;
    const int h = id % a.n_kv_heads; id /= a.n_kv_heads;
    const int grp = id % groups; id /= groups;
    const int split = id % nsplit, s = id / nsplit;
    const void *const *table = gmem(a.tables)[s];                          // (here: one wait for all of a sequence's numbers)
    const int t0 = max(gmem(a.start)[s], 0), cached = min(max(gmem(a.cached)[s], 0), a.max_positions);
    const int n = min(min(gmem(a.start)[s + 1], a.n_tokens) - t0, min(a.max_tokens, a.max_positions - cached)), end = cached + n;
    const int R = n * G, r0 = grp * 16;
    if (r0 >= R) return;
    // the positions that this workgroup's rows see: first row's window start to the last row's own
    const int W = a.window ? a.window : INT32_MAX;
    const int at0 = cached + r0 / G, at1 = cached + (min(r0 + 16, R) - 1) / G, lo = max(at0 - W + 1, 0);
    // this split's pages (of a sequence shorter than the longest there are proportionally fewer)
    const int pg0 = lo / PAGE;
    const uint32_t np = at1 / PAGE + 1 - pg0;
    const uint32_t parts = max((np * nsplit + pages - 1) / pages, (np + CACHE_PAGES - 1) / CACHE_PAGES);          // (2^14 x 64 at most)
    const int b0 = pg0 + np * min((uint32_t)split, parts) / parts, b1 = pg0 + np * min((uint32_t)split + 1, parts) / parts;
    float *po = (float *)a.work, *pml = po + (size_t)a.n_tokens * a.n_heads * nsplit * HD;
    auto row_of = [&](int r) { return (size_t)(t0 + r / G) * a.n_heads + h * G + r % G; };
    if (nsplit > 1 && b0 >= b1) {
        const int r = r0 + threadIdx.x;
        if (threadIdx.x < 16 && r < R) *gmem((v2f *)(pml + 2 * (row_of(r) * nsplit + split))) = (v2f){-INFINITY, 0.0f};
        return;
    }
    const size_t kat = (size_t)h * PAGE * HD, vat = (size_t)(a.n_kv_heads + h) * PAGE * HD, sat = (size_t)a.n_kv_heads * 2 * PAGE * HD + 16 * h;
    v4i K[4][KS], V[CT];
    v4f ks, vs;
    auto load_k = [&](const uint8_t *pg) {
        #pragma unroll
        for (int u = 0; u < 4; u++)
            #pragma unroll
            for (int e = 0; e < KS; e++) K[u][e] = *gmem((const v4i *)(pg + kat + (16 * u + l16) * HD + 64 * e + 16 * g));
        ks = *gmem((const v4f *)(pg + sat));
    };
    auto load_v = [&](const uint8_t *pg) {
        #pragma unroll
        for (int c = 0; c < CT; c++) V[c] = *gmem((const v4i *)(pg + vat + (16 * c + l16) * PAGE + 16 * g));
        vs = *gmem((const v4f *)(pg + sat + 16 * a.n_kv_heads));
    };
    auto page_at = [&](int lp) { return (const uint8_t *)gmem(table)[a.ring_pages ? lp % a.ring_pages : lp]; };
    for (int i = threadIdx.x; i < b1 - b0; i += NT) s_page[i] = page_at(b0 + i);
    // q's digits, [64 dims][digit][lane] 16 bytes: lane (g, l) has row l, dims 64 e + 16 g ..
    const bool any_page = b0 + wave < b1;
    float x[2][8];
    if (wave < KS) {
        const int r = min(r0 + l16, R - 1);
        const T *q = (const T *)a.q + (size_t)(t0 + r / G) * a.q_stride + (size_t)(h * G + r % G) * HD + 64 * wave + 16 * g;
        load_values(q, x[0]);
        load_values(q + 8, x[1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (any_page) {                                                        // on their way while q is taken apart
        const uint8_t *pg = uniform(page_at(b0 + wave));
        load_k(pg);
        load_v(pg);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (wave < KS) {
        uint32_t big = 0;                                                  // as bits: NaN is above infinity
        #pragma unroll
        for (int k = 0; k < 16; k++) big = max(big, __float_as_uint(x[k / 8][k % 8]) & 0x7FFFFFFFu);
        big = max(big, (uint32_t)__shfl_xor((int)big, 16, 64));
        big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
        if (lane < 16) s_big[wave][l16] = big;
    }
    __syncthreads();
    uint32_t big = 0;
    #pragma unroll
    for (int e = 0; e < KS; e++) big = max(big, s_big[e][l16]);
    const float up = fminf(DIGITS<T> / __uint_as_float(big), 3e38f);       // (of zeros and the smallest denormals the largest)
    const float qs = big < 0x7F800000u ? a.scale * LOG2E_F / up : NAN;
    const int at = cached + min(r0 + l16, R - 1) / G;
    if (wave < KS) {
        v4i q[ND];
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t w[4], p[ND];
            #pragma unroll
            for (int j = 0; j < 4; j++) w[j] = (uint32_t)(int)rintf(x[k / 2][4 * (k % 2) + j] * up) + (ND == 3 ? 0x808080u : 0x8080u);
            byte_planes(w, p);
            #pragma unroll
            for (int d = 0; d < ND; d++) q[d][k] = (int)(p[d] ^ 0x80808080u);
        }
        #pragma unroll
        for (int d = 0; d < ND; d++) s_q[wave * ND + d][lane] = q[d];
    }
    v4f O[CT];
    float m = -INFINITY, l = 0.0f;
    #pragma unroll
    for (int c = 0; c < CT; c++) O[c] = (v4f){0, 0, 0, 0};
    __syncthreads();
    for (int b = b0 + wave; b < b1; b += NW) {
        const bool more = b + NW < b1;
        const uint8_t *pn = uniform(s_page[(more ? b + NW : b) - b0]);
        // some row of the workgroup does not see the page whole
        const bool ragged = b * PAGE + PAGE - 1 > at0 || b * PAGE < at1 - W + 1;
        float S[4][4];
        #pragma unroll
        for (int u0 = 0; u0 < 4; u0 += UB) {
            asm volatile("" : : : "memory");                           // q's digits are read again: 12 registers for each 64 dims
            v4i acc[UB][ND] = {};
            #pragma unroll
            for (int e = 0; e < KS; e++) {
                v4i q[ND];
                #pragma unroll
                for (int d = 0; d < ND; d++) q[d] = s_q[e * ND + d][lane];
                #pragma unroll
                for (int u = 0; u < UB; u++)
                    #pragma unroll
                    for (int d = 0; d < ND; d++) acc[u][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(K[u0 + u][e], q[d], acc[u][d], 0, 0, 0);
            }
            #pragma unroll
            for (int u = 0; u < UB; u++) {
                const float f = qs * fmaf(ks[u0 + u], 0.0f, ks[u0 + u]);       // NaN of an infinite scale
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (ND == 3) S[u0 + u][i] = f * joined(acc[u][0][i], acc[u][1][i], acc[u][2][i]);
                    else S[u0 + u][i] = f * joined(acc[u][0][i], acc[u][1][i]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_k(pn);
        __builtin_amdgcn_sched_barrier(0);
        v4i Pd[ND];
        uint32_t seen = 0xFFFF;
        if (ragged) {
            seen = 0;
            #pragma unroll
            for (int k = 0; k < 16; k++) {
                const int p = b * PAGE + 16 * (k / 4) + 4 * g + k % 4;
                const bool on = p <= at && p > at - W;
                seen |= (uint32_t)on << k;
                S[k / 4][k % 4] = on ? S[k / 4][k % 4] : -INFINITY;
            }
        }
        float mx = -INFINITY;
        #pragma unroll
        for (int k = 0; k < 16; k++) mx = fmaxf(mx, S[k / 4][k % 4]);
        if (__any(mx > m + 16.0f)) {
            mx = rows_max(mx);
            const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
            #pragma unroll
            for (int i = 0; i < 4; i++) {                              // O's rows are 4 g + i
                const float f = __shfl(al, 4 * g + i, 64);
                #pragma unroll
                for (int c = 0; c < CT; c++) O[c][i] *= f;
            }
        }
        const float ms = m == -INFINITY ? 0.0f : m;
        float top = 0.0f;                                                 // (weights up to 2^16, V of 2^90, 2^20 positions: sums below 2^126)
        #pragma unroll
        for (int u = 0; u < 4; u++) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const float w = __builtin_amdgcn_exp2f(S[u][i] - ms);
                l += w;
                S[u][i] = w * vs[u];
            }
            if ((__float_as_uint(vs[u]) & 0x7F800000u) == 0x7F800000u) {  // uniform: a scale that is not finite
                if (seen >> 4 * u & 15) l = NAN;
                #pragma unroll
                for (int i = 0; i < 4; i++) S[u][i] = 0.0f;
            }
            #pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, S[u][i]);
        }
        top = rows_max(top);
        // weights to integers up to DIGITS; 2^23 + x has x in its low bits, half a digit more in each but the last byte makes digits of them
        top = fmaxf(top, 1e-30f);
        const float up = DIGITS<T> / top;
        const float back = top * (1.0f / DIGITS<T>);
        #pragma unroll
        for (int u = 0; u < 4; u++) {
            uint32_t w[4], p[ND];
            #pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __float_as_uint(fmaf(S[u][i], up, 8388608.0f)) + (ND == 3 ? 0x8080u : 0x80u);
            byte_planes(w, p);
            #pragma unroll
            for (int d = 0; d < ND; d++) Pd[d][u] = (int)(d < ND - 1 ? p[d] ^ 0x80808080u : p[d]);
        }
        float f[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __shfl(back, 4 * g + i, 64);
        #pragma unroll
        for (int c = 0; c < CT; c++) {
            v4i acc[ND];
            #pragma unroll
            for (int d = 0; d < ND; d++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(Pd[d], V[c], (v4i){0, 0, 0, 0}, 0, 0, 0);
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (ND == 3) O[c][i] = fmaf(f[i], joined(acc[0][i], acc[1][i], acc[2][i]), O[c][i]);
                else O[c][i] = fmaf(f[i], joined(acc[0][i], acc[1][i]), O[c][i]);
            }
            if (c % 2) asm volatile("" : "+v"(O[c - 1]), "+v"(O[c]));       // here, not behind all columns' products: their registers
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v(pn);
        __builtin_amdgcn_sched_barrier(0);
    }
    // join the waves
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < 16) { s_m[wave][l16] = m; s_l[wave][l16] = l; }
    #pragma unroll
    for (int c = 0; c < CT; c++)
        #pragma unroll
        for (int i = 0; i < 4; i++) s_o[wave][4 * g + i][16 * c + l16] = O[c][i];
    __syncthreads();
    if (threadIdx.x < 16) {
        float M = s_m[0][l16], L = 0.0f;
        #pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, s_m[w][l16]);
        const float Ms = M == -INFINITY ? 0.0f : M;
        #pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][l16] - Ms);
            L += s_l[w][l16] != 0.0f ? f * s_l[w][l16] : 0.0f;          // NaN sums stay, empty ones add nothing
            s_m[w][l16] = f;
        }
        s_M[l16] = M; s_L[l16] = L;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * HD / 4; i += NT) {
        const int k = i / (HD / 4), c = i % (HD / 4) * 4, r = r0 + k;
        if (r >= R) continue;
        v4f x = {0, 0, 0, 0};
        #pragma unroll
        for (int w = 0; w < NW; w++) x += *(const v4f *)&s_o[w][k][c] * s_m[w][k];
        const float L = s_L[k];
        if (nsplit == 1) {
            const float inv = 1.0f / L;                                    // (0: no score is above -inf; 0 x inf is NaN)
            float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
            store_values((T *)a.out + (size_t)(t0 + r / G) * a.out_stride + (size_t)(h * G + r % G) * HD + c, y);
        } else {
            const size_t at = row_of(r) * nsplit + split;
            *gmem((v4f *)(po + at * HD + c)) = x;
            if (c == 0) *gmem((v2f *)(pml + 2 * at)) = (v2f){s_M[k], L};
        }
    }
}

// Joins a row's parts: a workgroup a row, a thread four columns of every NG-th part.
template <typename T, int HD, int NT>
__global__ __launch_bounds__(NT) void k_cache_merge(sp_hipkv_cache_args a, int nsplit) {
    constexpr int NG = 4 * NT / HD;
    __shared__ float s_f[64], s_L;
    __shared__ v4f s_x[NT];
    const size_t row = blockIdx.x;
    const int c = threadIdx.x % (HD / 4), grp = threadIdx.x / (HD / 4), token = (int)(row / a.n_heads);
    if (token < gmem(a.start)[0] || token >= gmem(a.start)[a.n_seqs]) return;               // of no sequence: left as it was
    const float *ml = (const float *)a.work + (size_t)a.n_tokens * a.n_heads * nsplit * HD + 2 * row * nsplit;
    if (threadIdx.x < 64) {
        const bool in = (int)threadIdx.x < nsplit;
        const float m = in ? ml[2 * threadIdx.x] : -INFINITY, l = in ? ml[2 * threadIdx.x + 1] : 0.0f, M = wave_allmax(m);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
        s_f[threadIdx.x] = l == 0.0f ? -1.0f : f;                          // a part without a position of this row is not read
        const float L = wave_allsum(l == 0.0f ? 0.0f : f * l);
        if (threadIdx.x == 0) s_L = L;
    }
    __syncthreads();
    const v4f *po = (const v4f *)((const float *)a.work + row * nsplit * HD) + c;
    v4f x = {0, 0, 0, 0};
    #pragma unroll 4
    for (int k = grp; k < nsplit; k += NG) {
        const float f = s_f[k];
        if (f >= 0.0f) x += po[(size_t)k * (HD / 4)] * f;
    }
    s_x[threadIdx.x] = x;
    __syncthreads();
    if (grp) return;
    #pragma unroll
    for (int k = 1; k < NG; k++) x += s_x[k * (HD / 4) + c];
    const float inv = 1.0f / s_L;
    float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    store_values((T *)a.out + (size_t)token * a.out_stride + (row % a.n_heads) * HD + 4 * c, y);
}

// How a launch is cut: workgroups along a sequence's rows (groups, of 16 rows), parts of its pages
// (nsplit), for the least time estimated of
//   a workgroup's fixed 5, 7.5, 8 us (dims of 64, 128, 256) and 1.2, 1.8, 2.7 a page and wave, a quarter
//   more for each that shares its unit (3, 2, 1 can), as often as the units are filled;
//   memory at 4.8 TB/s (several sequences are taken to be 0.6 of the longest), and a quarter of
//   the lesser of the two on top;
//   3.5 us to join parts.
// From sweeps of nsplit: one token of 16 heads at 32703 (dims of 256) takes 32.1, 31.5, 39.5 us with
// 24, 32, 48 parts; 30 sessions at 914 (32 heads of 128) 15.7, 18.4, 23.3 with 1, 2, 4; 24 tokens at 12000
// 27.9, 28.2, 32.9 with 4, 8, 12.  Against filling 1024 workgroups: 4 x 48 tokens with a window of 1024
// 23 us for 45.
struct CachePlan { int groups, nsplit, pages; };
CachePlan cache_plan(const sp_hipkv_cache_args &a) {
    CachePlan p{};
    p.groups = std::max(1, (int)(((int64_t)a.max_tokens * (a.n_heads / a.n_kv_heads) + 15) / 16));
    const int64_t span = a.window ? std::min<int64_t>(a.max_positions, (int64_t)a.window + 16 + PAGE) : a.max_positions;
    p.pages = (int)std::max<int64_t>(1, (span + PAGE - 1) / PAGE);
    const double fixed = a.head_dim == 256 ? 8 : a.head_dim == 128 ? 7.5 : 5, page = a.head_dim == 256 ? 2.7 : a.head_dim == 128 ? 1.8 : 1.2;
    const int units = a.head_dim == 256 ? 1 : a.head_dim == 128 ? 2 : 3;
    const double seqs = (double)a.n_kv_heads * std::max(a.n_seqs, 1);
    const double mem = fixed / 2 + (a.n_seqs > 1 ? 0.6 : 1.0) * seqs * p.pages * 2 * PAGE * a.head_dim / 4.8e6;
    double best = 0;
    for (int n = (p.pages + CACHE_PAGES - 1) / CACHE_PAGES; n <= 64 && n <= p.pages; n++) {
        const int each = (p.pages + n - 1) / n;
        const double wgs = std::ceil(seqs * p.groups * n / 256), at_once = std::min<double>(wgs, units);
        const double run = std::ceil(wgs / units) * (fixed + page * (0.75 + 0.25 * at_once) * ((each + CACHE_WAVES - 1) / CACHE_WAVES + 0.05 * each));
        const double us = std::max(run, mem) + 0.25 * std::min(run, mem) + (n > 1 ? 3.5 + 1.6e-6 * a.n_tokens * a.n_heads * n * a.head_dim : 0.0);
        if (!p.nsplit || us < best) { best = us; p.nsplit = n; }
    }
    return p;
}
int64_t cache_grid(const sp_hipkv_cache_args &a, const CachePlan &p) { return (int64_t)a.n_kv_heads * p.groups * p.nsplit * a.n_seqs; }

int cache_check(const char *who, const sp_hipkv_cache_args *a) {
    if (serve_check(who, a)) return 1;
    OP_NEED(a->max_tokens <= 512, "max_tokens above 512");
    OP_NEED(a->max_positions >= 0 && a->max_positions <= 1 << 20, "max_positions outside [0, 2^20]");
    OP_NEED((int64_t)a->n_tokens * a->n_heads <= 1 << 22, "more than 2^22 rows (n_tokens x n_heads)");
    OP_NEED(a->window >= 0 && a->ring_pages >= 0, "negative window or ring_pages");
    // positions from the first token's window to the last token, wherever in a page they begin
    OP_NEED(!a->ring_pages || a->max_positions <= (int64_t)a->ring_pages * PAGE ||
            (a->window && (int64_t)a->window + a->max_tokens - 1 + PAGE - 1 <= (int64_t)a->ring_pages * PAGE),
            "ring_pages hold less than window + max_tokens positions and a page more");
    return 0;
}
int cache_check_arrays(const char *who, const sp_hipkv_cache_args *a, size_t need) {
    OP_NEED(std::isfinite(a->scale), "scale is not finite");
    OP_NEED(a->start && a->cached && a->tables, "null array");
    OP_NEED(aligned(a->tables, 8), "misaligned array");
    if (serve_rows(who, a, a->q, a->q_stride, a->n_heads) || serve_rows(who, a, a->out, a->out_stride, a->n_heads)) return 1;
    OP_NEED(!need || (a->work && a->work_bytes >= need && aligned(a->work, 16)), "work is missing, too small or not 16-byte aligned");
    return 0;
}

template <typename T, int HD> hipError_t cache_go(const sp_hipkv_cache_args &a, hipStream_t s) {
    const CachePlan p = cache_plan(a);
    hipError_t e = op_launch(k_cache<T, HD>, dim3((uint32_t)cache_grid(a, p)), dim3(64 * CACHE_WAVES), s, a, p.groups, p.nsplit, p.pages);
    if (e != hipSuccess || p.nsplit == 1) return e;
    // (32 parts of 16 rows: 4.8 us with 1024 threads a row, 7.5 with 256; 2 parts of 2048 rows: 10.6, 4.8.  A
    // launch has fewer than 2^32 threads.)
    const dim3 rows((uint32_t)((int64_t)a.n_tokens * a.n_heads));
    if (p.nsplit > 8 && rows.x <= 1 << 20) return op_launch(k_cache_merge<T, HD, 1024>, rows, dim3(1024), s, a, p.nsplit);
    return op_launch(k_cache_merge<T, HD, 256>, rows, dim3(256), s, a, p.nsplit);
}
template <typename T> hipError_t cache_type(const sp_hipkv_cache_args &a, hipStream_t s) {
    return a.head_dim == 256 ? cache_go<T, 256>(a, s) : a.head_dim == 128 ? cache_go<T, 128>(a, s) : cache_go<T, 64>(a, s);
}

}  // namespace

hipError_t launch_cache(const sp_hipkv_cache_args &a, hipStream_t s) {
    return a.type == SP_HIPKV_F32 ? cache_type<float>(a, s) : cache_type<Bf16>(a, s);
}

}  // namespace kvd

extern "C" int sp_hipkv_cache_attention_work(const sp_hipkv_cache_args *a, size_t *bytes) {
    using namespace kvd;
    const char *who = "sp_hipkv_cache_attention_work";
    if (cache_check(who, a)) return 1;
    OP_NEED(bytes, "null bytes");
    *bytes = 0;
    const CachePlan p = cache_plan(*a);
    OP_NEED(cache_grid(*a, p) <= 1 << 22, "too many sequences, heads and tokens for one launch");
    if (p.nsplit > 1) *bytes = (size_t)a->n_tokens * a->n_heads * p.nsplit * (a->head_dim + 2) * 4;
    return 0;
}

extern "C" int sp_hipkv_cache_attention(const sp_hipkv_cache_args *a, void *stream) {
    using namespace kvd;
    const char *who = "sp_hipkv_cache_attention";
    if (cache_check(who, a)) return 1;
    if (!a->n_tokens) return 0;
    size_t need = 0;
    if (sp_hipkv_cache_attention_work(a, &need) || cache_check_arrays(who, a, need)) return 1;
    OpDevice dev((hipStream_t)stream);
    return op_done(who, dev.err != hipSuccess ? dev.err : launch_cache(*a, (hipStream_t)stream));
}
