// kvd_tree.hip -- attention of drafted token trees over the paged cache.
//
// Row (node, q head) sees the cached positions from its window start on and the
// nodes whose bit is set in its mask; out = sum_p w_p v_p / sum_p w_p with
//   f32, Spinor rows   w_p = e^(s_p - M), s_p = scale q.k_p, M the row's largest;
//   exact rows         z_p = llround(f32(<qi, ki_p> / 2^32) scale 2^14), qi = rne(q 2^16),
//                      w_p = exp_fixed((z_p - M) 2^16) >> 8, out = RNE(sum w vq / (2^16 sum w)),
// the decode attention's integers (kvd_attn.hip).
//
// f32 and Spinor rows run on the f32 matrix cores in one pass over K and V
// (k_tree_float), exact rows on the int8 matrix cores in two (k_tree_xscore, _xsum).
#include "kvd_op.h"
#include "kvd_exact.h"
#include "kvd_vec.h"
#include <algorithm>

namespace kvd {

namespace {

// What a workgroup needs of its sequence.
struct TreeSeq {
    const void *const *table;
    int cached, nodes, node0;
};
__device__ __forceinline__ TreeSeq tree_seq(const sp_hipkv_tree_args &a, int s) {
    TreeSeq q;
    q.node0 = max(a.node_start[s], 0);
    q.cached = min(max(a.cached[s], 0), a.max_positions);
    q.nodes = min(min(a.node_start[s + 1], a.n_nodes) - q.node0, min(a.max_nodes, a.max_positions - q.cached));
    q.table = gmem(a.tables)[s];
    return q;
}
__device__ __forceinline__ int tree_low(const sp_hipkv_tree_args &a, const TreeSeq &q, int node) {
    if (!a.window) return 0;
    const int lo = q.cached + min(max(a.depth[q.node0 + node], 0), 511) - a.window + 1;
    return min(max(lo, 0), q.cached);
}
__device__ __forceinline__ const uint8_t *tree_page(const sp_hipkv_tree_args &a, const TreeSeq &q, int pos) {
    const int lp = pos / PAGE;
    return (const uint8_t *)gmem(q.table)[a.ring_pages ? lp % a.ring_pages : lp];
}

__device__ __forceinline__ const uint8_t *uniform(const uint8_t *x) {
    const uint64_t p = (uint64_t)x;
    return (const uint8_t *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)p));
}

// ---------------------------------------------------------------- f32 and Spinor rows
// The q heads of a kv head share its K and V rows: the rows of one kv head are
// r = node G + q head of the group, 16 to a matrix tile, RT tiles to a workgroup.
// Its four waves take the 16-position quarters of the pages of a range (a split)
// in turn, each with all RT tiles, a running maximum, sum and output of its own; they
// meet in LDS at the end, the splits in k_tree_merge.
//
// K and V go from memory into the operands' registers directly, each byte once:
//   scores, transposed:  S^T = K Q^T, v_mfma_f32_16x16x4_f32, K the A operand (position
//     lane % 16, 4 consecutive dims of group lane / 16), Q the B operand, from LDS;
//   then lane l holds row l % 16 and positions 4 (l / 16) + i, as the A operand of
//     O += P V needs them; V is the B operand, a float4 of a row per lane.
// Two register buffers alternate, so that a stage (8 KiB a wave) is on its way while
// the one before is multiplied.  f32 products and sums throughout.
//
// The running maximum only moves when a score exceeds it by 2^8 in the exponent (base
// 2): weights stay below 2^8 and nothing is lost, and a tile needs one ballot instead of
// a reduction over lanes.  The sums are joined over lanes once at the end.
//
// A position that a row does not see has weight 0, which a V row that is not finite
// would turn into NaN: tiles that some row does not see whole look for such values
// first and are then put off to a loop behind the main one, which adds positions one
// by one (inside the main loop that path costs twice the output's registers).
typedef float v4f __attribute__((ext_vector_type(4)));
constexpr int TT = 16;                       // positions per tile: a quarter of a page
constexpr float LOG2E_F = 1.44269504088896341f;

__device__ __forceinline__ bool finite1(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

template <int ROWS, int EPL, int RT>
__global__ __launch_bounds__(256, 2) void k_tree_float(sp_hipkv_tree_args a, int groups, int nsplit) {
    constexpr int HD = EPL * 64, CPR = HD / 16, RB = row_bytes_of(ROWS, HD);
    constexpr bool SPN = ROWS == SP_HIPKV_ROWS_SPINOR;
    constexpr int NST = !SPN && EPL == 4 ? 2 : 1, NB = 4 * EPL / NST;      // stages of K (and of V) per tile, float4s per stage
    constexpr int LDS_F = RT * 16 * HD > 4 * 8 * HD ? RT * 16 * HD : 4 * 8 * HD;
    __shared__ __align__(16) float lds[LDS_F];                             // q rows, then the waves' outputs
    __shared__ float s_m[4][RT * 16], s_l[4][RT * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads;
    int id = blockIdx.x;
    const int h = id % a.n_kv_heads; id /= a.n_kv_heads;
    const int grp = id % groups; id /= groups;
    const int split = id % nsplit;
    const TreeSeq q = tree_seq(a, id / nsplit);
    const int R = q.nodes * G, r0 = grp * RT * 16;
    if (r0 >= R) return;
    const int end = q.cached + q.nodes;
    // this lane's rows, one of each tile: where it starts to see, its mask
    int low[RT], nodei[RT], lo_min = INT32_MAX, lo_max = 0;
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        const int r = r0 + t * 16 + l16;
        nodei[t] = (r < R ? r : R - 1) / G;
        low[t] = tree_low(a, q, nodei[t]);
        lo_min = min(lo_min, low[t]); lo_max = max(lo_max, low[t]);
    }
    if (a.window) {
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1) { lo_min = min(lo_min, __shfl_xor(lo_min, o, 64)); lo_max = max(lo_max, __shfl_xor(lo_max, o, 64)); }
    }
    lo_min = __builtin_amdgcn_readfirstlane(lo_min); lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    // this split's pages, and this wave's of them
    const int pg0 = lo_min / PAGE, pg1 = (end + PAGE - 1) / PAGE, per = (pg1 - pg0 + nsplit - 1) / nsplit;
    int w0 = pg0 + split * per, w1 = min(w0 + per, pg1);
    if (w0 < w1 && w0 * PAGE + wave * TT + TT <= lo_min) w0++;
    if (w0 < w1 && (w1 - 1) * PAGE + wave * TT >= end) w1--;
    v4f *qs = (v4f *)lds;
    for (int i = threadIdx.x; i < RT * 16 * (HD / 4); i += 256) {
        const int r = i / (HD / 4), c = i % (HD / 4), rr = r0 + r < R ? r0 + r : R - 1;
        qs[r * (HD / 4) + (c ^ (r & 15))] = *(const v4f *)(a.q + (size_t)(q.node0 + rr / G) * a.q_stride + (size_t)(h * G + rr % G) * HD + 4 * c);
    }
    v4f O[RT][CPR], S[RT];
    float m[RT], l[RT];
    uint32_t see[RT];
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        m[t] = -INFINITY; l[t] = 0.0f; see[t] = 15;
        #pragma unroll
        for (int c = 0; c < CPR; c++) O[t][c] = (v4f){0, 0, 0, 0};
    }
    __syncthreads();
    const uint32_t kslice = (uint32_t)h * PAGE * RB, vslice = (uint32_t)(a.n_kv_heads + h) * PAGE * RB;
    // page addresses are the wave's: rows load as address + 32-bit lane offset
    auto page = [&](int lp) { return uniform(tree_page(a, q, lp * PAGE)); };
    // positions past the last one repeat it
    auto row_off = [&](int lp, int x) { const int p = lp * PAGE + wave * TT + x; return (uint32_t)((p < end ? p : end - 1) & (PAGE - 1)) * RB; };
    // tiles that some row does not see whole, and those of them put off to the end:
    // nodes span at most 9 pages, so do the rows' window starts
    auto ragged = [&](int lp) { const int p0 = lp * PAGE + wave * TT; return p0 < lo_max || p0 + TT > q.cached; };
    const int tail_pg = q.cached / PAGE;
    uint32_t later = 0;
    auto put_off = [&](int lp) { later |= lp >= tail_pg ? 1u << (lp - tail_pg) : 65536u << (lp - pg0); };
    auto next_off = [&] {
        const int b = __builtin_ctz(later);
        later &= later - 1;
        return b < 16 ? tail_pg + b : pg0 + b - 16;
    };
    // scores in base 2, masked; weights into S
    auto softmax = [&](int lp) {
        const int p0 = lp * PAGE + wave * TT;
        const bool whole = !ragged(lp);
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            float mx = -INFINITY;
            #pragma unroll
            for (int i = 0; i < 4; i++) S[t][i] *= a.scale * LOG2E_F;
            if (!whole) {
                see[t] = 0;
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int p = p0 + 4 * g + i, j = p - q.cached;
                    bool v = p >= low[t];
                    if (j >= 0) v = j < q.nodes && (gmem(a.visible)[(size_t)(q.node0 + nodei[t]) * a.mask_words + (j >> 6)] >> (j & 63) & 1);
                    see[t] |= (uint32_t)v << i;
                    S[t][i] = v ? S[t][i] : -INFINITY;
                }
            }
            #pragma unroll
            for (int i = 0; i < 4; i++) mx = fmaxf(mx, S[t][i]);
            if (__any(mx > m[t] + 8.0f)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m[t], mx), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                l[t] *= al;
                #pragma unroll
                for (int i = 0; i < 4; i++) {                              // O's rows are 4 g + i
                    const float f = __shfl(al, 4 * g + i, 64);
                    #pragma unroll
                    for (int c = 0; c < CPR; c++) O[t][c][i] *= f;
                }
            }
            const float ms = m[t] == -INFINITY ? 0.0f : m[t];
            #pragma unroll
            for (int i = 0; i < 4; i++) { S[t][i] = __builtin_amdgcn_exp2f(S[t][i] - ms); l[t] += S[t][i]; }
        }
    };
    // O[t][c0 + c] += P x(e, c), positions 4 g + e, N columns
    auto pv = [&](auto n, int c0, auto &&x) {
        constexpr int N = decltype(n)::value;
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            #pragma unroll
            for (int c = 0; c < N; c++) {
                const float v = x(e, c);
                #pragma unroll
                for (int t = 0; t < RT; t++) O[t][c0 + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[t][e], v, O[t][c0 + c], 0, 0, 0);
                if (SPN && c % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // the same position by position, for the rows that see it; x4(p, k): columns 4 k .. of this lane
    auto pv_slow = [&](int lp, auto &&x4) {
        for (int p = 0; p < TT && lp * PAGE + wave * TT + p < end; p++) {
            const int from = (p >> 2) * 16, pe = p & 3;
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                const float we = pe == 0 ? S[t][0] : pe == 1 ? S[t][1] : pe == 2 ? S[t][2] : S[t][3];
                float w[4];
                bool on[4];
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    w[i] = __shfl(we, from + 4 * g + i, 64);
                    on[i] = __shfl(see[t], from + 4 * g + i, 64) >> pe & 1;
                }
                #pragma unroll
                for (int k = 0; k < CPR / 4; k++) {
                    const v4f v = x4(p, k);
                    #pragma unroll
                    for (int c = 0; c < 4; c++)
                        #pragma unroll
                        for (int i = 0; i < 4; i++) O[t][4 * k + c][i] = on[i] ? O[t][4 * k + c][i] + w[i] * v[c] : O[t][4 * k + c][i];
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };
    auto zero_s = [&] {
        #pragma unroll
        for (int t = 0; t < RT; t++) S[t] = (v4f){0, 0, 0, 0};
    };
    if constexpr (!SPN) {
        // column of O[t][c], row 4 g + i: 64 (c / 4) + 4 l16 + c % 4
        auto load_k = [&](v4f (&x)[NB], const uint8_t *pg, int lp, int st) {
            const uint32_t off = kslice + row_off(lp, l16) + 16 * g + st * NB * 64;
            #pragma unroll
            for (int s = 0; s < NB; s++) x[s] = *gmem((const v4f *)(pg + off + 64 * s));
        };
        auto load_v = [&](v4f (&x)[NB], const uint8_t *pg, int lp, int st) {
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t off = vslice + row_off(lp, 4 * g + e) + 16 * l16 + st * NB * 64;
                #pragma unroll
                for (int u = 0; u < NB / 4; u++) x[e * (NB / 4) + u] = *gmem((const v4f *)(pg + off + 256 * u));
            }
        };
        auto scores = [&](const v4f (&x)[NB], int st) {
            #pragma unroll
            for (int s = 0; s < NB; s++) {
                v4f qv[RT];
                #pragma unroll
                for (int t = 0; t < RT; t++) qv[t] = qs[(t * 16 + l16) * (HD / 4) + ((4 * (st * NB + s) + g) ^ l16)];
                #pragma unroll
                for (int e = 0; e < 4; e++)
                    #pragma unroll
                    for (int t = 0; t < RT; t++) S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s][e], qv[t][e], S[t], 0, 0, 0);
                if (s % 2) __builtin_amdgcn_sched_barrier(0);              // few q reads ahead at a time
            }
        };
        auto values = [&](const v4f (&x)[NB], int st) {
            pv(std::integral_constant<int, NB>{}, st * NB, [&](int e, int c) { return x[e * (NB / 4) + c / 4][c % 4]; });
        };
        v4f A[NB], B[NB];
        const uint8_t *pg = nullptr, *pn = nullptr;
        if (w0 < w1) {
            pg = page(w0);
            load_k(A, pg, w0, 0);
            if (NST == 2) load_k(B, pg, w0, 1); else load_v(B, pg, w0, 0);
            pn = page(min(w0 + 1, w1 - 1));
        }
        for (int lp = w0; lp < w1; lp++) {
            const int nx = min(lp + 1, w1 - 1);
            zero_s();
            scores(A, 0);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (NST == 2) {
                load_v(A, pg, lp, 0);
                __builtin_amdgcn_sched_barrier(0);
                scores(B, 1);
                __builtin_amdgcn_sched_barrier(0);
                load_v(B, pg, lp, 1);
            } else {
                load_k(A, pn, nx, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            bool bad = false;
            if (ragged(lp)) {
                #pragma unroll
                for (int s = 0; s < NB; s++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) bad |= !finite1(B[s][e]) || (NST == 2 && !finite1(A[s][e]));
            }
            bad = __any(bad);
            if (bad) put_off(lp); else softmax(lp);
            if constexpr (NST == 2) {
                if (!bad) values(A, 0);
                __builtin_amdgcn_sched_barrier(0);
                load_k(A, pn, nx, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (!bad) values(B, 1);
                __builtin_amdgcn_sched_barrier(0);
                load_k(B, pn, nx, 1);
            } else {
                if (!bad) values(B, 0);
                __builtin_amdgcn_sched_barrier(0);
                load_v(B, pn, nx, 0);
            }
            pg = pn;
            pn = page(min(lp + 2, w1 - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        while (later) {
            const int lp = next_off();
            pg = page(lp);
            zero_s();
            for (int st = 0; st < NST; st++) { load_k(A, pg, lp, st); scores(A, st); }
            softmax(lp);
            pv_slow(lp, [&](int p, int k) { return *gmem((const v4f *)(pg + vslice + row_off(lp, p) + 16 * l16 + 256 * k)); });
        }
    } else {
        // K: 16 codes of dims 64 i + 16 g.. a load; V: the CPR codes of columns CPR l16..
        // (O[t][c] is column CPR l16 + c), and the multipliers of the at most two
        // chunks that they lie in
        constexpr int NM = spn_blocks(HD);
        struct KRow { uint4 c[EPL]; float m[NM]; };
        struct VRow { uint32_t c[EPL]; float m0, m1; };
        const int d0v = CPR * l16, b0v = spn_block_of(HD, d0v), bnd0 = spn_block_start(HD, b0v + 1), b1v = bnd0 < d0v + CPR ? b0v + 1 : b0v;
        int bndv = bnd0;
        auto load_k = [&](KRow &x, const uint8_t *pg, int lp) {
            const uint8_t *row = pg + kslice + row_off(lp, l16);
            #pragma unroll
            for (int i = 0; i < EPL; i++) x.c[i] = *gmem((const uint4 *)(row + 64 * i + 16 * g));
            #pragma unroll
            for (int b = 0; b < NM; b++) x.m[b] = *gmem((const float *)(row + HD + 4 * b));
        };
        auto load_v = [&](VRow (&x)[4], const uint8_t *pg, int lp) {
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint8_t *row = pg + vslice + row_off(lp, 4 * g + e);
                #pragma unroll
                for (int i = 0; i < EPL; i++) x[e].c[i] = *gmem((const uint32_t *)(row + d0v + 4 * i));
                x[e].m0 = *gmem((const float *)(row + HD + 4 * b0v));
                x[e].m1 = *gmem((const float *)(row + HD + 4 * b1v));
            }
        };
        auto code = [](uint32_t w, int t) { return (float)(int32_t)(int8_t)(w >> (8 * t)); };
        auto scores = [&](const KRow &x) {
            #pragma unroll
            for (int i = 0; i < EPL; i++) {
                const int d0 = 64 * i + 16 * g, b = spn_block_of(HD, d0);
                int bnd = spn_block_start(HD, b + 1);
                asm volatile("" : "+v"(bnd));                              // compared where used: kept masks would fill the scalar registers
                float m0 = x.m[0], m1 = x.m[0];
                #pragma unroll
                for (int bb = 1; bb < NM; bb++) { if (b == bb) m0 = x.m[bb]; if (b + 1 == bb) m1 = x.m[bb]; }
                const uint32_t w[4] = {x.c[i].x, x.c[i].y, x.c[i].z, x.c[i].w};
                #pragma unroll
                for (int k = 0; k < 4; k++) {
                    v4f qv[RT];
                    #pragma unroll
                    for (int t = 0; t < RT; t++) qv[t] = qs[(t * 16 + l16) * (HD / 4) + ((16 * i + 4 * g + k) ^ l16)];
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float kv = code(w[k], e) * (d0 + 4 * k + e < bnd ? m0 : m1);
                        #pragma unroll
                        for (int t = 0; t < RT; t++) S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv, qv[t][e], S[t], 0, 0, 0);
                    }
                    if (k % 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        KRow K;
        VRow V[4];
        const uint8_t *pg = nullptr, *pn = nullptr;
        if (w0 < w1) {
            pg = page(w0);
            load_k(K, pg, w0);
            load_v(V, pg, w0);
            pn = page(min(w0 + 1, w1 - 1));
        }
        for (int lp = w0; lp < w1; lp++) {
            const int nx = min(lp + 1, w1 - 1);
            zero_s();
            scores(K);
            __builtin_amdgcn_sched_barrier(0);
            load_k(K, pn, nx);
            __builtin_amdgcn_sched_barrier(0);
            bool bad = false;
            if (ragged(lp)) {
                #pragma unroll
                for (int e = 0; e < 4; e++) bad |= !finite1(127.0f * V[e].m0) || !finite1(127.0f * V[e].m1);
            }
            if (__any(bad)) {
                put_off(lp);
            } else {
                softmax(lp);
                asm volatile("" : "+v"(bndv));
                pv(std::integral_constant<int, CPR>{}, 0, [&](int e, int c) { return code(V[e].c[c / 4], c % 4) * (d0v + c < bndv ? V[e].m0 : V[e].m1); });
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(V, pn, nx);
            pg = pn;
            pn = page(min(lp + 2, w1 - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        while (later) {
            const int lp = next_off();
            pg = page(lp);
            zero_s();
            load_k(K, pg, lp);
            scores(K);
            softmax(lp);
            pv_slow(lp, [&](int p, int k) {
                const uint8_t *row = pg + vslice + row_off(lp, p);
                const uint32_t w = *gmem((const uint32_t *)(row + d0v + 4 * k));
                const float m0 = *gmem((const float *)(row + HD + 4 * b0v)), m1 = *gmem((const float *)(row + HD + 4 * b1v));
                v4f v;
                #pragma unroll
                for (int c = 0; c < 4; c++) v[c] = code(w, c) * (d0v + 4 * k + c < bndv ? m0 : m1);
                return v;
            });
        }
    }
    // the four waves' parts: m and l first
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
        if (g == 0) { s_m[wave][t * 16 + l16] = m[t]; s_l[wave][t * 16 + l16] = l[t]; }
    }
    __syncthreads();                                                       // ... and nobody reads q any more
    float *po = (float *)a.work, *pml = po + (size_t)a.n_nodes * a.n_heads * nsplit * HD;
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int ih = 0; ih < 2; ih++) {                                   // rows 4 g + 2 ih, + 1
            #pragma unroll
            for (int i = 2 * ih; i < 2 * ih + 2; i++) {
                const int r = t * 16 + 4 * g + i;
                const float M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
                const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[wave][r] - M);
                v4f *dst = (v4f *)lds + ((wave * 8 + 2 * g + (i & 1)) * (HD / 4));
                #pragma unroll
                for (int c = 0; c < CPR; c += 4) {
                    const v4f x = {O[t][c][i], O[t][c + 1][i], O[t][c + 2][i], O[t][c + 3][i]};
                    dst[SPN ? (CPR / 4) * l16 + c / 4 : 4 * c + l16] = f == 0.0f ? (v4f){0, 0, 0, 0} : x * f;
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 8 * (HD / 4); i += 256) {
                const int k = i / (HD / 4), c = i % (HD / 4), rl = t * 16 + 4 * (k >> 1) + 2 * ih + (k & 1), r = r0 + rl;
                if (r >= R) continue;
                const v4f *src = (const v4f *)lds + k * (HD / 4) + c;
                v4f x = (src[0] + src[8 * (HD / 4)]) + (src[16 * (HD / 4)] + src[24 * (HD / 4)]);
                const float M = fmaxf(fmaxf(s_m[0][rl], s_m[1][rl]), fmaxf(s_m[2][rl], s_m[3][rl]));
                float L = 0.0f;
                if (M > -INFINITY)
                    #pragma unroll
                    for (int w = 0; w < 4; w++) L += s_l[w][rl] * __builtin_amdgcn_exp2f(s_m[w][rl] - M);
                const int node = q.node0 + r / G, head = h * G + r % G;
                if (nsplit == 1) {
                    *(v4f *)(a.out + (size_t)node * a.out_stride + (size_t)head * HD + 4 * c) = M == -INFINITY ? (v4f){0, 0, 0, 0} : x / L;
                } else {
                    const size_t at = ((size_t)node * a.n_heads + head) * nsplit + split;
                    if (M > -INFINITY) *(v4f *)(po + at * HD + 4 * c) = x;
                    if (c == 0) { pml[2 * at] = M; pml[2 * at + 1] = L; }
                }
            }
            if (t < RT - 1 || ih == 0) __syncthreads();
        }
}

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c; HD / 4 threads a row
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(sp_hipkv_tree_args a, int nsplit) {
    const size_t row = (size_t)blockIdx.x * (1024 / HD) + threadIdx.x / (HD / 4);
    if (row >= (size_t)a.n_nodes * a.n_heads) return;
    const int c = threadIdx.x % (HD / 4);
    const v4f *po = (const v4f *)((const float *)a.work + row * nsplit * HD) + c;
    const float *ml = (const float *)a.work + (size_t)a.n_nodes * a.n_heads * nsplit * HD + 2 * row * nsplit;
    float M = -INFINITY, L = 0.0f;
    for (int k = 0; k < nsplit; k++) M = fmaxf(M, ml[2 * k]);
    v4f x = {0, 0, 0, 0};
    #pragma unroll 8
    for (int k = 0; k < nsplit; k++) {
        const float mk = ml[2 * k];
        if (!(mk > -INFINITY)) continue;                                   // a part without a position of this row
        const float f = __builtin_amdgcn_exp2f(mk - M);
        L += f * ml[2 * k + 1];
        x += f * po[(size_t)k * (HD / 4)];
    }
    *(v4f *)(a.out + (row / a.n_heads) * a.out_stride + (row % a.n_heads) * HD + 4 * c) = M > -INFINITY ? x / L : (v4f){0, 0, 0, 0};
}

// ---------------------------------------------------------------- exact rows
// Integer sums are exact in any order, so both products run on the int8 matrix cores
// (v_mfma_i32_16x16x64_i8) over balanced base-256 digits, three of each number where
// they fit (|x| <= 127 (1 + 2^8 + 2^16)); products of equal place share an int32 sum.
//   k_tree_xscore: z of every (row, position) into `work`, and each split's maxima;
//   k_tree_xsum:   weights (22 bits) from z and M, V sums as int64 of a split;
//   k_tree_xdiv:   the splits' sums, divided.
// The weights need M before the first of them, hence z in memory: 4 bytes a row and
// position, written and read once, against 8 HD bytes of K and V for all G nodes rows.
//
// Scores: as in the f32 kernel a wave takes 16 positions straight into registers, here
// as the B operand (16 dims a lane and step, in an order that q's digits in LDS
// share), makes their digits once and multiplies them with all row tiles.
// V sums: a wave owns 32 columns and takes a page a step: lane l 16 positions of two
// columns, which are the B operand after their digits are formed; no transposition.
// The weights' digits are made once for all waves and pass through LDS.
typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int DIG3 = 127 * (1 + 256 + 65536);                    // largest |x| of three balanced digits
constexpr int DIG4 = 127 * (1 + 256 + 65536 + 16777216);         // ... of four

// x = d0 + 2^8 d1 + 2^16 d2 + 2^24 d3, d in [-128, 127]; four values' digits, one dword per place
__device__ __forceinline__ void digits_of(const int32_t x[4], uint32_t w[4]) {
    uint32_t d[4];
    #pragma unroll
    for (int e = 0; e < 4; e++) d[e] = ((uint32_t)x[e] + 0x80808080u) ^ 0x80808080u;
    const uint32_t ab0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), ab2 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
    const uint32_t cd0 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), cd2 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u); w[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u); w[3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}
// 1: |x| needs a fourth digit, 2: more than four
__device__ __forceinline__ int level_of(int32_t x) {
    return ((uint32_t)x + (uint32_t)DIG3 > 2u * DIG3 ? 1 : 0) | ((uint32_t)x + (uint32_t)DIG4 > 2u * DIG4 ? 2 : 0);
}
// exp_fixed((z - M) 2^16) >> 8 for z <= M: 2^-g, g = ceil((M - z) log2(e) 2^30 / 2^14) in 30 bits
__device__ __forceinline__ int32_t weight_of(int32_t z, int32_t M) {
    const uint64_t g = ((uint64_t)((uint32_t)M - (uint32_t)z) * (uint32_t)LOG2E + 16383) >> 14;
    const uint32_t n = (uint32_t)(g >> FB), r = (uint32_t)g & (uint32_t)(ONE - 1);
    if (n >= 23) return 0;
    return r ? (int32_t)(exp2_frac((uint32_t)ONE - r) >> (n + 9)) : (int32_t)((uint32_t)ONE >> (n + 8));
}

// Work of exact rows: z [row][zstride], maxima [row][nsplit], V sums [row][vsplit][HD],
// denominators [row][vsplit]; row = node n_heads + head.
struct XWork { int32_t *z, *zmax; int64_t *sum, *den; int zstride, nsplit, vsplit; };
// z is kept by position less the first page's that any node of the sequence sees
__device__ __forceinline__ int z_first(const sp_hipkv_tree_args &a, const TreeSeq &q) {
    return a.window ? max(q.cached - a.window + 1, 0) & ~(PAGE - 1) : 0;
}
// the span of pages that rows [r0, r1) of a kv head see
struct Span { int lo_min, lo_max, pg0, pg1; };
__device__ __forceinline__ Span rows_span(const sp_hipkv_tree_args &a, const TreeSeq &q, int G, int r0, int r1) {
    Span s = {0, 0, 0, (q.cached + q.nodes + PAGE - 1) / PAGE};
    if (a.window) {
        s.lo_min = INT32_MAX;
        for (int r = r0 + (int)(threadIdx.x & 63); r < r1; r += 64) {
            const int lo = tree_low(a, q, r / G);
            s.lo_min = min(s.lo_min, lo); s.lo_max = max(s.lo_max, lo);
        }
        s.lo_max = wave_allmax_i(s.lo_max);
        s.lo_min = -wave_allmax_i(-s.lo_min);
    }
    s.pg0 = s.lo_min / PAGE;
    return s;
}
__device__ __forceinline__ bool row_sees(const sp_hipkv_tree_args &a, const TreeSeq &q, int node, int p) {
    const int j = p - q.cached;
    if (j < 0) return p >= tree_low(a, q, node);
    return j < q.nodes && (gmem(a.visible)[(size_t)(q.node0 + node) * a.mask_words + (j >> 6)] >> (j & 63) & 1);
}

template <int EPL, int RT>
__global__ __launch_bounds__(256, 2) void k_tree_xscore(sp_hipkv_tree_args a, XWork x, int groups) {
    constexpr int HD = EPL * 64, KS = EPL, QROW = HD + 16;
    __shared__ __align__(16) int8_t qd[4][RT * 16][QROW];          // q's digits [place][row][64 ks + 16 g + 4 quarter + e]
    __shared__ int s_level, s_mx[4][RT * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads;
    int id = blockIdx.x;
    const int h = id % a.n_kv_heads; id /= a.n_kv_heads;
    const int grp = id % groups; id /= groups;
    const int split = id % x.nsplit;
    const TreeSeq q = tree_seq(a, id / x.nsplit);
    const int R = q.nodes * G, r0 = grp * RT * 16;
    if (r0 >= R) return;
    if (threadIdx.x == 0) s_level = 0;
    __syncthreads();
    const int end = q.cached + q.nodes, z0 = z_first(a, q);
    int level = 0;
    for (int i = threadIdx.x; i < RT * 16 * (HD / 4); i += 256) {
        const int r = i / (HD / 4), c = i % (HD / 4);
        int32_t v[4] = {0, 0, 0, 0};
        if (r0 + r < R) {
            const float4 f = *(const float4 *)(a.q + (size_t)(q.node0 + (r0 + r) / G) * a.q_stride + (size_t)(h * G + (r0 + r) % G) * HD + 4 * c);
            v[0] = (int32_t)rintf(f.x * 65536.0f); v[1] = (int32_t)rintf(f.y * 65536.0f);
            v[2] = (int32_t)rintf(f.z * 65536.0f); v[3] = (int32_t)rintf(f.w * 65536.0f);
        }
        uint32_t w[4];
        #pragma unroll
        for (int e = 0; e < 4; e++) level |= level_of(v[e]);
        digits_of(v, w);
        // dims 64 ks + 16 quarter + 4 g + e
        const int at = (c / 16) * 64 + (c % 4) * 16 + (c / 4 % 4) * 4;
        #pragma unroll
        for (int b = 0; b < 4; b++) *(uint32_t *)&qd[b][r][at] = w[b];
    }
    level = (__any(level & 1) ? 1 : 0) | (__any(level & 2) ? 2 : 0);
    if (level && lane == 0) atomicOr(&s_level, level);
    const Span sp = rows_span(a, q, G, r0, min(r0 + RT * 16, R));
    const int per = (sp.pg1 - sp.pg0 + x.nsplit - 1) / x.nsplit;
    int w0 = sp.pg0 + split * per, w1 = min(w0 + per, sp.pg1);
    if (w0 < w1 && w0 * PAGE + wave * TT + TT <= sp.lo_min) w0++;
    if (w0 < w1 && (w1 - 1) * PAGE + wave * TT >= end) w1--;
    // this lane's output rows: 4 g + i of each tile
    int mx[RT][4], zrow[RT][4];
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + t * 16 + 4 * g + i;
            mx[t][i] = INT32_MIN;
            zrow[t][i] = r < R ? (q.node0 + r / G) * a.n_heads + h * G + r % G : -1;
        }
    __syncthreads();
    const int qlevel = s_level;
    const uint32_t kslice = (uint32_t)h * PAGE * HD * 4;
    auto page = [&](int lp) { return uniform(tree_page(a, q, lp * PAGE)); };
    auto load_k = [&](v4i (&k)[4 * KS], const uint8_t *pg, int lp) {
        const int p = lp * PAGE + wave * TT + l16;
        const uint32_t off = kslice + (uint32_t)((p < end ? p : end - 1) & (PAGE - 1)) * (HD * 4) + 16 * g;
        #pragma unroll
        for (int s = 0; s < 4 * KS; s++) k[s] = *gmem((const v4i *)(pg + off + 64 * s));
    };
    v4i K[4 * KS];
    const uint8_t *pg = nullptr, *pn = nullptr;
    if (w0 < w1) {
        pg = page(w0);
        load_k(K, pg, w0);
        pn = page(min(w0 + 1, w1 - 1));
    }
    for (int lp = w0; lp < w1; lp++) {
        const int p0 = lp * PAGE + wave * TT, p = p0 + l16;
        const bool whole = p0 >= sp.lo_max && p0 + TT <= q.cached;
        v4i B[4][KS];
        int lv = 0;
        #pragma unroll
        for (int s = 0; s < 4 * KS; s++) {
            const int32_t v[4] = {K[s][0], K[s][1], K[s][2], K[s][3]};
            uint32_t w[4];
            #pragma unroll
            for (int e = 0; e < 4; e++) lv |= level_of(v[e]);
            digits_of(v, w);
            #pragma unroll
            for (int b = 0; b < 4; b++) B[b][s / 4][s % 4] = (int)w[b];
        }
        lv = qlevel | (__any(lv & 1) ? 1 : 0) | (__any(lv & 2) ? 2 : 0);
        __builtin_amdgcn_sched_barrier(0);
        load_k(K, pn, min(lp + 1, w1 - 1));
        __builtin_amdgcn_sched_barrier(0);
        auto dots = [&](auto nd, int t, int64_t (&ip)[4]) {
            constexpr int ND = decltype(nd)::value;
            v4i acc[2 * ND - 1];
            #pragma unroll
            for (int k = 0; k < 2 * ND - 1; k++) acc[k] = (v4i){0, 0, 0, 0};
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                v4i A[ND];
                #pragma unroll
                for (int b = 0; b < ND; b++) A[b] = *(const v4i *)&qd[b][t * 16 + l16][64 * ks + 16 * g];
                #pragma unroll
                for (int u = 0; u < ND; u++)
                    #pragma unroll
                    for (int b = 0; b < ND; b++) acc[u + b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[u], B[b][ks], acc[u + b], 0, 0, 0);
            }
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                ip[i] = acc[2 * ND - 2][i];
                #pragma unroll
                for (int k = 2 * ND - 3; k >= 0; k--) ip[i] = ip[i] * 256 + acc[k][i];
            }
        };
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            int64_t ip[4];
            if (lv == 0) dots(std::integral_constant<int, 3>{}, t, ip);
            else if (lv == 1) dots(std::integral_constant<int, 4>{}, t, ip);
            else {                                                         // more than four digits: from the numbers
                const int32_t *kr = (const int32_t *)(pg + kslice) + (size_t)((p < end ? p : end - 1) & (PAGE - 1)) * HD;
                for (int i = 0; i < 4; i++) {
                    const int r = min(r0 + t * 16 + 4 * g + i, R - 1);
                    const float *qr = a.q + (size_t)(q.node0 + r / G) * a.q_stride + (size_t)(h * G + r % G) * HD;
                    int64_t s = 0;
                    for (int d = 0; d < HD; d++) s += (int64_t)(int32_t)rintf(qr[d] * 65536.0f) * gmem(kr)[d];
                    ip[i] = s;
                }
            }
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const float sc = (float)((double)ip[i] / 4294967296.0) * a.scale;
                const int32_t z = (int32_t)llround_pow2<14>(sc);
                if (zrow[t][i] >= 0 && p < end) {
                    x.z[(size_t)zrow[t][i] * x.zstride + (p - z0)] = z;
                    if (whole || row_sees(a, q, zrow[t][i] / a.n_heads - q.node0, p)) mx[t][i] = max(mx[t][i], z);
                }
            }
        }
        pg = pn;
        pn = page(min(lp + 2, w1 - 1));
    }
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            #pragma unroll
            for (int o = 1; o < 16; o <<= 1) mx[t][i] = max(mx[t][i], __shfl_xor(mx[t][i], o, 64));
            if (l16 == 0) s_mx[wave][t * 16 + 4 * g + i] = mx[t][i];
        }
    __syncthreads();
    if (threadIdx.x < RT * 16 && r0 + (int)threadIdx.x < R) {
        const int r = r0 + threadIdx.x, k = threadIdx.x;
        x.zmax[((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * x.nsplit + split] = max(max(s_mx[0][k], s_mx[1][k]), max(s_mx[2][k], s_mx[3][k]));
    }
}

// waves: HD / 32; one page a step
template <int EPL, int RT>
__global__ __launch_bounds__(EPL * 128, 2) void k_tree_xsum(sp_hipkv_tree_args a, XWork x, int groups) {
    constexpr int HD = EPL * 64, NT = EPL * 128, ROWS = RT * 16, WROW = PAGE + 16;
    constexpr int QUADS = (ROWS * 16 + NT - 1) / NT;                           // position quads of a thread and step
    __shared__ __align__(16) int8_t wd[2][3][ROWS][WROW];                      // weights' digits [step parity][place][row][position]
    __shared__ int s_M[ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads;
    int id = blockIdx.x;
    const int h = id % a.n_kv_heads; id /= a.n_kv_heads;
    const int grp = id % groups; id /= groups;
    const int split = id % x.vsplit;
    const TreeSeq q = tree_seq(a, id / x.vsplit);
    const int R = q.nodes * G, r0 = grp * ROWS;
    if (r0 >= R) return;
    const int end = q.cached + q.nodes, z0 = z_first(a, q);
    const Span sp = rows_span(a, q, G, r0, min(r0 + ROWS, R));
    const int per = (sp.pg1 - sp.pg0 + x.vsplit - 1) / x.vsplit, b0 = sp.pg0 + split * per, b1 = min(b0 + per, sp.pg1);
    for (int k = threadIdx.x; k < ROWS; k += NT) {
        int M = INT32_MIN;
        if (r0 + k < R) {
            const int32_t *m = x.zmax + ((size_t)(q.node0 + (r0 + k) / G) * a.n_heads + h * G + (r0 + k) % G) * x.nsplit;
            for (int c = 0; c < x.nsplit; c++) M = max(M, m[c]);
        }
        s_M[k] = M;
    }
    __syncthreads();
    // this thread's weights: positions 4 (tid % 16) .. of rows tid / 16 + k NT / 16
    const int quad = threadIdx.x & 15;
    int64_t den[QUADS];
    int zrow[QUADS], M[QUADS], node[QUADS];
    #pragma unroll
    for (int k = 0; k < QUADS; k++) {
        const int rl = threadIdx.x / 16 + k * (NT / 16), r = r0 + rl;
        den[k] = 0;
        const bool live = rl < ROWS && r < R && s_M[rl < ROWS ? rl : 0] > INT32_MIN;   // (no position seen: weights stay 0)
        node[k] = live ? r / G : -1;
        zrow[k] = live ? (q.node0 + r / G) * a.n_heads + h * G + r % G : 0;
        M[k] = s_M[rl < ROWS ? rl : 0];
    }
    int4 z[QUADS];
    auto load_z = [&](int lp) {
        #pragma unroll
        for (int k = 0; k < QUADS; k++)
            if (node[k] >= 0) z[k] = *(const int4 *)(x.z + (size_t)zrow[k] * x.zstride + (lp * PAGE - z0 + 4 * quad));
    };
    auto weights = [&](int lp, int par) {
        const int p0 = lp * PAGE;
        const bool whole = p0 >= sp.lo_max && p0 + PAGE <= q.cached;
        #pragma unroll
        for (int k = 0; k < QUADS; k++) {
            if ((int)threadIdx.x / 16 + k * (NT / 16) >= ROWS) break;
            int32_t w[4] = {0, 0, 0, 0};
            if (node[k] >= 0) {
                const int32_t zz[4] = {z[k].x, z[k].y, z[k].z, z[k].w};
                #pragma unroll
                for (int e = 0; e < 4; e++)
                    if (whole || row_sees(a, q, node[k], p0 + 4 * quad + e)) w[e] = weight_of(zz[e], M[k]);
            }
            den[k] += (int64_t)w[0] + w[1] + w[2] + w[3];
            uint32_t d[4];
            digits_of(w, d);
            #pragma unroll
            for (int b = 0; b < 3; b++) *(uint32_t *)&wd[par][b][threadIdx.x / 16 + k * (NT / 16)][4 * quad] = d[b];
        }
    };
    const uint32_t vslice = (uint32_t)(a.n_kv_heads + h) * PAGE * HD * 4;
    typedef int v2i __attribute__((ext_vector_type(2)));
    v2i V[16];
    // lane: positions 16 g + j of columns 32 wave + 2 l16, + 1
    auto load_v = [&](const uint8_t *pg, int lp) {
        const uint32_t col = vslice + (32 * wave + 2 * l16) * 4;
        #pragma unroll
        for (int j = 0; j < 16; j++) {
            const int p = lp * PAGE + 16 * g + j;
            V[j] = *gmem((const v2i *)(pg + col + (uint32_t)((p < end ? p : end - 1) & (PAGE - 1)) * (HD * 4)));
        }
    };
    v4i acc[RT][2][5];
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int c = 0; c < 2; c++)
            #pragma unroll
            for (int k = 0; k < 5; k++) acc[t][c][k] = (v4i){0, 0, 0, 0};
    auto page = [&](int lp) { return uniform(tree_page(a, q, lp * PAGE)); };
    if (b0 < b1) { load_z(b0); load_v(page(b0), b0); }
    for (int lp = b0; lp < b1; lp++) {
        const int par = (lp - b0) & 1, nx = min(lp + 1, b1 - 1);
        const uint8_t *pn = page(nx);
        weights(lp, par);
        load_z(nx);
        __syncthreads();                                                   // (the other parity's readers are past it too)
        // |v| may exceed three digits by little: what is left goes through once more
        for (bool more = true; more;) {
            v4i B[2][3];
            int left = 0;
            #pragma unroll
            for (int c = 0; c < 2; c++)
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    int32_t v[4];
                    uint32_t d[4];
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        v[e] = min(max(V[4 * j + e][c], -DIG3), DIG3);
                        V[4 * j + e][c] -= v[e];
                        left |= V[4 * j + e][c];
                    }
                    digits_of(v, d);
                    #pragma unroll
                    for (int b = 0; b < 3; b++) B[c][b][j] = (int)d[b];
                }
            more = __any(left != 0);
            if (!more) {
                __builtin_amdgcn_sched_barrier(0);
                load_v(pn, nx);
                __builtin_amdgcn_sched_barrier(0);
            }
            #pragma unroll
            for (int t = 0; t < RT; t++)
                #pragma unroll
                for (int u = 0; u < 3; u++) {
                    const v4i A = *(const v4i *)&wd[par][u][t * 16 + l16][16 * g];
                    #pragma unroll
                    for (int b = 0; b < 3; b++)
                        #pragma unroll
                        for (int c = 0; c < 2; c++) acc[t][c][u + b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A, B[c][b], acc[t][c][u + b], 0, 0, 0);
                }
        }
    }
    // denominators: over a row's 16 threads
    #pragma unroll
    for (int k = 0; k < QUADS; k++) {
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1) den[k] += __shfl_xor(den[k], o, 64);
        const int rl = threadIdx.x / 16 + k * (NT / 16), r = r0 + rl;
        if (rl < ROWS && quad == 0 && r < R) x.den[((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * x.vsplit + split] = den[k];
    }
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + t * 16 + 4 * g + i;
            int64_t s[2];
            #pragma unroll
            for (int c = 0; c < 2; c++) {
                s[c] = acc[t][c][4][i];
                #pragma unroll
                for (int k = 3; k >= 0; k--) s[c] = s[c] * 256 + acc[t][c][k][i];
            }
            if (r < R) {
                int64_t *dst = x.sum + (((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * x.vsplit + split) * HD + 32 * wave + 2 * l16;
                dst[0] = s[0]; dst[1] = s[1];
            }
        }
}

// one output element per thread
template <int HD>
__global__ __launch_bounds__(256) void k_tree_xdiv(sp_hipkv_tree_args a, XWork x) {
    const size_t row = (size_t)blockIdx.x * (256 / HD) + threadIdx.x / HD;
    const int d = threadIdx.x % HD;
    if (row >= (size_t)a.n_nodes * a.n_heads) return;
    const int64_t *s = x.sum + row * x.vsplit * HD + d, *dn = x.den + row * x.vsplit;
    int64_t t = 0, den = 0;
    #pragma unroll 8
    for (int k = 0; k < x.vsplit; k++) { t += s[(size_t)k * HD]; den += dn[k]; }
    a.out[(row / a.n_heads) * a.out_stride + (row % a.n_heads) * HD + d] = den > 0 ? rne_div_to_float((i128)t, den, 16) : 0.0f;
}

// How a launch is cut: row tiles of a workgroup, workgroups along a sequence's rows,
// splits of its positions.
struct TreePlan { int rt, groups, nsplit; };
TreePlan tree_plan(const sp_hipkv_tree_args &a) {
    TreePlan p;
    const int most = a.head_dim == 256 ? 2 : 4, tiles = std::max(1, (a.max_nodes * (a.n_heads / a.n_kv_heads) + 15) / 16);
    p.groups = (tiles + most - 1) / most;
    p.rt = (tiles + p.groups - 1) / p.groups;
    const int span = a.window ? std::min(a.max_positions, a.window + a.max_nodes + PAGE) : a.max_positions;
    const int64_t base = (int64_t)a.n_kv_heads * p.groups * std::max(a.n_seqs, 1);
    const int64_t pages = std::max(1, (span + PAGE - 1) / PAGE);
    p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + base - 1) / base, (pages + 1) / 2, 64}));
    return p;
}

int tree_check(const char *who, const sp_hipkv_tree_args *a) {
    OP_NEED(a, "null arguments");
    OP_NEED(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256, "head_dim is not 64, 128 or 256");
    OP_NEED(a->n_kv_heads > 0 && a->n_heads > 0 && a->n_heads % a->n_kv_heads == 0 && a->n_heads / a->n_kv_heads <= 16 && a->n_heads <= 4096,
            "n_heads is not n_kv_heads times 1 to 16");
    OP_NEED(a->rows == SP_HIPKV_ROWS_F32 || a->rows == SP_HIPKV_ROWS_EXACT || a->rows == SP_HIPKV_ROWS_SPINOR, "unknown row format");
    OP_NEED(a->n_seqs >= 0 && a->n_seqs <= 4096, "n_seqs outside [0, 4096]");
    OP_NEED(a->n_nodes >= 0, "negative n_nodes");
    OP_NEED(a->max_nodes >= 0 && a->max_nodes <= 512, "max_nodes outside [0, 512]");
    OP_NEED(a->max_positions >= 0 && a->max_positions <= (a->rows == SP_HIPKV_ROWS_EXACT ? 1 << 18 : 1 << 20),
            "max_positions outside [0, 2^20] (exact rows: 2^18)");
    OP_NEED(a->n_nodes <= (int64_t)a->n_seqs * a->max_nodes, "n_nodes is more than n_seqs times max_nodes");
    OP_NEED((int64_t)a->n_nodes * a->n_heads <= 1 << 28, "more than 2^28 rows (n_nodes x n_heads)");
    OP_NEED(a->window >= 0 && a->ring_pages >= 0, "negative window or ring_pages");
    return 0;
}
int tree_check_arrays(const char *who, const sp_hipkv_tree_args *a, size_t need) {
    const int64_t row = (int64_t)a->n_heads * a->head_dim;
    OP_NEED(std::isfinite(a->scale), "scale is not finite");
    OP_NEED(a->mask_words >= (a->max_nodes + 63) / 64, "mask_words holds fewer than max_nodes bits");
    OP_NEED(a->node_start && a->cached && a->visible && a->tables && a->q && a->out, "null array");
    OP_NEED(a->depth || !a->window, "a window needs the nodes' depth");
    OP_NEED(a->q_stride >= row && a->out_stride >= row && a->q_stride % 4 == 0 && a->out_stride % 4 == 0,
            "q_stride or out_stride is below n_heads * head_dim or not a multiple of 4");
    OP_NEED(aligned(a->q, 16) && aligned(a->out, 16) && aligned(a->visible, 8) && aligned(a->tables, 8), "misaligned array");
    OP_NEED(!need || (a->work && a->work_bytes >= need && aligned(a->work, 16)), "work is missing, too small or not 16-byte aligned");
    return 0;
}

int64_t tree_grid(const sp_hipkv_tree_args &a, const TreePlan &p) { return (int64_t)a.n_kv_heads * p.groups * p.nsplit * a.n_seqs; }

template <int ROWS> void tree_float(const sp_hipkv_tree_args &a, hipStream_t s) {
    const TreePlan p = tree_plan(a);
    const dim3 grid((uint32_t)tree_grid(a, p)), wg(256);
#define TREE_RUN(EPL, RT) hipLaunchKernelGGL((k_tree_float<ROWS, EPL, RT>), grid, wg, 0, s, a, p.groups, p.nsplit)
    if (a.head_dim == 256) { if (p.rt == 1) TREE_RUN(4, 1); else TREE_RUN(4, 2); }
    else if (a.head_dim == 128) { if (p.rt == 1) TREE_RUN(2, 1); else if (p.rt == 2) TREE_RUN(2, 2); else if (p.rt == 3) TREE_RUN(2, 3); else TREE_RUN(2, 4); }
    else { if (p.rt == 1) TREE_RUN(1, 1); else if (p.rt == 2) TREE_RUN(1, 2); else if (p.rt == 3) TREE_RUN(1, 3); else TREE_RUN(1, 4); }
#undef TREE_RUN
    if (p.nsplit == 1) return;
    const int64_t rows = (int64_t)a.n_nodes * a.n_heads, per = 1024 / a.head_dim;
    const dim3 mg((uint32_t)((rows + per - 1) / per));
    if (a.head_dim == 256) hipLaunchKernelGGL(k_tree_merge<256>, mg, wg, 0, s, a, p.nsplit);
    else if (a.head_dim == 128) hipLaunchKernelGGL(k_tree_merge<128>, mg, wg, 0, s, a, p.nsplit);
    else hipLaunchKernelGGL(k_tree_merge<64>, mg, wg, 0, s, a, p.nsplit);
}

// Exact rows: both passes take up to 48 rows a workgroup; a V split's int32 sums hold
// 2 x 3 x 2^14 a position (values that need a second round of digits), so at most 2^14 positions.
struct XPlan { int rt, groups; XWork w; size_t bytes; };
XPlan tree_xplan(const sp_hipkv_tree_args &a) {
    XPlan p{};
    const int tiles = std::max(1, (a.max_nodes * (a.n_heads / a.n_kv_heads) + 15) / 16);
    const int most = a.head_dim == 64 ? 2 : 3;                   // row tiles whose sums a wave's registers hold
    p.groups = (tiles + most - 1) / most;
    p.rt = (tiles + p.groups - 1) / p.groups;
    const int span = a.window ? (int)std::min<int64_t>(a.max_positions, (int64_t)a.window + a.max_nodes + PAGE) : a.max_positions;
    const int64_t base = (int64_t)a.n_kv_heads * p.groups * std::max(a.n_seqs, 1), pages = std::max(1, (span + PAGE - 1) / PAGE + 1);
    p.w.zstride = (int)pages * PAGE;
    p.w.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + base - 1) / base, (pages + 1) / 2, 64}));
    p.w.vsplit = (int)std::max<int64_t>((pages * PAGE + 16383) >> 14, p.w.nsplit);
    const size_t rows = (size_t)a.n_nodes * a.n_heads;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    const size_t zb = up(rows * p.w.zstride * 4), mb = up(rows * p.w.nsplit * 4), sb = rows * p.w.vsplit * a.head_dim * 8;
    uint8_t *at = (uint8_t *)a.work;
    p.w.z = (int32_t *)at; p.w.zmax = (int32_t *)(at + zb); p.w.sum = (int64_t *)(at + zb + mb); p.w.den = (int64_t *)(at + zb + mb + sb);
    p.bytes = zb + mb + sb + up(rows * p.w.vsplit * 8);
    return p;
}
template <int EPL, int RT> void tree_xgo(const sp_hipkv_tree_args &a, const XPlan &p, hipStream_t s) {
    const int64_t one = (int64_t)a.n_kv_heads * p.groups * a.n_seqs, rows = (int64_t)a.n_nodes * a.n_heads, per = 256 / (EPL * 64);
    hipLaunchKernelGGL((k_tree_xscore<EPL, RT>), dim3((uint32_t)(one * p.w.nsplit)), dim3(256), 0, s, a, p.w, p.groups);
    hipLaunchKernelGGL((k_tree_xsum<EPL, RT>), dim3((uint32_t)(one * p.w.vsplit)), dim3(EPL * 128), 0, s, a, p.w, p.groups);
    hipLaunchKernelGGL(k_tree_xdiv<EPL * 64>, dim3((uint32_t)((rows + per - 1) / per)), dim3(256), 0, s, a, p.w);
}
template <int EPL> void tree_xgo(const sp_hipkv_tree_args &a, const XPlan &p, hipStream_t s) {
    if (p.rt == 1) tree_xgo<EPL, 1>(a, p, s);
    else if (EPL == 1 || p.rt == 2) tree_xgo<EPL, 2>(a, p, s);
    else if constexpr (EPL > 1) tree_xgo<EPL, 3>(a, p, s);
}
void tree_exact(const sp_hipkv_tree_args &a, hipStream_t s) {
    const XPlan p = tree_xplan(a);
    if (a.head_dim == 256) tree_xgo<4>(a, p, s);
    else if (a.head_dim == 128) tree_xgo<2>(a, p, s);
    else tree_xgo<1>(a, p, s);
}

}  // namespace

void launch_tree(const sp_hipkv_tree_args &a, hipStream_t s) {
    if (a.rows == SP_HIPKV_ROWS_EXACT) tree_exact(a, s);
    else if (a.rows == SP_HIPKV_ROWS_F32) tree_float<SP_HIPKV_ROWS_F32>(a, s);
    else tree_float<SP_HIPKV_ROWS_SPINOR>(a, s);
}

}  // namespace kvd

extern "C" int sp_hipkv_tree_attention_work(const sp_hipkv_tree_args *a, size_t *bytes) {
    using namespace kvd;
    const char *who = "sp_hipkv_tree_attention_work";
    if (tree_check(who, a)) return 1;
    OP_NEED(bytes, "null bytes");
    *bytes = 0;
    if (a->rows == SP_HIPKV_ROWS_EXACT) {
        sp_hipkv_tree_args b = *a;
        b.work = nullptr;
        const XPlan p = tree_xplan(b);
        OP_NEED((int64_t)a->n_kv_heads * p.groups * a->n_seqs * p.w.vsplit <= 1 << 22, "too many sequences, heads and nodes for one launch");
        *bytes = p.bytes;
        return 0;
    }
    const TreePlan p = tree_plan(*a);
    OP_NEED(tree_grid(*a, p) <= 1 << 23, "too many sequences, heads and nodes for one launch");
    if (p.nsplit > 1) *bytes = (size_t)a->n_nodes * a->n_heads * p.nsplit * (a->head_dim + 2) * 4;
    return 0;
}

extern "C" int sp_hipkv_tree_attention(const sp_hipkv_tree_args *a, void *stream) {
    using namespace kvd;
    const char *who = "sp_hipkv_tree_attention";
    if (tree_check(who, a)) return 1;
    if (!a->n_nodes) return 0;
    size_t need = 0;
    if (sp_hipkv_tree_attention_work(a, &need) || tree_check_arrays(who, a, need)) return 1;
    OpDevice dev((hipStream_t)stream);
    if (dev.err == hipSuccess) launch_tree(*a, (hipStream_t)stream);
    return op_done(who, dev);
}
