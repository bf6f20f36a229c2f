// kvd_tree.hip -- attention of drafted token trees over the paged cache.
//
// Row (node, q head) sees the cached positions from its window start on and the
// nodes whose bit is set in its mask; out = sum_p w_p v_p / sum_p w_p with
//   f32, Spinor rows   w_p = e^(s_p - M), s_p = scale q.k_p, M the row's largest;
//   exact rows         z_p = llround(f32(<qi, ki_p> / 2^32) scale 2^14), qi = rne(q 2^16),
//                      w_p = exp_fixed((z_p - M) 2^16) >> 8, out = RNE(sum w vq / (2^16 sum w)),
// the decode attention's integers (kvd_attn.hip).
//
// f32 and Spinor rows run in one pass over K and V (k_tree_float), on the bf16 matrix
// cores in exact pieces; exact rows on the int8 matrix cores in two passes (k_tree_xscore,
// _xsum).
#include "kvd_op.h"
#include "kvd_exact.h"
#include "kvd_vec.h"
#include "kvd_pass.h"
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
// whether some sequence has the node, for this thread's share t, t + n, .. of the sequences
__device__ __forceinline__ bool tree_has(const sp_hipkv_tree_args &a, int node, int t, int n) {
    bool has = false;
    for (int s = t; s < a.n_seqs; s += n) {
        const TreeSeq q = tree_seq(a, s);
        has |= node >= q.node0 && node - q.node0 < q.nodes;
    }
    return has;
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
// Its waves take the tiles of a range of pages (a split) in turn, each with all RT row
// tiles, a running maximum, sum and output of its own; they meet in LDS at the end, the
// splits in k_tree_merge.  K and V are read once for all nodes and q heads of a workgroup.
//
// Scores are made transposed, S^T = K Q^T (K the A operand, Q the B operand, from LDS): a
// lane then holds a row's scores of the positions that O += P V needs from it as its A
// operand, so weights stay in registers between the two products.
//
// f32 rows (8 waves, 32 positions a tile).  The f32 matrix cores bound the first form of
// this kernel: 16x16x4 takes 32 cycles, 154 TF, 223 us of the 322 that 64 nodes of 16
// heads at 32k took (8 kv heads of 256 dims).  A product of two f32 as six products
// of bf16 pieces (below) costs 2.7 times fewer cycles and errs by 2^-26 of it, less than
// f32 accumulation does: 229 us.  What bounds it now is a sum, as variants with one part
// taken out showed: forming the pieces (3 roundings and 2 subtractions for each element) a third, the
// matrix products a third, the wait for memory and for the slowest wave the rest; in a
// wave they hardly overlap, and the registers (O: 16 RT x HD f32 a wave) allow 2 waves
// a SIMD.  Memory comes through LDS by direct loads: held in registers on
// the way, a tile cost 64 more of them (250 us).
//
// Spinor rows (4 waves, 32 positions a tile): a code is a bf16 number as it is, so three
// products with q's or the weights' pieces are exact, and a chunk's multiplier (one number for a
// position) joins outside the product: on the scores of the chunk's dims, and on the weights
// before they are taken apart.  Dims and columns are therefore dealt to steps and tiles by
// chunk, as windows of 64 dims of which 51 (43, 32) count.  16 nodes at 6k of 16 heads (8 kv
// heads of 256 dims) take 26.4 us; as f32 products of codes times multipliers, which was the first form,
// 36.5, and 30 nodes of 32 heads at 12k 50 for 82 us.  The codes' conversion bounds it now, 1.5
// instructions a code, and below 20 us what is fixed.
//
// The running maximum only moves when a score exceeds it by 2^8 in the exponent (base
// 2): weights stay below 2^8 and nothing is lost, and a tile needs one ballot instead of
// a reduction over lanes.  The sums are joined over lanes once at the end.
//
// A position that a row does not see has weight 0, which a V value whose pieces are not
// finite would turn into NaN: tiles that some row does not see whole look for such values
// first and are then put off to a loop behind the main one, which adds positions one
// by one (inside the main loop that path costs twice the output's registers).
typedef float v4f __attribute__((ext_vector_type(4)));
constexpr float LOG2E_F = 1.44269504088896341f;
constexpr int TREE_PAGES = 256;              // pages of a split at most
constexpr int tree_waves(int rows) { return rows == SP_HIPKV_ROWS_SPINOR ? 4 : 8; }

__device__ __forceinline__ bool finite1(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
// whether bf16 pieces hold x: not infinities, NaN, nor the magnitudes above the midpoint of the
// largest bf16 number and the next power of two, which round up to an infinite first piece
constexpr uint32_t PIECES_END = 0x7F7F8000u;
__device__ __forceinline__ bool pieces_hold(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) < PIECES_END; }

// Of an f32 its three bf16 pieces, which sum to it exactly: x = h + m + l, |m| <= 2^-9 |x|,
// |l| <= 2^-18 |x| (magnitudes from PIECES_END on round up to infinity and make NaN, with a weight of 0
// too; below 2^-110 l is lost to denormals bit by bit).  Cutting bits off instead of rounding saves 4% of a call, and
// 2^-21 of a product would be missing for 2^-26.
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));
typedef uint32_t v2u32 __attribute__((ext_vector_type(2), aligned(4)));
struct Pieces { bf8 p[3]; };
template <typename X> __device__ __forceinline__ Pieces pieces_of(X &&x) {                 // of x(0) .. x(7)
    v4u32 w[3];
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        float a = x(2 * k), b = x(2 * k + 1);
        #pragma unroll
        for (int n = 0; n < 3; n++) {
            const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, bf2));
            w[n][k] = u;
            if (n < 2) { a -= __uint_as_float(u << 16); b -= __uint_as_float(u & 0xFFFF0000u); }
        }
    }
    return {{__builtin_bit_cast(bf8, w[0]), __builtin_bit_cast(bf8, w[1]), __builtin_bit_cast(bf8, w[2])}};
}
// The products of a's pieces with b's that make up a b to 2^-26, smallest first
__device__ constexpr int MUL_A[6] = {2, 1, 0, 1, 0, 0}, MUL_B[6] = {0, 1, 2, 0, 1, 0};
__device__ __forceinline__ v4f mfma_piece(const Pieces &a, const Pieces &b, int n, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[MUL_A[n]], b.p[MUL_B[n]], c, 0, 0, 0);
}

// The first dword of a window of `win` bytes of a Spinor row that holds chunk b's codes and ends inside the row
__device__ constexpr int spn_window(int hd, int b, int win) {
    const int d = spn_block_start(hd, b) / 4, most = (row_bytes_of(SP_HIPKV_ROWS_SPINOR, hd) - win) / 4;
    return d < most ? d : most;
}

template <int ROWS, int EPL, int RT>
__global__ __launch_bounds__(64 * tree_waves(ROWS), 2) void k_tree_float(sp_hipkv_tree_args a, int groups, int nsplit, int pages) {
    constexpr int HD = EPL * 64, RB = row_bytes_of(ROWS, HD);
    constexpr bool SPN = ROWS == SP_HIPKV_ROWS_SPINOR;
    constexpr int TP = 32;                                                 // positions a wave takes at a time
    constexpr int NW = tree_waves(ROWS), NT = 64 * NW;
    // Spinor: a chunk's dims as a window of WIN from a multiple of 4 on; its columns as four tiles
    constexpr int NB = SPN ? spn_blocks(HD) : 0, WIN = HD == 64 ? 32 : 64, QD = SPN ? NB * WIN : HD;
    constexpr int CPR = SPN ? 4 * NB : HD / 16;                            // column tiles
    // q, [piece][row][dim] bf16, and the waves' rings or multipliers; then the waves' outputs
    constexpr int Q_B = RT * 16 * QD * 6, UNIT = SPN ? 2048 : 4096, OUT_B = NW * 16 * HD * 4;
    constexpr int RING = SPN ? 1 : 152 * 1024 - Q_B >= 4 * NW * UNIT ? 4 : 3;
    constexpr int LDS_B = Q_B + NW * RING * UNIT > OUT_B ? Q_B + NW * RING * UNIT : OUT_B;
    __shared__ __align__(1024) uint8_t lds[LDS_B];
    __shared__ float s_m[NW][RT * 16], s_l[NW][RT * 16], s_M[RT * 16], s_L[RT * 16];
    __shared__ int s_node[RT * 16], s_low[RT * 16];
    __shared__ const uint8_t *s_page[TREE_PAGES];                         // this split's
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
    // each row's node and where it starts to see (rows past the last repeat it)
    int lo_min = INT32_MAX, lo_max = 0;
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        const int r = r0 + t * 16 + l16, node = (r < R ? r : R - 1) / G, lo = tree_low(a, q, node);
        lo_min = min(lo_min, lo); lo_max = max(lo_max, lo);
        if (threadIdx.x < 16) { s_node[t * 16 + l16] = q.node0 + node; s_low[t * 16 + l16] = lo; }
    }
    if (a.window) {
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1) { lo_min = min(lo_min, __shfl_xor(lo_min, o, 64)); lo_max = max(lo_max, __shfl_xor(lo_max, o, 64)); }
    }
    lo_min = __builtin_amdgcn_readfirstlane(lo_min); lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    // this split's tiles with a position that is seen, and this wave's: w0, w0 + NW, .. below w1
    // (a sequence shorter than the longest has proportionally fewer parts)
    const int pg0 = lo_min / PAGE, np = (end + PAGE - 1) / PAGE - pg0;
    const int parts = max((int)(((int64_t)np * nsplit + pages - 1) / pages), (np + TREE_PAGES - 1) / TREE_PAGES);
    const int b0 = pg0 + (int)((int64_t)np * min(split, parts) / parts), b1 = pg0 + (int)((int64_t)np * min(split + 1, parts) / parts);
    const int t0 = max(b0 * (PAGE / TP), lo_min / TP), w1 = min(b1 * (PAGE / TP), (end + TP - 1) / TP), w0 = t0 + wave;
    float *po = (float *)a.work, *pml = po + (size_t)a.n_nodes * a.n_heads * nsplit * HD;
    if (nsplit > 1 && t0 >= w1) {                                          // nothing here (splits past this sequence's parts)
        const int r = r0 + threadIdx.x;
        if (threadIdx.x < RT * 16 && r < R)
            *(v2f *)(pml + 2 * (((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * nsplit + split)) = (v2f){-INFINITY, 0.0f};
        return;
    }
    auto row_q = [&](int r) {
        const int rr = r0 + r < R ? r0 + r : R - 1;
        return a.q + (size_t)(q.node0 + rr / G) * a.q_stride + (size_t)(h * G + rr % G) * HD;
    };
    // 16-byte pieces of a row in an order that spreads a column over the banks
    for (int i = threadIdx.x; i < b1 - b0 && i < TREE_PAGES; i += NT) s_page[i] = tree_page(a, q, (b0 + i) * PAGE);
    for (int i = threadIdx.x; i < RT * 16 * (QD / 8); i += NT) {
        const int r = i / (QD / 8), c = i % (QD / 8);
        Pieces p;
        if constexpr (SPN) {                                               // zeros beside the chunk's dims
            const int b = c / (WIN / 8), d0 = 4 * spn_window(HD, b, WIN) + 8 * (c % (WIN / 8));
            const int lo = spn_block_start(HD, b) - d0, hi = spn_block_start(HD, b + 1) - d0;
            const float *x = row_q(r) + d0;
            const v4f zero = {0, 0, 0, 0}, y0 = d0 < HD ? *(const v4f *)x : zero, y1 = d0 + 4 < HD ? *(const v4f *)(x + 4) : zero;
            p = pieces_of([&](int k) { return k >= lo && k < hi ? (k < 4 ? y0[k & 3] : y1[k & 3]) : 0.0f; });
        } else {
            const v4f x = *(const v4f *)(row_q(r) + 8 * c), y = *(const v4f *)(row_q(r) + 8 * c + 4);
            p = pieces_of([&](int k) { return k < 4 ? x[k] : y[k - 4]; });
        }
        #pragma unroll
        for (int n = 0; n < 3; n++) ((bf8 *)lds)[(n * RT * 16 + r) * (QD / 8) + (c ^ (r & (WIN == 32 && SPN ? 3 : 7)))] = p.p[n];
    }
    v4f O[RT][CPR], S[RT][2];
    float m[RT], l[RT];
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        m[t] = -INFINITY; l[t] = 0.0f;
        #pragma unroll
        for (int c = 0; c < CPR; c++) O[t][c] = (v4f){0, 0, 0, 0};
    }
    __syncthreads();
    const uint32_t kslice = (uint32_t)h * PAGE * RB, vslice = (uint32_t)(a.n_kv_heads + h) * PAGE * RB;
    // page addresses are the wave's: rows load as address + 32-bit lane offset
    auto page_at = [&](int tile) { return uniform(s_page[tile / (PAGE / TP) - b0]); };
    // tiles that some row does not see whole, and those of them with a V value that
    // pieces do not hold: nodes span at most 10 pages, so do the rows' window starts
    auto ragged = [&](int tile) { return tile * TP < lo_max || tile * TP + TP > q.cached; };
    const int tail = q.cached / TP, head = lo_min / TP;
    uint64_t later = 0;
    auto put_off = [&](int tile) { later |= tile >= tail ? 1ull << (tile - tail) : 1ull << (32 + tile - head); };
    // whether this lane's row of tile t sees positions p0 + 4 g + i, as bits
    auto seen4 = [&](int t, int p0) {
        uint32_t see = 0;
        const int lo = s_low[t * 16 + l16];
        const uint64_t *mask = a.visible + (size_t)s_node[t * 16 + l16] * a.mask_words;
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = p0 + 4 * g + i, j = p - q.cached;
            bool v = p >= lo;
            if (j >= 0) v = j < q.nodes && (gmem(mask)[j >> 6] >> (j & 63) & 1);
            see |= (uint32_t)v << i;
        }
        return see;
    };
    // scores in base 2, masked; weights into S
    auto softmax = [&](int tile, bool rag) {
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            float mx = -INFINITY;
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                #pragma unroll
                for (int i = 0; i < 4; i++) S[t][u][i] *= a.scale * LOG2E_F;
                if (rag) {
                    const uint32_t see = seen4(t, tile * TP + 16 * u);
                    #pragma unroll
                    for (int i = 0; i < 4; i++) S[t][u][i] = see >> i & 1 ? S[t][u][i] : -INFINITY;
                }
                #pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, S[t][u][i]);
            }
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
            for (int u = 0; u < 2; u++)
                #pragma unroll
                for (int i = 0; i < 4; i++) { S[t][u][i] = __builtin_amdgcn_exp2f(S[t][u][i] - ms); l[t] += S[t][u][i]; }
        }
    };
    // V values that pieces do not hold, as infinities and NaN for the rows that see them; x4(page, row offset, k): columns 4 k .. of this lane
    auto add_later = [&](auto &&x4) {
        while (later) {
            const int b = __builtin_ctzll(later), tile = b < 32 ? tail + b : head + b - 32;
            later &= later - 1;
            const uint8_t *pg = page_at(tile);
            for (int p = tile * TP; p < tile * TP + TP && p < end; p++) {
                #pragma unroll
                for (int t = 0; t < RT; t++) {
                    bool on[4];
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int k = t * 16 + 4 * g + i, j = p - q.cached;
                        on[i] = j < 0 ? p >= s_low[k] : (gmem(a.visible)[(size_t)s_node[k] * a.mask_words + (j >> 6)] >> (j & 63) & 1);
                    }
                    #pragma unroll
                    for (int k = 0; k < CPR / 4; k++) {
                        const v4f v = x4(pg + vslice + (uint32_t)(p & (PAGE - 1)) * RB, k);
                        #pragma unroll
                        for (int c = 0; c < 4; c++)
                            #pragma unroll
                            for (int i = 0; i < 4; i++) O[t][4 * k + c][i] += on[i] && !pieces_hold(v[c]) ? v[c] * INFINITY : 0.0f;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    auto zero_s = [&] {
        #pragma unroll
        for (int t = 0; t < RT; t++)
            #pragma unroll
            for (int u = 0; u < 2; u++) S[t][u] = (v4f){0, 0, 0, 0};
    };
    if constexpr (!SPN) {
        // A tile's memory comes in units of 32 rows x 128 bytes, straight into a ring of the
        // wave's own in LDS (no registers, no barrier: the wave waits for its own loads):
        // K steps of 32 dims, then V as 32 columns.  16-byte piece c of a row lies at place
        // c ^ (slot % 8) of its slot; rows are in order for K, by (row % 4, row / 4) for V,
        // which is how the operands' reads meet no bank twice.
        constexpr int NK = HD / 32, NU = 2 * NK;
        const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)(lds + Q_B + wave * RING * UNIT);
        const uint8_t *ringp = lds + Q_B + wave * RING * UNIT;
        const int rj = lane >> 3, vo_k = rj * RB + ((lane & 7) ^ rj) * 16, vo_v = (16 * (rj >> 2) + 4 * (rj & 3)) * RB + ((lane & 7) ^ rj) * 16;
        auto load = [&](const uint8_t *pg, int tile, int n, uint32_t slot) {
            const int row = tile * TP & (PAGE - 1);
            const bool v = n >= NK;
            const v4i rs = rsrc_of(pg + (v ? vslice : kslice) + row * RB + (n - (v ? NK : 0)) * 128, (TP - 1) * RB + 128);
            #pragma unroll
            for (int k = 0; k < 4; k++) dma16(ring + slot * UNIT + k * 1024, v ? vo_v : vo_k, rs, (v ? k : 8 * k) * RB);
        };
        int kb[2];
        #pragma unroll
        for (int e = 0; e < 2; e++) kb[e] = l16 * (HD / 8) + ((4 * e + g) ^ (l16 & 7));
        const bf8 *qs = (const bf8 *)lds;
        // this lane's places in a unit: K piece 2 g (and ^ 1) of row l16 (+ 16), V columns 2 l16, + 1 of row 4 g + e (slot 8 e + g)
        const int kp = l16 * 128 + ((2 * g) ^ (l16 & 7)) * 16;
        int vp[2];
        #pragma unroll
        for (int u = 0; u < 2; u++) vp[u] = (4 * u + g) * 128 + (((l16 >> 1) ^ (4 * u + g)) * 16) + 8 * (l16 & 1);
        // Unit n is read from the ring into x while unit n - 1 is multiplied, q's pieces while
        // the operand's are formed.
        uint32_t slot = 0;                                                 // of the unit after the one in x
        float x[16];
        auto arrive = [&] { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * (RING - 1)) : "memory"); };
        auto read = [&](int n) {
            const uint8_t *un = ringp + slot * UNIT;
            if (n < NK) {
                #pragma unroll
                for (int u = 0; u < 2; u++) {
                    *(v4f *)(x + 8 * u) = *(const v4f *)(un + kp + 2048 * u);
                    *(v4f *)(x + 8 * u + 4) = *(const v4f *)(un + (kp ^ 16) + 2048 * u);
                }
            } else {
                #pragma unroll
                for (int k = 0; k < 8; k++) *(v2f *)(x + 2 * k) = *(const v2f *)(un + vp[k >> 2] + 1024 * (k & 3));
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        const uint8_t *pg = nullptr, *pn = nullptr;
        if (w0 < w1) {
            pg = page_at(w0);
            #pragma unroll
            for (int n = 0; n < RING; n++) load(pg, w0, n, n);
            arrive();
            read(0);
        }
        for (int tile = w0; tile < w1; tile += NW) {
            const int nx = tile + NW < w1 ? tile + NW : tile;
            const bool rag = ragged(tile);
            pn = page_at(nx);
            // x is read: unit n's slot takes the unit RING later
            auto refill = [&](int n) {
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
                if (n + RING < NU) load(pg, tile, n + RING, slot); else load(pn, nx, n + RING - NU, slot);
                slot = slot == RING - 1 ? 0 : slot + 1;
            };
            zero_s();
            #pragma unroll
            for (int n = 0; n < NK; n++) {
                Pieces K[2], Q[2];
                auto load_q = [&](int t) {
                    #pragma unroll
                    for (int k = 0; k < 3; k++) Q[t & 1].p[k] = qs[kb[n & 1] + (k * RT + t) * 2 * HD + 8 * (n >> 1)];
                    __builtin_amdgcn_sched_barrier(0);
                };
                load_q(0);
                #pragma unroll
                for (int u = 0; u < 2; u++) K[u] = pieces_of([&](int k) { return x[8 * u + k]; });
                refill(n);
                #pragma unroll
                for (int t = 0; t < RT; t++) {
                    if (t + 1 < RT) load_q(t + 1);
                    #pragma unroll
                    for (int k = 0; k < 6; k++)
                        #pragma unroll
                        for (int u = 0; u < 2; u++) S[t][u] = mfma_piece(K[u], Q[t & 1], k, S[t][u]);
                    if (t == 0) { arrive(); read(n + 1); }
                }
            }
            softmax(tile, rag);
            Pieces P[RT];
            #pragma unroll
            for (int t = 0; t < RT; t++) P[t] = pieces_of([&](int k) { return S[t][k >> 2][k & 3]; });
            uint32_t bad = 0;                                              // largest magnitude of a row before the end
            #pragma unroll
            for (int n = NK; n < NU; n++) {
                if (rag) {
                    #pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const uint32_t f = __float_as_uint(x[k]) & 0x7FFFFFFFu;
                        bad = max(bad, tile * TP + 16 * (k >> 3) + 4 * g + (k >> 1 & 3) < end ? f : 0u);
                        x[k] = f >= PIECES_END ? 0.0f : x[k];
                        if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
                }
                Pieces V[2];
                #pragma unroll
                for (int c = 0; c < 2; c++) V[c] = pieces_of([&](int k) { return x[2 * k + c]; });
                refill(n);
                #pragma unroll
                for (int t = 0; t < RT; t++) {
                    #pragma unroll
                    for (int k = 0; k < 6; k++)
                        #pragma unroll
                        for (int c = 0; c < 2; c++) O[t][2 * (n - NK) + c] = mfma_piece(P[t], V[c], k, O[t][2 * (n - NK) + c]);
                    if (t == 0) { arrive(); read(n + 1 < NU ? n + 1 : 0); }
                }
            }
            if (__any(bad >= PIECES_END)) put_off(tile);
            pg = pn;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");                 // nothing lands in LDS after this
        add_later([&](const uint8_t *row, int k) {
            const v2f x = *gmem((const v2f *)(row + 8 * l16 + 256 * k)), y = *gmem((const v2f *)(row + 8 * l16 + 256 * k + 128));
            return (v4f){x[0], x[1], y[0], y[1]};
        });
    } else {
        // Codes are bf16 numbers as they are.  A chunk's multiplier is one number for a position:
        // scores of a chunk's dims are multiplied by it when they are summed, and for a chunk's
        // columns the weights are, before their pieces are taken.  Multipliers go through
        // LDS, [K, V][chunk][position], from the rows' lanes to those of the scores.
        constexpr int KD = WIN / 16;                                       // dwords of a lane in a window
        float (*mul)[8][32] = (float (*)[8][32])(lds + Q_B + wave * UNIT);
        const bf8 *qs = (const bf8 *)lds;
        struct Row { uint32_t c[KD]; };
        Row K[NB][2];
        uint32_t V[NB][8];
        v4f km, vm;
        // positions past the last one repeat it
        auto row_off = [&](int tile, int x) { const int p = tile * TP + x; return (uint32_t)((p < end ? p : end - 1) & (PAGE - 1)) * RB; };
        const int part = NB > 4 ? lane >> 5 : 0;                           // chunks 4 part .. of row lane % 32
        auto load_k = [&](const uint8_t *pg, int tile) {
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint8_t *row = pg + kslice + row_off(tile, 16 * u + l16) + 4 * KD * g;
                #pragma unroll
                for (int b = 0; b < NB; b++)
                    #pragma unroll
                    for (int d = 0; d < KD; d += 2) {
                        const v2u32 w = *gmem((const v2u32 *)(row + 4 * spn_window(HD, b, WIN) + 4 * d));
                        K[b][u].c[d] = w[0]; K[b][u].c[d + 1] = w[1];
                    }
            }
            km = *gmem((const v4f *)(pg + kslice + row_off(tile, lane & 31) + HD + 16 * part));
        };
        auto load_v = [&](const uint8_t *pg, int tile) {
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint8_t *row = pg + vslice + row_off(tile, 16 * (j >> 2) + 4 * g + (j & 3)) + 4 * l16;
                #pragma unroll
                for (int b = 0; b < NB; b++) V[b][j] = *gmem((const uint32_t *)(row + 4 * spn_window(HD, b, 64)));
            }
            vm = *gmem((const v4f *)(pg + vslice + row_off(tile, lane & 31) + HD + 16 * part));
        };
        auto put_mul = [&](int kv, v4f x) {
            #pragma unroll
            for (int i = 0; i < 4; i++) mul[kv][4 * part + i][lane & 31] = x[i];
            __builtin_amdgcn_wave_barrier();
        };
        auto code = [](uint32_t w, int t) { return (float)(int32_t)(int8_t)(w >> (8 * t)); };
        auto codes = [&](auto &&x) {                                       // of x(0) .. x(7), exactly
            v4u32 w;
            #pragma unroll
            for (int k = 0; k < 4; k++) w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){x(2 * k), x(2 * k + 1)}, bf2));
            return __builtin_bit_cast(bf8, w);
        };
        const uint8_t *pg = nullptr, *pn = nullptr;
        if (w0 < w1) {
            pg = page_at(w0);
            load_k(pg, w0);
            load_v(pg, w0);
        }
        for (int tile = w0; tile < w1; tile += NW) {
            const int nx = tile + NW < w1 ? tile + NW : tile;
            const bool rag = ragged(tile);
            pn = page_at(nx);
            zero_s();
            // infinities become NaN: scores of -infinity would count as positions that nobody sees
            #pragma unroll
            for (int i = 0; i < 4; i++) km[i] = fmaf(km[i], 0.0f, km[i]);
            put_mul(0, km);
            #pragma unroll
            for (int b = 0; b < NB; b++) {
                v4f C[RT][2];
                #pragma unroll
                for (int t = 0; t < RT; t++)
                    #pragma unroll
                    for (int u = 0; u < 2; u++) C[t][u] = (v4f){0, 0, 0, 0};
                #pragma unroll
                for (int ks = 0; ks < KD / 2; ks++) {
                    bf8 A[2];
                    #pragma unroll
                    for (int u = 0; u < 2; u++) A[u] = codes([&](int k) { return code(K[b][u].c[2 * ks + k / 4], k % 4); });
                    #pragma unroll
                    for (int t = 0; t < RT; t++) {
                        bf8 Q[3];
                        const int c = b * (WIN / 8) + KD / 2 * g + ks;
                        #pragma unroll
                        for (int n = 0; n < 3; n++) Q[n] = qs[(n * RT * 16 + t * 16 + l16) * (QD / 8) + (c ^ (l16 & (WIN == 32 ? 3 : 7)))];
                        #pragma unroll
                        for (int n = 2; n >= 0; n--)
                            #pragma unroll
                            for (int u = 0; u < 2; u++) C[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A[u], Q[n], C[t][u], 0, 0, 0);
                    }
                }
                #pragma unroll
                for (int u = 0; u < 2; u++) {
                    const v4f mk = *(const v4f *)&mul[0][b][16 * u + 4 * g];
                    #pragma unroll
                    for (int t = 0; t < RT; t++)
                        #pragma unroll
                        for (int i = 0; i < 4; i++) S[t][u][i] = fmaf(mk[i], C[t][u][i], S[t][u][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            load_k(pn, nx);
            __builtin_amdgcn_sched_barrier(0);
            softmax(tile, rag);
            if (rag) {
                bool bad = false;
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool f = finite1(127.0f * vm[i]) || 4 * part + i >= NB;
                    bad |= !f;
                    vm[i] = f ? vm[i] : 0.0f;
                }
                if (__any(bad)) put_off(tile);
            }
            put_mul(1, vm);
            #pragma unroll
            for (int b = 0; b < NB; b++) {
                const v4f m0 = *(const v4f *)&mul[1][b][4 * g], m1 = *(const v4f *)&mul[1][b][16 + 4 * g];
                Pieces P[RT];
                #pragma unroll
                for (int t = 0; t < RT; t++) P[t] = pieces_of([&](int k) { return S[t][k >> 2][k & 3] * (k < 4 ? m0[k & 3] : m1[k & 3]); });
                #pragma unroll
                for (int c = 0; c < 4; c++) {
                    const bf8 B = codes([&](int k) { return code(V[b][k], c); });
                    #pragma unroll
                    for (int t = 0; t < RT; t++)
                        #pragma unroll
                        for (int n = 2; n >= 0; n--) O[t][4 * b + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(P[t].p[n], B, O[t][4 * b + c], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            load_v(pn, nx);
            __builtin_amdgcn_sched_barrier(0);
            pg = pn;
        }
        add_later([&](const uint8_t *row, int b) {                         // multipliers that are not finite
            const float m = *gmem((const float *)(row + HD + 4 * b));
            return finite1(127.0f * m) ? (v4f){0, 0, 0, 0} : (v4f){NAN, NAN, NAN, NAN};
        });
    }
    // the waves' parts: m and l first, then the outputs, 16 rows at a time
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
        if (g == 0) { s_m[wave][t * 16 + l16] = m[t]; s_l[wave][t * 16 + l16] = l[t]; }
    }
    __syncthreads();                                                       // ... and nobody reads q any more
    if (threadIdx.x < RT * 16) {
        const int k = threadIdx.x;
        float M = -INFINITY, L = 0.0f, f[NW];
        #pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, s_m[w][k]);
        #pragma unroll
        for (int w = 0; w < NW; w++) {
            f[w] = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][k] - M);
            L += f[w] * s_l[w][k];
        }
        #pragma unroll
        for (int w = 0; w < NW; w++) s_m[w][k] = f[w];
        s_M[k] = M; s_L[k] = L;
    }
    __syncthreads();
    #pragma unroll
    for (int t = 0; t < RT; t++) {
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = s_m[wave][t * 16 + 4 * g + i];                 // 0 times NaN is NaN: what a row sees reaches it
            float *dst = (float *)lds + (wave * 16 + 4 * g + i) * HD;
            if constexpr (SPN) {                                           // tile 4 b + c: columns 4 (window + lane) + c of chunk b
                #pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int d0 = 4 * (spn_window(HD, b, 64) + l16);
                    #pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (d0 + c >= spn_block_start(HD, b) && d0 + c < spn_block_start(HD, b + 1)) dst[d0 + c] = O[t][4 * b + c][i] * f;
                }
            } else {
                #pragma unroll
                for (int c = 0; c < CPR; c += 2) {
                    const v2f x = {O[t][c][i], O[t][c + 1][i]};
                    ((v2f *)dst)[8 * c + l16] = x * f;
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 4 * HD; i += NT) {                   // 16 rows of HD / 4 pieces
            const int k = i / (HD / 4), c = i % (HD / 4), rl = t * 16 + k, r = r0 + rl;
            if (r >= R) continue;
            const v4f *src = (const v4f *)lds + i;
            v4f x = (src[0] + src[4 * HD]) + (src[8 * HD] + src[12 * HD]);
            if constexpr (NW == 8) x += (src[16 * HD] + src[20 * HD]) + (src[24 * HD] + src[28 * HD]);
            const float M = s_M[rl], L = s_L[rl];
            const int node = q.node0 + r / G, head = h * G + r % G;
            if (nsplit == 1) {
                *(v4f *)(a.out + (size_t)node * a.out_stride + (size_t)head * HD + 4 * c) = L == 0.0f ? (v4f){0, 0, 0, 0} : x / L;
            } else {
                const size_t at = ((size_t)node * a.n_heads + head) * nsplit + split;
                if (M > -INFINITY) *(v4f *)(po + at * HD + 4 * c) = x;
                if (c == 0) { pml[2 * at] = M; pml[2 * at + 1] = L; }
            }
        }
        if (t < RT - 1) __syncthreads();
    }
}

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c: a workgroup per row, HD / 4
// threads along it, the others share the (at most 64) parts.  Rows of no sequence stay
// as they were.
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(sp_hipkv_tree_args a, int nsplit) {
    constexpr int NG = 1024 / HD;
    __shared__ float s_f[64], s_L;
    __shared__ v4f s_x[256];
    const size_t row = blockIdx.x;
    const int c = threadIdx.x % (HD / 4), grp = threadIdx.x / (HD / 4);
    const float *ml = (const float *)a.work + (size_t)a.n_nodes * a.n_heads * nsplit * HD + 2 * row * nsplit;
    if (threadIdx.x < 64) {
        const bool in = (int)threadIdx.x < nsplit;
        const float m = in ? ml[2 * threadIdx.x] : -INFINITY, l = in ? ml[2 * threadIdx.x + 1] : 0.0f, M = wave_allmax(m);
        const bool none = m == -INFINITY;                                 // a part without a position of this row, or without a score
        const float f = none ? 0.0f : __builtin_amdgcn_exp2f(m - M);
        s_f[threadIdx.x] = none ? -1.0f : f;
        const float L = wave_allsum(f * l);                               // NaN scores: l is NaN also where m is -inf
        if (threadIdx.x == 0) s_L = L;
    }
    if (!__syncthreads_or(tree_has(a, (int)(row / a.n_heads), threadIdx.x, 256))) return;
    const v4f *po = (const v4f *)((const float *)a.work + row * nsplit * HD) + c;
    v4f x = {0, 0, 0, 0};
    #pragma unroll 4
    for (int k = grp; k < nsplit; k += NG) {
        const v4f v = po[(size_t)k * (HD / 4)];
        const float f = s_f[k];
        x += f < 0.0f ? (v4f){0, 0, 0, 0} : f * v;                        // ... whose output was not written
    }
    s_x[threadIdx.x] = x;
    __syncthreads();
    if (grp) return;
    #pragma unroll
    for (int k = 1; k < NG; k++) x += s_x[k * (HD / 4) + c];
    const float L = s_L;
    *(v4f *)(a.out + (row / a.n_heads) * a.out_stride + (row % a.n_heads) * HD + 4 * c) = L == 0.0f ? (v4f){0, 0, 0, 0} : x / L;
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
// Scores: a wave takes 16 positions straight into registers as the B operand (16 dims a
// lane and step, in an order that q's digits in LDS share), makes their digits once and
// multiplies them with all row tiles, up to 6 (96 rows), so that K is read and taken
// apart once for that many.  Tiles whose numbers, or whose q, need a fourth digit are put off to a
// loop behind: in the main one its registers spilled, which cost 30 us of 150.
// V sums: a wave owns 32 columns and takes a page a step: lane l 16 positions of two
// columns, which are the B operand after their digits are formed; no transposition.
// The weights' digits are made once for all waves and pass through LDS; half of the waves
// make the next page's before the products, half after.
//
// 48 nodes of 16 heads at 32k (8 kv heads of 256 dims): scores 100 us, sums 114, division
// 6; reading K and V once is 113 us, z (100 MB) written and read once some 42 more, and variants
// with one part taken out name none that would give more than 40 (memory's wait; the int8
// products, digits, weights and epilogues 10 each).  7 nodes at 4k: 10.5 + 11.2 + 3.9 us, where no
// part but the first loads (3 us) shows: launches and dependent loads.
//
// The V sums of head dim 64, and of 128 with two row tiles or more, are slower than their
// work: from four position pairs a thread on the compiler leaves `weights` a function, and
// what it takes by reference lies in scratch memory, 352 to 416 bytes a lane.  24 nodes of 32
// heads at 4k (8 kv heads of 128 dims) take 90 us, of 16 heads with 256 dims 49.
constexpr int DIG3 = 127 * (1 + 256 + 65536);                    // largest |x| of three balanced digits

// x = d0 + 2^8 d1 + 2^16 d2 + 2^24 d3, d in [-128, 127]; four values' digits, one dword per
// place.  w[3] == 0: three digits hold them all; a digit of -128 there: perhaps not even four.
__device__ __forceinline__ void digits_of(const int32_t x[4], uint32_t w[4]) {
    uint32_t d[4];
    #pragma unroll
    for (int e = 0; e < 4; e++) d[e] = ((uint32_t)x[e] + 0x80808080u) ^ 0x80808080u;
    const uint32_t ab0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), ab2 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
    const uint32_t cd0 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), cd2 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u); w[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u); w[3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}
__device__ __forceinline__ bool four_fail(uint32_t w3) { return (w3 & 0x80808080u & ~((w3 & 0x7F7F7F7Fu) + 0x7F7F7F7Fu)) != 0; }
// sum_k 2^(8 k) a[k]
template <int N> __device__ __forceinline__ int64_t places(const int32_t (&a)[N]) {
    static_assert(N == 5 || N == 7, "");
    int64_t s = (int64_t)a[1] * 256 + a[0];
    s += (int64_t)a[2] * 65536;
    s += (int64_t)a[3] * 16777216;
    int64_t hi = a[4];
    if constexpr (N == 7) hi += (int64_t)a[5] * 256 + (int64_t)a[6] * 65536;
    return s + (int64_t)((uint64_t)hi << 32);
}
// f32(ip / 2^32): one rounding to double, one to f32
__device__ __forceinline__ float ip_float(int64_t ip) {
    return (float)fma((double)(uint32_t)ip, 0x1p-32, (double)(int32_t)(ip >> 32));
}
// exp_fixed((z - M) 2^16) >> 8 for z <= M: 2^-g, g = ceil((M - z) log2(e) 2^30 / 2^14) in
// 30 bits; exp2_frac without a branch, each step one 32 x 32 + 64 bit product
__device__ __forceinline__ int32_t weight_of(int32_t z, int32_t M) {
    const uint64_t g = ((uint64_t)((uint32_t)M - (uint32_t)z) * (uint32_t)LOG2E + 16383) >> 14;
    const uint32_t n = (uint32_t)(g >> FB), r = (uint32_t)g & (uint32_t)(ONE - 1), f = (uint32_t)ONE - r;
    uint32_t e = (uint32_t)EXPC[6];
    #pragma unroll
    for (int k = 5; k >= 0; k--) {
        const uint64_t t = (uint64_t)e * f + ((uint64_t)EXPC[k] << FB);
        e = __builtin_amdgcn_alignbit((uint32_t)(t >> 32), (uint32_t)t, FB);
    }
    e = r ? e : 0x80000000u;
    return n < 23 ? (int32_t)(e >> ((n + 9) & 31)) : 0;
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
    __shared__ __align__(16) int8_t qd[3][RT * 16][QROW];          // q's digits [place][row][64 ks + 16 g + 4 quarter + e]
    __shared__ int s_level, s_mx[4][RT * 16];
    __shared__ __align__(16) int s_row[RT * 16];                   // node n_heads + head; past the last row again the last
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads;
    int id = blockIdx.x;
    const int h = id % a.n_kv_heads; id /= a.n_kv_heads;
    const int grp = id % groups; id /= groups;
    const int split = id % x.nsplit;
    const TreeSeq q = tree_seq(a, id / x.nsplit);
    const int R = q.nodes * G, r0 = grp * RT * 16;
    if (r0 >= R) return;
    const int end = q.cached + q.nodes, z0 = z_first(a, q);
    const Span sp = rows_span(a, q, G, r0, min(r0 + RT * 16, R));
    const int per = (sp.pg1 - sp.pg0 + x.nsplit - 1) / x.nsplit;
    int w0 = sp.pg0 + split * per, w1 = min(w0 + per, sp.pg1);
    if (w0 < w1 && w0 * PAGE + wave * 16 + 16 <= sp.lo_min) w0++;
    if (w0 < w1 && (w1 - 1) * PAGE + wave * 16 >= end) w1--;
    const uint32_t kslice = (uint32_t)h * PAGE * HD * 4;
    auto page = [&](int lp) { return uniform(tree_page(a, q, lp * PAGE)); };
    // positions past the last one repeat it
    auto row_at = [&](int lp) {
        const int p = lp * PAGE + wave * 16 + l16;
        return kslice + (uint32_t)((p < end ? p : end - 1) & (PAGE - 1)) * (HD * 4) + 16 * g;
    };
    auto load_k = [&](v4i (&k)[4 * KS], const uint8_t *pg, int lp) {
        const uint32_t off = row_at(lp);
        #pragma unroll
        for (int s = 0; s < 4 * KS; s++) k[s] = *gmem((const v4i *)(pg + off + 64 * s));
    };
    auto row_q = [&](int r) {
        const int rr = r0 + r < R ? r0 + r : R - 1;
        return a.q + (size_t)(q.node0 + rr / G) * a.q_stride + (size_t)(h * G + rr % G) * HD;
    };
    auto grid_of = [](float4 f, int32_t (&v)[4]) {
        v[0] = (int32_t)rintf(f.x * 65536.0f); v[1] = (int32_t)rintf(f.y * 65536.0f);
        v[2] = (int32_t)rintf(f.z * 65536.0f); v[3] = (int32_t)rintf(f.w * 65536.0f);
    };
    v4i K[4 * KS];
    const uint8_t *pn = nullptr;
    if (w0 < w1) {                                                         // K first: q's digits are made while it comes
        load_k(K, page(w0), w0);
        pn = page(min(w0 + 1, w1 - 1));
    }
    if (threadIdx.x == 0) s_level = 0;
    if (threadIdx.x < RT * 16) {
        const int r = min(r0 + (int)threadIdx.x, R - 1);
        s_row[threadIdx.x] = (q.node0 + r / G) * a.n_heads + h * G + r % G;
    }
    __syncthreads();
    uint32_t over = 0;
    #pragma unroll 4
    for (int i = threadIdx.x; i < RT * 16 * (HD / 4); i += 256) {
        const int r = i / (HD / 4), c = i % (HD / 4);
        int32_t v[4];
        uint32_t w[4];
        grid_of(*(const float4 *)(row_q(r) + 4 * c), v);
        digits_of(v, w);
        over |= w[3];
        // dims 64 ks + 16 quarter + 4 g + e
        const int at = (c / 16) * 64 + (c % 4) * 16 + (c / 4 % 4) * 4;
        #pragma unroll
        for (int b = 0; b < 3; b++) *(uint32_t *)&qd[b][r][at] = w[b];
    }
    if (__any(over != 0) && lane == 0) atomicOr(&s_level, 1);
    int mx[RT][4];                                                         // of rows 4 g + i of each tile
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int i = 0; i < 4; i++) mx[t][i] = INT32_MIN;
    __syncthreads();
    const bool qbig = s_level != 0;
    const float zscale = a.scale * 16384.0f;
    // scores into z and the maxima
    auto finish = [&](int lp, int t, int rowg, const int64_t (&ip)[4]) {
        const int p0 = lp * PAGE + wave * 16, p = p0 + l16;
        const int4 rows = *(const int4 *)&s_row[t * 16 + rowg];
        const int row[4] = {rows.x, rows.y, rows.z, rows.w};
        int32_t z[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) z[i] = (int32_t)round_away(ip_float(ip[i]) * zscale);   // scale 2^14 is exact: the same product
        if (p0 >= sp.lo_max && p0 + 16 <= q.cached) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                x.z[(size_t)row[i] * x.zstride + (p - z0)] = z[i];
                mx[t][i] = max(mx[t][i], z[i]);
            }
        } else if (p < end) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                x.z[(size_t)row[i] * x.zstride + (p - z0)] = z[i];
                mx[t][i] = row_sees(a, q, row[i] / a.n_heads - q.node0, p) ? max(mx[t][i], z[i]) : mx[t][i];
            }
        }
    };
    bool later = qbig;
    for (int lp = qbig ? w1 : w0; lp < w1; lp++) {
        v4i B[3][KS];
        uint32_t over = 0;
        #pragma unroll
        for (int s = 0; s < 4 * KS; s++) {
            const int32_t v[4] = {K[s][0], K[s][1], K[s][2], K[s][3]};
            uint32_t w[4];
            digits_of(v, w);
            over |= w[3];
            #pragma unroll
            for (int b = 0; b < 3; b++) B[b][s / 4][s % 4] = (int)w[b];
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(K, pn, min(lp + 1, w1 - 1));
        pn = page(min(lp + 2, w1 - 1));
        __builtin_amdgcn_sched_barrier(0);
        if (__any(over != 0)) { later = true; continue; }
        int rowg = 4 * g;
        asm volatile("" : "+v"(rowg));                                     // rows' numbers read where used, not kept
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            v4i acc[5];
            #pragma unroll
            for (int k = 0; k < 5; k++) acc[k] = (v4i){0, 0, 0, 0};
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                v4i A[3];
                #pragma unroll
                for (int b = 0; b < 3; b++) A[b] = *(const v4i *)&qd[b][t * 16 + l16][64 * ks + 16 * g];
                #pragma unroll
                for (int u = 0; u < 3; u++)
                    #pragma unroll
                    for (int b = 0; b < 3; b++) acc[u + b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[u], B[b][ks], acc[u + b], 0, 0, 0);
            }
            int64_t ip[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int32_t c[5] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i], acc[4][i]};
                ip[i] = places(c);
            }
            finish(lp, t, rowg, ip);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // tiles put off, with four digits, q and K read again
    for (int lp = later ? w0 : w1; lp < w1; lp++) {
        const uint8_t *kr = page(lp) + row_at(lp);
        uint32_t over = qbig ? 1 : 0;
        for (int s = 0; s < 4 * KS; s++) {
            const v4i k = *gmem((const v4i *)(kr + 64 * s));
            const int32_t v[4] = {k[0], k[1], k[2], k[3]};
            uint32_t w[4];
            digits_of(v, w);
            over |= w[3];
        }
        if (!__any(over != 0)) continue;
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            v4i acc[7];
            bool fail = false;
            #pragma unroll
            for (int k = 0; k < 7; k++) acc[k] = (v4i){0, 0, 0, 0};
            const float *qr = row_q(t * 16 + l16) + 4 * g;
            #pragma unroll 1
            for (int ks = 0; ks < KS; ks++) {
                v4i A[4], C[4];
                #pragma unroll
                for (int s = 0; s < 4; s++) {
                    int32_t v[4];
                    uint32_t w[4];
                    grid_of(*(const float4 *)(qr + 64 * ks + 16 * s), v);
                    digits_of(v, w);
                    fail |= four_fail(w[3]);
                    #pragma unroll
                    for (int b = 0; b < 4; b++) A[b][s] = (int)w[b];
                    const v4i k = *gmem((const v4i *)(kr + 256 * ks + 64 * s));
                    const int32_t vk[4] = {k[0], k[1], k[2], k[3]};
                    digits_of(vk, w);
                    fail |= four_fail(w[3]);
                    #pragma unroll
                    for (int b = 0; b < 4; b++) C[b][s] = (int)w[b];
                }
                #pragma unroll
                for (int u = 0; u < 4; u++)
                    #pragma unroll
                    for (int b = 0; b < 4; b++) acc[u + b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[u], C[b], acc[u + b], 0, 0, 0);
            }
            int64_t ip[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int32_t c[7] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i], acc[4][i], acc[5][i], acc[6][i]};
                ip[i] = places(c);
            }
            if (__any(fail)) {                                             // more than four: from the numbers
                const int32_t *kn = (const int32_t *)(kr - 16 * g);
                for (int i = 0; i < 4; i++) {
                    const float *qn = row_q(t * 16 + 4 * g + i);
                    int64_t s = 0;
                    for (int d = 0; d < HD; d++) s += (int64_t)(int32_t)rintf(qn[d] * 65536.0f) * gmem(kn)[d];
                    ip[i] = s;
                }
            }
            finish(lp, t, 4 * g, ip);
        }
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
    if (threadIdx.x < RT * 16) {
        const int k = threadIdx.x;
        x.zmax[(size_t)s_row[k] * x.nsplit + split] = max(max(s_mx[0][k], s_mx[1][k]), max(s_mx[2][k], s_mx[3][k]));
    }
}

// waves: HD / 32; one page a step
template <int EPL, int RT>
__global__ __launch_bounds__(EPL * 128, 2) void k_tree_xsum(sp_hipkv_tree_args a, XWork x, int groups) {
    constexpr int HD = EPL * 64, NT = EPL * 128, ROWS = RT * 16, WROW = PAGE + 16;
    constexpr int PAIRS = ROWS * 32 / NT, RSTEP = NT / 32;                     // position pairs of a thread and step, rows apart
    __shared__ __align__(16) int8_t wd[2][3][ROWS][WROW];                      // weights' digits [step parity][place][row][position]
    __shared__ int s_M[ROWS], s_row[ROWS];
    __shared__ const uint8_t *s_page[TREE_PAGES];                              // this split's (at most 2^14 positions)
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
    const uint32_t vslice = (uint32_t)(a.n_kv_heads + h) * PAGE * HD * 4;
    typedef int v2i __attribute__((ext_vector_type(2)));
    v2i V[16];
    auto page = [&](int lp) { return uniform(s_page[lp - b0]); };
    // lane: positions 16 g + j of columns 32 wave + 2 l16, + 1
    const uint32_t vo = (16 * g * HD + 32 * wave + 2 * l16) * 4;
    auto load_v = [&](const uint8_t *pg) {
        #pragma unroll
        for (int j = 0; j < 16; j++) V[j] = *gmem((const v2i *)(pg + vslice + j * (HD * 4) + vo));
    };
    for (int i = threadIdx.x; i < b1 - b0; i += NT) s_page[i] = tree_page(a, q, (b0 + i) * PAGE);
    if (b0 < b1) load_v(uniform(tree_page(a, q, b0 * PAGE)));
    // rows' maxima, 8 threads a row; rows without a position or past the last: no row, the least number
    for (int k = threadIdx.x / 8; k < ROWS; k += NT / 8) {
        int M = INT32_MIN;
        const int r = r0 + k, row = (q.node0 + r / G) * a.n_heads + h * G + r % G;
        if (r < R)
            for (int c = threadIdx.x & 7; c < x.nsplit; c += 8) M = max(M, x.zmax[(size_t)row * x.nsplit + c]);
        #pragma unroll
        for (int o = 1; o < 8; o <<= 1) M = max(M, __shfl_xor(M, o, 64));
        s_M[k] = M;
        s_row[k] = r < R && M > INT32_MIN ? row : -1;
    }
    __syncthreads();
    // this thread's weights: positions 2 (tid % 32), + 1 of rows tid / 32 + k RSTEP
    const int pair = threadIdx.x & 31;
    int64_t den[PAIRS];
    int2 z[PAIRS];
    #pragma unroll
    for (int k = 0; k < PAIRS; k++) { den[k] = 0; z[k] = make_int2(0, 0); }
    auto load_z = [&](int lp) {
        #pragma unroll
        for (int k = 0; k < PAIRS; k++) {
            const int row = s_row[threadIdx.x / 32 + k * RSTEP];
            if (row >= 0) z[k] = *(const int2 *)(x.z + (size_t)row * x.zstride + (lp * PAGE - z0 + 2 * pair));
        }
    };
    auto weights = [&](int lp, int par) {
        const int p0 = lp * PAGE;
        const bool whole = p0 >= sp.lo_max && p0 + PAGE <= q.cached;
        #pragma unroll
        for (int k = 0; k < PAIRS; k++) {
            int rl = threadIdx.x / 32 + k * RSTEP;
            asm volatile("" : "+v"(rl));                                   // what follows from it is made here, not kept
            const int M = s_M[rl];
            int32_t w[2] = {weight_of(z[k].x, M), weight_of(z[k].y, M)};   // (of no row: z = 0 below the least M)
            if (!whole) {
                const int node = min(r0 + rl, R - 1) / G;
                #pragma unroll
                for (int e = 0; e < 2; e++) w[e] = row_sees(a, q, node, p0 + 2 * pair + e) ? w[e] : 0;
            }
            den[k] += (int64_t)w[0] + w[1];
            const uint32_t d0 = ((uint32_t)w[0] + 0x808080u) ^ 0x808080u, d1 = ((uint32_t)w[1] + 0x808080u) ^ 0x808080u;
            const uint32_t lo = __builtin_amdgcn_perm(d1, d0, 0x05010400u), hi = __builtin_amdgcn_perm(d1, d0, 0x0C0C0602u);
            *(uint16_t *)&wd[par][0][rl][2 * pair] = (uint16_t)lo;
            *(uint16_t *)&wd[par][1][rl][2 * pair] = (uint16_t)(lo >> 16);
            *(uint16_t *)&wd[par][2][rl][2 * pair] = (uint16_t)hi;
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    v4i acc[RT][2][5];
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int c = 0; c < 2; c++)
            #pragma unroll
            for (int k = 0; k < 5; k++) acc[t][c][k] = (v4i){0, 0, 0, 0};
    // Two waves share a SIMD: half of the waves make their weights of the next page before
    // the products, half after, so that the vector and the matrix units both have work.
    const bool first = wave < NT / 128;
    if (b0 < b1) {
        load_z(b0);
        weights(b0, 0);
        load_z(min(b0 + 1, b1 - 1));
    }
    for (int lp = b0; lp < b1; lp++) {
        const int par = (lp - b0) & 1, nx = min(lp + 1, b1 - 1);
        const uint8_t *pn = page(nx);
        auto next_weights = [&] {
            if (lp + 1 < b1) {
                weights(lp + 1, par ^ 1);
                load_z(min(lp + 2, b1 - 1));
            }
        };
        __syncthreads();                                                   // this page's weights are there, the last one's are read
        if (first) next_weights();
        if (lp * PAGE + PAGE > end) {                                      // places behind the last position
            #pragma unroll
            for (int j = 0; j < 16; j++)
                if (lp * PAGE + 16 * g + j >= end) V[j] = (v2i){0, 0};
        }
        // |v| may exceed three digits by little: what is left goes through once more
        for (bool more = true; more;) {
            v4i B[2][3];
            uint32_t over = 0;
            #pragma unroll
            for (int c = 0; c < 2; c++)
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int32_t v[4] = {V[4 * j][c], V[4 * j + 1][c], V[4 * j + 2][c], V[4 * j + 3][c]};
                    uint32_t d[4];
                    digits_of(v, d);
                    over |= d[3];
                    #pragma unroll
                    for (int b = 0; b < 3; b++) B[c][b][j] = (int)d[b];
                }
            more = __any(over != 0);
            if (more) {
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
            }
            if (!more) {
                __builtin_amdgcn_sched_barrier(0);
                load_v(pn);
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
        if (!first) next_weights();
    }
    // denominators: over a row's 32 threads
    #pragma unroll
    for (int k = 0; k < PAIRS; k++) {
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) den[k] += __shfl_xor(den[k], o, 64);
        const int r = r0 + threadIdx.x / 32 + k * RSTEP;
        if (pair == 0 && r < R) x.den[((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * x.vsplit + split] = den[k];
    }
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + t * 16 + 4 * g + i;
            int64_t s[2];
            #pragma unroll
            for (int c = 0; c < 2; c++) {
                const int32_t k[5] = {acc[t][c][0][i], acc[t][c][1][i], acc[t][c][2][i], acc[t][c][3][i], acc[t][c][4][i]};
                s[c] = places(k);
            }
            if (r < R) {
                int64_t *dst = x.sum + (((size_t)(q.node0 + r / G) * a.n_heads + h * G + r % G) * x.vsplit + split) * HD + 32 * wave + 2 * l16;
                dst[0] = s[0]; dst[1] = s[1];
            }
        }
}

// a workgroup per row, its parts shared by NG groups of threads
template <int HD>
__global__ __launch_bounds__(512) void k_tree_xdiv(sp_hipkv_tree_args a, XWork x) {
    constexpr int NG = 512 / HD;
    __shared__ int64_t s_t[512], s_d[NG];
    const size_t row = blockIdx.x;
    const int d = threadIdx.x % HD, grp = threadIdx.x / HD;
    const int64_t *s = x.sum + row * x.vsplit * HD + d, *dn = x.den + row * x.vsplit;
    int64_t t = 0, den = 0;
    #pragma unroll 8
    for (int k = grp; k < x.vsplit; k += NG) { t += s[(size_t)k * HD]; den += dn[k]; }
    s_t[threadIdx.x] = t;
    if (d == 0) s_d[grp] = den;
    // a row of no sequence stays as it was
    if (!__syncthreads_or(tree_has(a, (int)(row / a.n_heads), threadIdx.x, 512)) || grp) return;
    #pragma unroll
    for (int k = 1; k < NG; k++) { t += s_t[k * HD + d]; den += s_d[k]; }
    a.out[(row / a.n_heads) * a.out_stride + (row % a.n_heads) * HD + d] = den > 0 ? rne_div_to_float((i128)t, den, 16) : 0.0f;
}

// How a launch is cut: row tiles of a workgroup (rt), workgroups along a sequence's rows
// (groups), parts of its positions (nsplit): whatever the least time is estimated for.
//   f32: a round of tiles, one a wave, 1.1 us for each row tile and 64 dims, and one more
//   (0.6 of it where one wave of a SIMD has a tile); a workgroup 4.5 us and 1.5 for each row
//   tile (set-up, q, joining its waves).
//   Spinor: a round 0.7 us, and for each 128 dims 0.45 and 0.9 for each row tile (1.7 times it
//   where two workgroups share a unit); a workgroup 4 us for each row tile and 1 for each 32
//   dims.  Several sequences are taken to be 0.6 of the longest (8 of 300 to 4000: 39 us for 55;
//   for f32's one workgroup a unit that misleads: 16 sessions 112 us for 99).
//   The groups read K and V again from L2: 25 TB/s.  Joining parts: 4 us.
// From stamps of workgroups, and sweeps of both numbers.  Against one fixed choice (most row
// tiles, 256 workgroups): one node at 100 12.2 -> 9.0 us (one part for two), 8 nodes at 600
// 15.5 -> 12.4 (two groups for one), 24 nodes at 4k 28.5 -> 25.9 (8 parts for 16).
struct TreePlan { int rt, groups, nsplit, pages; };
TreePlan tree_plan(const sp_hipkv_tree_args &a) {
    TreePlan p{};
    const bool spn = a.rows == SP_HIPKV_ROWS_SPINOR;
    // row tiles whose outputs a wave's registers hold (with one more they spill, and loads from scratch wait behind
    // the prefetched tiles: 10 us a page for 3)
    const int most = (a.head_dim == 256 ? 2 : a.head_dim == 128 ? 3 : 4) - (spn ? 1 : 0);
    const int tiles = std::max(1, (a.max_nodes * (a.n_heads / a.n_kv_heads) + 15) / 16);
    const int64_t span = a.window ? std::min<int64_t>(a.max_positions, (int64_t)a.window + a.max_nodes + PAGE) : a.max_positions;
    p.pages = (int)std::max<int64_t>(1, (span + PAGE - 1) / PAGE);
    const int waves = tree_waves(a.rows);
    const double seqs = (double)a.n_kv_heads * (spn && a.n_seqs > 1 ? 0.6 * a.n_seqs : std::max(a.n_seqs, 1));
    const double mb = seqs * p.pages * PAGE * 2 * row_bytes_of(a.rows, a.head_dim) * 1e-6;
    double best = 0;
    for (int m = most; m >= 1; m--) {
        const int groups = (tiles + m - 1) / m, rt = (tiles + groups - 1) / groups;
        if (rt < m) continue;                                                                   // the same as a smaller m
        const double round = spn ? 0.7 + a.head_dim / 128.0 * (0.45 + 0.9 * rt) : 1.0 + 1.1 * rt * (a.head_dim / 64);
        for (int n = (p.pages + TREE_PAGES - 1) / TREE_PAGES; n <= 64 && n <= p.pages; n++) {
            const int t = (PAGE / 32 * p.pages + n - 1) / n, lots = (int)std::ceil(seqs * groups * n / 256);   // tiles of a workgroup; workgroups of a unit
            const int rounds = (t + waves - 1) / waves;
            double us = 0.04 * mb * groups + (n > 1 ? 4.0 + 0.05 * n : 0.0);
            if (spn) us += (lots + 1) / 2 * (a.head_dim / 32 + 4.0 * rt) + round * rounds * (lots / 2 * 1.7 + lots % 2);
            else us += lots * (4.5 + 1.5 * rt + round * (rounds - ((t - 1) % waves < waves / 2 ? 0.4 : 0.0)));
            if (!p.nsplit || us < best) { best = us; p.nsplit = n; p.rt = rt; p.groups = groups; }
        }
    }
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
    OP_NEED((int64_t)a->n_nodes * a->n_heads <= 1 << 22, "more than 2^22 rows (n_nodes x n_heads)");
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

template <int ROWS> hipError_t tree_float(const sp_hipkv_tree_args &a, hipStream_t s) {
    const TreePlan p = tree_plan(a);
    const dim3 grid((uint32_t)tree_grid(a, p)), wg(256);
    hipError_t e = hipSuccess;
#define TREE_RUN(EPL, RT) e = op_launch(k_tree_float<ROWS, EPL, RT>, grid, dim3(64 * tree_waves(ROWS)), s, a, p.groups, p.nsplit, p.pages)
    if (a.head_dim == 256) {
        if constexpr (ROWS == SP_HIPKV_ROWS_F32) { if (p.rt == 2) TREE_RUN(4, 2); else TREE_RUN(4, 1); }
        else TREE_RUN(4, 1);
    } else if (a.head_dim == 128) { if (p.rt == 1) TREE_RUN(2, 1); else if (p.rt == 2) TREE_RUN(2, 2); else if constexpr (ROWS == SP_HIPKV_ROWS_F32) TREE_RUN(2, 3); }
    else { if (p.rt == 1) TREE_RUN(1, 1); else if (p.rt == 2) TREE_RUN(1, 2); else if (p.rt == 3) TREE_RUN(1, 3); else if constexpr (ROWS == SP_HIPKV_ROWS_F32) TREE_RUN(1, 4); }
#undef TREE_RUN
    if (e != hipSuccess || p.nsplit == 1) return e;
    const dim3 mg((uint32_t)((int64_t)a.n_nodes * a.n_heads));
    return op_launch(a.head_dim == 256 ? k_tree_merge<256> : a.head_dim == 128 ? k_tree_merge<128> : k_tree_merge<64>, mg, wg, s, a, p.nsplit);
}

// Exact rows: a workgroup's row tiles for the scores, whose q digits two workgroups' LDS
// holds, and for the sums, whose registers hold their accumulators; splits for 512
// workgroups, for as many as can run at once.  A V split's int32 sums hold
// 2 x 3 x 2^14 a position (values that need a second round of digits), so at most 2^14 positions.
struct XPlan { int rt, groups, srt, sgroups; XWork w; size_t bytes; };
XPlan tree_xplan(const sp_hipkv_tree_args &a) {
    XPlan p{};
    const int tiles = std::max(1, (a.max_nodes * (a.n_heads / a.n_kv_heads) + 15) / 16);
    const int most = a.head_dim == 64 ? 2 : 3;
    p.groups = (tiles + most - 1) / most;
    p.rt = (tiles + p.groups - 1) / p.groups;
    p.sgroups = (tiles + 5) / 6;
    p.srt = (tiles + p.sgroups - 1) / p.sgroups;
    const int span = a.window ? (int)std::min<int64_t>(a.max_positions, (int64_t)a.window + a.max_nodes + PAGE) : a.max_positions;
    const int64_t base = (int64_t)a.n_kv_heads * std::max(a.n_seqs, 1), pages = std::max(1, (span + PAGE - 1) / PAGE + 1);
    auto splits = [&](int64_t wgs, int64_t each) { return (int)std::max<int64_t>(1, std::min<int64_t>({(wgs + each - 1) / each, (pages + 1) / 2, 64})); };
    p.w.zstride = (int)pages * PAGE;
    p.w.nsplit = splits(512, base * p.sgroups);
    p.w.vsplit = std::max((int)((pages * PAGE + 16383) >> 14), splits(65536 / a.head_dim, base * p.groups));
    const size_t rows = (size_t)a.n_nodes * a.n_heads;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    const size_t zb = up(rows * p.w.zstride * 4), mb = up(rows * p.w.nsplit * 4), sb = rows * p.w.vsplit * a.head_dim * 8;
    uint8_t *at = (uint8_t *)a.work;
    p.w.z = (int32_t *)at; p.w.zmax = (int32_t *)(at + zb); p.w.sum = (int64_t *)(at + zb + mb); p.w.den = (int64_t *)(at + zb + mb + sb);
    p.bytes = zb + mb + sb + up(rows * p.w.vsplit * 8);
    return p;
}
template <int EPL> hipError_t tree_xgo(const sp_hipkv_tree_args &a, const XPlan &p, hipStream_t s) {
    const int64_t base = (int64_t)a.n_kv_heads * a.n_seqs;
    hipError_t e = hipSuccess;
#define TREE_SCORE(RT) e = op_launch(k_tree_xscore<EPL, RT>, dim3((uint32_t)(base * p.sgroups * p.w.nsplit)), dim3(256), s, a, p.w, p.sgroups)
#define TREE_SUM(RT) e = op_launch(k_tree_xsum<EPL, RT>, dim3((uint32_t)(base * p.groups * p.w.vsplit)), dim3(EPL * 128), s, a, p.w, p.groups)
    if (p.srt == 1) TREE_SCORE(1); else if (p.srt == 2) TREE_SCORE(2); else if (p.srt == 3) TREE_SCORE(3); else if (p.srt == 4) TREE_SCORE(4); else TREE_SCORE(6);
    if (e != hipSuccess) return e;
    if (p.rt == 1) TREE_SUM(1);
    else if (EPL == 1 || p.rt == 2) TREE_SUM(2);
    else if constexpr (EPL > 1) TREE_SUM(3);
    if (e != hipSuccess) return e;
    return op_launch(k_tree_xdiv<EPL * 64>, dim3((uint32_t)((int64_t)a.n_nodes * a.n_heads)), dim3(512), s, a, p.w);
#undef TREE_SCORE
#undef TREE_SUM
}
hipError_t tree_exact(const sp_hipkv_tree_args &a, hipStream_t s) {
    const XPlan p = tree_xplan(a);
    return a.head_dim == 256 ? tree_xgo<4>(a, p, s) : a.head_dim == 128 ? tree_xgo<2>(a, p, s) : tree_xgo<1>(a, p, s);
}

}  // namespace

hipError_t launch_tree(const sp_hipkv_tree_args &a, hipStream_t s) {
    if (a.rows == SP_HIPKV_ROWS_EXACT) return tree_exact(a, s);
    return a.rows == SP_HIPKV_ROWS_F32 ? tree_float<SP_HIPKV_ROWS_F32>(a, s) : tree_float<SP_HIPKV_ROWS_SPINOR>(a, s);
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
        OP_NEED((int64_t)a->n_kv_heads * a->n_seqs * std::max(p.groups * p.w.vsplit, p.sgroups * p.w.nsplit) <= 1 << 22, "too many sequences, heads and nodes for one launch");
        *bytes = p.bytes;
        return 0;
    }
    const TreePlan p = tree_plan(*a);
    OP_NEED(tree_grid(*a, p) <= 1 << 22, "too many sequences, heads and nodes for one launch");
    if (p.nsplit > 1) *bytes = (size_t)a->n_nodes * a->n_heads * p.nsplit * (a->head_dim + 2) * 4;
    return 0;
}

extern "C" int sp_hipkv_tree_attention_plan(const sp_hipkv_tree_args *a, int32_t plan[4]) {
    using namespace kvd;
    const char *who = "sp_hipkv_tree_attention_plan";
    if (tree_check(who, a)) return 1;
    OP_NEED(plan, "null plan");
    if (a->rows == SP_HIPKV_ROWS_EXACT) {
        sp_hipkv_tree_args b = *a;
        b.work = nullptr;
        const XPlan p = tree_xplan(b);
        plan[0] = p.srt; plan[1] = p.w.nsplit; plan[2] = p.rt; plan[3] = p.w.vsplit;
    } else {
        const TreePlan p = tree_plan(*a);
        plan[0] = p.rt; plan[1] = p.nsplit; plan[2] = plan[3] = 0;
    }
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
    return op_done(who, dev.err != hipSuccess ? dev.err : launch_tree(*a, (hipStream_t)stream));
}
