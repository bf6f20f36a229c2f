// kvd_tree.hip -- attention of drafted token trees over the paged cache.
//
// Row (node, q head) sees the cached positions from its window start on and the
// nodes whose bit is set in its mask; out = sum_p w_p v_p / sum_p w_p with
//   f32, Spinor rows   w_p = e^(s_p - M), s_p = scale q.k_p, M the row's largest;
//   exact rows         z_p = llround(f32(<qi, ki_p> / 2^32) scale 2^14), qi = rne(q 2^16),
//                      w_p = exp_fixed((z_p - M) 2^16) >> 8, out = RNE(sum w vq / (2^16 sum w)),
// the decode attention's integers (kvd_attn.hip).
//
// One workgroup per row: its four waves take the positions in turn, each with a
// running maximum and sum, and meet in LDS.
#include "kvd_op.h"
#include "kvd_exact.h"
#include "kvd_vec.h"

namespace kvd {

namespace {

constexpr int TREE_WAVES = 4;

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
    const int64_t lo = (int64_t)q.cached + a.depth[q.node0 + node] - a.window + 1;
    return lo < 0 ? 0 : lo > q.cached ? q.cached : (int)lo;
}
__device__ __forceinline__ const uint8_t *tree_page(const sp_hipkv_tree_args &a, const TreeSeq &q, int pos) {
    const int lp = pos / PAGE;
    return (const uint8_t *)gmem(q.table)[a.ring_pages ? lp % a.ring_pages : lp];
}

template <int ROWS, int EPL>
__global__ __launch_bounds__(64 * TREE_WAVES) void k_tree_row(sp_hipkv_tree_args a) {
    constexpr int HD = EPL * 64, RB = row_bytes_of(ROWS, HD);
    const int head = blockIdx.x, node = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const TreeSeq q = tree_seq(a, blockIdx.z);
    if (node >= q.nodes) return;
    const int h = head / (a.n_heads / a.n_kv_heads), low = tree_low(a, q, node);
    const uint64_t *mask = a.visible + (size_t)(q.node0 + node) * a.mask_words;
    const float *qp = a.q + (size_t)(q.node0 + node) * a.q_stride + head * HD;
    float qf[EPL];
    int64_t qi[EPL];
    #pragma unroll
    for (int e = 0; e < EPL; e++) { qf[e] = qp[lane + 64 * e]; qi[e] = (int64_t)rintf(qf[e] * 65536.0f); }
    auto row_of = [&](int p, int v) { return tree_page(a, q, p) + ((size_t)(v * a.n_kv_heads + h) * PAGE + (p & (PAGE - 1))) * RB; };
    auto value = [&](const uint8_t *row, int e) {
        const int d = lane + 64 * e;
        if constexpr (ROWS == SP_HIPKV_ROWS_SPINOR) return (float)((const int8_t *)row)[d] * ((const float *)(row + HD))[spn_block_of(HD, d)];
        else return ((const float *)row)[d];
    };
    auto sees = [&](int p) { return p < q.cached ? p >= low : (mask[(p - q.cached) >> 6] >> ((p - q.cached) & 63) & 1) != 0; };
    auto grid_score = [&](int p) {                       // exact rows
        const int32_t *k = (const int32_t *)row_of(p, 0);
        int64_t ip = 0;
        #pragma unroll
        for (int e = 0; e < EPL; e++) ip += qi[e] * k[lane + 64 * e];
        return (int)llround_pow2<14>((float)((double)wave_allsum(ip) / 4294967296.0) * a.scale);
    };
    __shared__ float sm[TREE_WAVES], sl[TREE_WAVES], so[TREE_WAVES][HD];
    __shared__ int zm[TREE_WAVES];
    __shared__ int64_t sw[TREE_WAVES], sv[TREE_WAVES][HD];
    const int end = q.cached + q.nodes;
    float *out = a.out + (size_t)(q.node0 + node) * a.out_stride + head * HD;
    if constexpr (ROWS == SP_HIPKV_ROWS_EXACT) {
        int M = INT32_MIN;
        for (int p = low + wave; p < end; p += TREE_WAVES)
            if (sees(p)) M = max(M, grid_score(p));
        if (lane == 0) zm[wave] = M;
        __syncthreads();
        for (int w = 0; w < TREE_WAVES; w++) M = max(M, zm[w]);
        int64_t S = 0, o[EPL] = {};
        for (int p = low + wave; p < end; p += TREE_WAVES)
            if (sees(p)) {
                const int64_t w = exp_fixed((((int64_t)grid_score(p) - M) * ONE) >> 14) >> 8;
                const int32_t *v = (const int32_t *)row_of(p, 1);
                S += w;
                #pragma unroll
                for (int e = 0; e < EPL; e++) o[e] += w * v[lane + 64 * e];
            }
        if (lane == 0) sw[wave] = S;
        #pragma unroll
        for (int e = 0; e < EPL; e++) sv[wave][lane + 64 * e] = o[e];
        __syncthreads();
        for (int d = threadIdx.x; d < HD; d += 64 * TREE_WAVES) {
            int64_t t = 0, den = 0;
            for (int w = 0; w < TREE_WAVES; w++) { t += sv[w][d]; den += sw[w]; }
            out[d] = den ? rne_div_to_float((i128)t, den, 16) : 0.0f;
        }
    } else {
        float m = -INFINITY, l = 0.0f, o[EPL] = {};
        for (int p = low + wave; p < end; p += TREE_WAVES)
            if (sees(p)) {
                float s = 0.0f;
                const uint8_t *k = row_of(p, 0), *v = row_of(p, 1);
                #pragma unroll
                for (int e = 0; e < EPL; e++) s += qf[e] * value(k, e);
                s = wave_allsum(s) * a.scale;
                const float mn = fmaxf(m, s), al = mn == -INFINITY ? 0.0f : expf(m - mn), w = mn == -INFINITY ? 0.0f : expf(s - mn);
                l = l * al + w;
                #pragma unroll
                for (int e = 0; e < EPL; e++) o[e] = o[e] * al + w * value(v, e);
                m = mn;
            }
        if (lane == 0) { sm[wave] = m; sl[wave] = l; }
        #pragma unroll
        for (int e = 0; e < EPL; e++) so[wave][lane + 64 * e] = o[e];
        __syncthreads();
        float M = -INFINITY;
        for (int w = 0; w < TREE_WAVES; w++) M = fmaxf(M, sm[w]);
        for (int d = threadIdx.x; d < HD; d += 64 * TREE_WAVES) {
            float t = 0.0f, den = 0.0f;
            for (int w = 0; w < TREE_WAVES; w++) {
                if (sm[w] == -INFINITY) continue;
                const float f = expf(sm[w] - M);
                t += f * so[w][d]; den += f * sl[w];
            }
            out[d] = den > 0.0f ? t / den : 0.0f;
        }
    }
}

int tree_check(const char *who, const sp_hipkv_tree_args *a) {
    OP_NEED(a, "null arguments");
    OP_NEED(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256, "head_dim is not 64, 128 or 256");
    OP_NEED(a->n_kv_heads > 0 && a->n_heads > 0 && a->n_heads % a->n_kv_heads == 0 && a->n_heads / a->n_kv_heads <= 16 && a->n_heads <= 65535,
            "n_heads is not n_kv_heads times 1 to 16");
    OP_NEED(a->rows == SP_HIPKV_ROWS_F32 || a->rows == SP_HIPKV_ROWS_EXACT || a->rows == SP_HIPKV_ROWS_SPINOR, "unknown row format");
    OP_NEED(a->n_seqs >= 0 && a->n_seqs <= 65535, "n_seqs outside [0, 65535]");
    OP_NEED(a->n_nodes >= 0, "negative n_nodes");
    OP_NEED(a->max_nodes >= 0 && a->max_nodes <= 512, "max_nodes outside [0, 512]");
    OP_NEED(a->max_positions >= 0 && a->max_positions <= (a->rows == SP_HIPKV_ROWS_EXACT ? 1 << 18 : 1 << 20),
            "max_positions outside [0, 2^20] (exact rows: 2^18)");
    OP_NEED(a->n_nodes <= (int64_t)a->n_seqs * a->max_nodes, "n_nodes is more than n_seqs times max_nodes");
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

template <int ROWS> void tree_go(const sp_hipkv_tree_args &a, hipStream_t s) {
    const dim3 grid(a.n_heads, a.max_nodes, a.n_seqs);
    if (a.head_dim == 256) hipLaunchKernelGGL((k_tree_row<ROWS, 4>), grid, dim3(64 * TREE_WAVES), 0, s, a);
    else if (a.head_dim == 128) hipLaunchKernelGGL((k_tree_row<ROWS, 2>), grid, dim3(64 * TREE_WAVES), 0, s, a);
    else hipLaunchKernelGGL((k_tree_row<ROWS, 1>), grid, dim3(64 * TREE_WAVES), 0, s, a);
}

}  // namespace

void launch_tree(const sp_hipkv_tree_args &a, hipStream_t s) {
    if (a.rows == SP_HIPKV_ROWS_F32) tree_go<SP_HIPKV_ROWS_F32>(a, s);
    else if (a.rows == SP_HIPKV_ROWS_EXACT) tree_go<SP_HIPKV_ROWS_EXACT>(a, s);
    else tree_go<SP_HIPKV_ROWS_SPINOR>(a, s);
}

}  // namespace kvd

extern "C" int sp_hipkv_tree_attention_work(const sp_hipkv_tree_args *a, size_t *bytes) {
    using namespace kvd;
    const char *who = "sp_hipkv_tree_attention_work";
    if (tree_check(who, a)) return 1;
    OP_NEED(bytes, "null bytes");
    *bytes = 0;
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
