// kvd_keep.hip -- keeping the accepted nodes of drafted token trees: rows
// cached + keep[i] -> cached + i of K and V, in place.
//
// The moves of one (table, K or V, kv head) overlap: the place of a later row
// may hold an earlier one's source.  A thread owns 16 bytes of every row of such a
// slice and takes the list in order, 8 rows at a time, all loads before the
// stores; since keep ascends, keep[i] >= i, and a row is read before or with the
// batch that writes over it.  Threads share nothing, so there is no barrier.
//
// The floor is the rows' bytes, read and written.  The rest is dependent loads (lists, page
// address, row), row after row: the compiler keeps the 8 rows of a batch in scratch memory
// (144 bytes a lane), and a row has arrived before it is stored there and the next one's
// load goes out.  A workgroup takes 256 pieces of a table's slices, so that rows below
// 1 KiB leave no lanes empty: 16 sequences of 36 layers, 8 kv heads of 128 f32, 4 rows each
// take 11.1 us (14.5 with one slice a workgroup of 64), a copy of as much 8.
#include "kvd_op.h"

namespace kvd {

namespace {

constexpr int KEEP_BATCH = 8;

__device__ __forceinline__ uint8_t *keep_row(const sp_hipkv_keep_args &a, const void *const *table, int ring, int pos, size_t slice) {
    const int lp = pos / PAGE;
    return (uint8_t *)gmem(table)[ring ? lp % ring : lp] + (slice * PAGE + (pos & (PAGE - 1))) * (size_t)a.row_bytes;
}

// grid (pieces of all slices / 256, 1, tables)
__global__ __launch_bounds__(256) void k_keep(sp_hipkv_keep_args a) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, pieces = (uint32_t)a.row_bytes / 16;
    const uint32_t slice = id / pieces, piece = id - slice * pieces;
    if (slice >= 2 * (uint32_t)a.n_kv_heads) return;
    for (int t = blockIdx.z; t < a.n_tables; t += gridDim.z) {
        const int s = a.seq ? a.seq[t] : t % a.n_seqs;
        if (s < 0 || s >= a.n_seqs) continue;
        const int k0 = a.keep_start[s], n = min(a.keep_start[s + 1] - k0, a.max_keep), base = a.cached[s];
        const int ring = a.ring_pages ? a.ring_pages[t] : 0;
        if (base < 0 || base >= a.max_positions) continue;
        const void *const *table = a.tables[t];
        int last = -1;
        for (int i0 = 0; i0 < n; i0 += KEEP_BATCH) {
            uint4 x[KEEP_BATCH];
            bool ok[KEEP_BATCH];
            #pragma unroll
            for (int u = 0; u < KEEP_BATCH; u++) {
                const int i = i0 + u, k = i < n ? a.keep[k0 + i] : -1;
                ok[u] = k > last && k >= i && k < a.max_positions - base;
                if (ok[u]) {
                    last = k;
                    ok[u] = k != i;
                    if (ok[u]) x[u] = gmem((const uint4 *)keep_row(a, table, ring, base + k, slice))[piece];
                }
            }
            #pragma unroll
            for (int u = 0; u < KEEP_BATCH; u++)
                if (ok[u]) gmem((uint4 *)keep_row(a, table, ring, base + i0 + u, slice))[piece] = x[u];
        }
    }
}

int keep_check(const sp_hipkv_keep_args *a) {
    const char *who = "sp_hipkv_keep_rows";
    OP_NEED(a, "null arguments");
    OP_NEED(a->n_kv_heads > 0 && a->n_kv_heads <= 32767, "n_kv_heads outside [1, 32767]");
    OP_NEED(a->row_bytes > 0 && a->row_bytes % 16 == 0 && a->row_bytes <= 65536, "row_bytes is not a multiple of 16 in [16, 65536]");
    OP_NEED(a->n_tables >= 0 && a->n_seqs >= 0 && (a->n_seqs > 0 || a->n_tables == 0), "negative n_tables or n_seqs, or tables without a sequence");
    OP_NEED(a->max_keep >= 0 && a->max_keep <= 512, "max_keep outside [0, 512]");
    OP_NEED(a->max_positions >= 0, "negative max_positions");
    OP_NEED(a->n_tables == 0 || a->max_keep == 0 || (a->tables && a->cached && a->keep_start && a->keep), "null array");
    return 0;
}

}  // namespace

hipError_t launch_keep(const sp_hipkv_keep_args &a, hipStream_t s) {
    const int64_t threads = (int64_t)(a.row_bytes / 16) * 2 * a.n_kv_heads;
    const dim3 grid((uint32_t)((threads + 255) / 256), 1, a.n_tables < 65535 ? a.n_tables : 65535);
    return op_launch(k_keep, grid, dim3(256), s, a);
}

}  // namespace kvd

extern "C" int sp_hipkv_keep_rows(const sp_hipkv_keep_args *a, void *stream) {
    using namespace kvd;
    if (keep_check(a)) return 1;
    if (!a->n_tables || !a->max_keep) return 0;
    OpDevice dev((hipStream_t)stream);
    return op_done("sp_hipkv_keep_rows", dev.err != hipSuccess ? dev.err : launch_keep(*a, (hipStream_t)stream));
}
