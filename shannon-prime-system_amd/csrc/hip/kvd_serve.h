// kvd_serve.h -- what the operators of serving from a paged cache (include/sp_hipkv.h:
// append, prompt attention, cache attention) share: value types, a call's sequences,
// the layout of 8-bit pages, checks.
#pragma once
#include "kvd_op.h"

namespace kvd {

constexpr int BLOCK8 = 16, PAGE_BLOCKS = PAGE / BLOCK8;                // positions with one scale; scales of a page's head
__host__ __device__ constexpr size_t block8_bytes(int nkv, int hd) { return (size_t)nkv * 2 * (PAGE * hd + PAGE_BLOCKS * 4); }

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------- values
struct Bf16 { uint16_t u; };
// N neighbouring values as f32, from an address aligned to as many
template <int N> __device__ __forceinline__ void load_values(const float *p, float (&x)[N]) {
    if constexpr (N == 2) { const v2f a = *gmem((const v2f *)p); x[0] = a[0]; x[1] = a[1]; }
    else {
        #pragma unroll
        for (int k = 0; k < N; k += 4) {
            const v4f a = *gmem((const v4f *)(p + k));
            #pragma unroll
            for (int j = 0; j < 4; j++) x[k + j] = a[j];
        }
    }
}
template <int N> __device__ __forceinline__ void load_values(const Bf16 *p, float (&x)[N]) {
    uint32_t w[N / 2];
    if constexpr (N == 2) w[0] = *gmem((const uint32_t *)p);
    else if constexpr (N == 4) { const v2u a = *gmem((const v2u *)p); w[0] = a[0]; w[1] = a[1]; }
    else {
        #pragma unroll
        for (int k = 0; k < N / 2; k += 4) {
            const v4u a = *gmem((const v4u *)(p + 2 * k));
            #pragma unroll
            for (int j = 0; j < 4; j++) w[k + j] = a[j];
        }
    }
    #pragma unroll
    for (int k = 0; k < N / 2; k++) { x[2 * k] = __uint_as_float(w[k] << 16); x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u); }
}
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, bf2));
}
template <int N> __device__ __forceinline__ void store_values(float *p, const float (&x)[N]) {
    if constexpr (N == 2) *gmem((v2f *)p) = (v2f){x[0], x[1]};
    else {
        #pragma unroll
        for (int k = 0; k < N; k += 4) *gmem((v4f *)(p + k)) = (v4f){x[k], x[k + 1], x[k + 2], x[k + 3]};
    }
}
template <int N> __device__ __forceinline__ void store_values(Bf16 *p, const float (&x)[N]) {
    if constexpr (N == 2) *gmem((uint32_t *)p) = bf16x2(x[0], x[1]);
    else if constexpr (N == 4) *gmem((v2u *)p) = (v2u){bf16x2(x[0], x[1]), bf16x2(x[2], x[3])};
    else {
        #pragma unroll
        for (int k = 0; k < N; k += 8)
            *gmem((v4u *)(p + k)) = (v4u){bf16x2(x[k], x[k + 1]), bf16x2(x[k + 2], x[k + 3]), bf16x2(x[k + 4], x[k + 5]), bf16x2(x[k + 6], x[k + 7])};
    }
}

// ---------------------------------------------------------------- sequences
// The work of a packed batch is cut into units of UNIT (tokens, rows) that start anew with
// each sequence.  Without a list of units, sequence s gets those from
// floor(mul start[s] / UNIT) + spare s on: a sequence with n of them has at most floor(n / UNIT) +
// spare where spare covers its cut ends, so ranges do not overlap, and `spare` units a sequence stay empty.
__device__ __forceinline__ int64_t unit_base(int start, int s, int mul, int unit, int spare) {
    return (int64_t)start * mul / unit + (int64_t)spare * s;
}
// The last sequence whose units start at or before u, and its start and end: each lane of a wave tries one, up
// to 64 sequences with one wait for memory, 4096 with two (a search by halves waits for one load after
// another, 1.5 us for 9 sequences).
struct UnitSeq { int s, start, end; };
__device__ __forceinline__ UnitSeq unit_seq(const int32_t *start, int n_seqs, int64_t u, int mul, int unit, int spare) {
    const int lane = threadIdx.x & 63;
    UnitSeq q{};
    for (int step = n_seqs > 64 ? 64 : 1; step; step /= 64) {
        const int t = min(q.s + lane * step, n_seqs - 1), from = gmem(start)[t], to = gmem(start)[t + 1];
        const uint64_t before = __ballot(q.s + lane * step < n_seqs && unit_base(from, t, mul, unit, spare) <= u);
        const int at = before ? 63 - __builtin_clzll(before) : 0;
        q = {q.s + at * step, __builtin_amdgcn_readlane(from, at), __builtin_amdgcn_readlane(to, at)};
    }
    return q;
}

// ---------------------------------------------------------------- checks (one block of arguments or another)
template <typename A> int serve_check(const char *who, const A *a) {
    OP_NEED(a, "null arguments");
    OP_NEED(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256, "head_dim is not 64, 128 or 256");
    OP_NEED(a->n_kv_heads > 0 && a->n_heads > 0 && a->n_heads % a->n_kv_heads == 0 && a->n_heads / a->n_kv_heads <= 16 && a->n_heads <= 4096,
            "n_heads is not n_kv_heads times 1 to 16");
    OP_NEED(a->type == SP_HIPKV_F32 || a->type == SP_HIPKV_BF16, "unknown type");
    OP_NEED(a->n_seqs >= 0 && a->n_seqs <= 4096, "n_seqs outside [0, 4096]");
    OP_NEED(a->n_tokens >= 0 && a->n_tokens <= 1 << 20, "n_tokens outside [0, 2^20]");
    OP_NEED(a->max_tokens >= 0 && a->n_tokens <= (int64_t)a->n_seqs * a->max_tokens, "n_tokens is more than n_seqs times max_tokens");
    return 0;
}
// a packed array of values: heads x head_dim of them a token
template <typename A> int serve_rows(const char *who, const A *a, const void *p, int64_t stride, int heads) {
    OP_NEED(p, "null array");
    OP_NEED(stride >= (int64_t)heads * a->head_dim && stride % (a->type == SP_HIPKV_F32 ? 4 : 8) == 0 && stride <= 1 << 22,
            "a stride is below heads * head_dim, above 2^22 or does not keep rows 16-byte aligned");
    OP_NEED(aligned(p, 16), "misaligned array");
    return 0;
}

}  // namespace kvd
