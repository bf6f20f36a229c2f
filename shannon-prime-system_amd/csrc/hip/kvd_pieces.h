// kvd_pieces.h -- products of f32 numbers on the bf16 matrix cores, in exact pieces.
#pragma once
#include "kvd_internal.h"

namespace kvd {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// whether bf16 pieces hold x: not infinities, NaN, nor the magnitudes above the midpoint of the
// largest bf16 number and the next power of two, which round up to an infinite first piece
constexpr uint32_t PIECES_END = 0x7F7F8000u;
__device__ __forceinline__ bool pieces_hold(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) < PIECES_END; }

// Of an f32 its three bf16 pieces, which sum to it exactly: x = h + m + l, |m| <= 2^-9 |x|,
// |l| <= 2^-18 |x| (magnitudes from PIECES_END on round up to infinity and make NaN, with a weight of 0
// too; below 2^-110 l is lost to denormals bit by bit).  Cutting bits off instead of rounding saves 4% of a call, and
// 2^-21 of a product would be missing for 2^-26.
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

}  // namespace kvd
