/* Floats as sums of three bfloat16, for products in 32 bits on the bfloat16
 * matrix cores. */
#ifndef PK_PIECES_H
#define PK_PIECES_H

#include <hip/hip_runtime.h>

#pragma clang fp contract(off)

namespace pkq8 {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f_c __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct Pieces {
    v8bf p[3];
};

/* Floats cut for a product of floats with floats: each piece the nearest
 * bfloat16 of what the ones before leave, so that the second is at most 2^-8
 * of the float's power of two, the third 2^-17, and the three sum to it exactly
 * (down to 2^-133, the smallest bfloat16). Of the nine products of two floats'
 * pieces the six largest are taken: those left out are 2^-24 of the product at
 * most, as much as a 32-bit product's own rounding. Whatever the other
 * dimensions hold: a row has no exponent in common. */
__device__ __forceinline__ Pieces cut_near(const float (&x)[8]) {
    Pieces r;
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v2f_c a = { x[2 * i], x[2 * i + 1] };
#pragma unroll
        for (int n = 0; n < 3; n++) {
            w[n][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(a, v2bf));
            a.x -= __uint_as_float(w[n][i] << 16);
            a.y -= __uint_as_float(w[n][i] & 0xffff0000u);
        }
    }
#pragma unroll
    for (int n = 0; n < 3; n++)
        r.p[n] = __builtin_bit_cast(v8bf, v4u{ w[n][0], w[n][1], w[n][2], w[n][3] });
    return r;
}

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

}  // namespace pkq8

#endif
