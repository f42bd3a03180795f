// The matrix products of paged attention on the two 16-bit types.
#pragma once

#include "mfma_common.h"
#include "paged.h"

namespace itak {

typedef __bf16 bfloat8 __attribute__((ext_vector_type(8)));

// S += A . B, A 16 x 32 and B 32 x 16: lane (i, g) holds row i of A (column i of B), elements 8g .. 8g + 7, and of S column i,
// rows 4g .. 4g + 3.
template <int PAGE>
__device__ __forceinline__ floatx4 mfma_16x16x32(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (PAGE == ITAK_ELEM_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
}

// Eight f32 as PIECES vectors of the pages' type whose sum they are: each piece the rounding of what the ones before leave.
template <int PAGE, int PIECES>
__device__ __forceinline__ void split_8(const float (&x)[8], u32x4 (&out)[PIECES]) {
    typedef typename Elem<PAGE>::type T;
    typedef T vec8 __attribute__((ext_vector_type(8)));
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        vec8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = T(rest[e]);
            if (p + 1 < PIECES) rest[e] -= float(v[e]);
        }
        out[p] = __builtin_bit_cast(u32x4, v);
    }
}

// Bit 15 or 31 of the result is set if the half there is an infinity or a NaN (its exponent field all ones: one more carries).
template <int PAGE>
__device__ __forceinline__ uint32_t not_finite_2(uint32_t x) {
    return PAGE == ITAK_ELEM_F16 ? (x & 0x7c007c00u) + 0x04000400u : (x & 0x7f807f80u) + 0x00800080u;
}

// The halves that are neither, zero in place of the others.
template <int PAGE>
__device__ __forceinline__ u32x4 finite_only(u32x4 x) {
    u32x4 y;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t bad = not_finite_2<PAGE>(x[c]) & 0x80008000u;
        y[c] = x[c] & ~((bad >> 15) * 0xffffu);
    }
    return y;
}

// The maximum over the four lanes that hold one column of S.
__device__ __forceinline__ float max_over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

}  // namespace itak
