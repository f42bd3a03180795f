// The matrix products of paged attention on the two 16-bit types.
#pragma once

#include "mfma_common.h"
#include "paged.h"

namespace itak {

typedef __bf16 bfloat8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// S += A . B, A 16 x 32 and B 32 x 16: lane (i, g) holds row i of A (column i of B), elements 8g .. 8g + 7, and of S column i,
// rows 4g .. 4g + 3.
template <int PAGE>
__device__ __forceinline__ floatx4 mfma_16x16x32(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (PAGE == ITAK_ELEM_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
}

// Over f16 pages a row's reference is kept 12 below its largest score (log2 domain): weights are up to 2^15, where f16 ends at 2^16, so that of
// f16 pieces those down to 2^-26 of the largest keep their precision and what is lost of a smaller one is 2^-37 of the largest. bf16
// has f32's range and values of it may end where the accumulators do: no lift. The reference
// moves only when a score passes it by more than 15: the rescaling of the accumulators then leaves the common path.
template <int PAGE>
constexpr float kWeightLift = PAGE == ITAK_ELEM_F16 ? 12.0f : 0.0f;
constexpr float kWeightMost = 15.0f;
// f32 queries enter f16 products times 16, and the scale makes up for it: f16 ends at 2^-24 below, and a query's last bits do
// then at 2^-28. (One beyond 4,094 is infinite to the products and is done over in f32, as all that is not finite.)
template <int PAGE, int ELEM>
constexpr float kQueryLift = PAGE == ITAK_ELEM_F16 && ELEM == ITAK_ELEM_F32 ? kPagedQueryLift : 1.0f;

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

// Eight channels of a query as they are loaded, on 16 bytes or element by element, and as operands: `in` = false gives zeros.
template <int ELEM>
struct QueryRaw {
    typedef u32x4 type;
};
typedef float floatx8 __attribute__((ext_vector_type(8)));
template <>
struct QueryRaw<ITAK_ELEM_F32> {
    typedef floatx8 type;
};
template <int ELEM, bool ON_16>
__device__ __forceinline__ typename QueryRaw<ELEM>::type load_query(const typename Elem<ELEM>::type *p) {
    typename QueryRaw<ELEM>::type x;
    if constexpr (ELEM == ITAK_ELEM_F32) {
        if constexpr (ON_16) {
            const floatx4 lo = *reinterpret_cast<const floatx4 *>(p), hi = *reinterpret_cast<const floatx4 *>(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = hi[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e];
        }
    } else if constexpr (ON_16) {
        x = *reinterpret_cast<const u32x4 *>(p);
    } else {
        const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = u[2 * e] | (uint32_t(u[2 * e + 1]) << 16);
    }
    return x;
}
template <int PAGE, int ELEM, int NQ, typename F>
__device__ __forceinline__ void split_query(const typename QueryRaw<ELEM>::type &raw, bool in, F store) {
    if constexpr (ELEM == ITAK_ELEM_F32) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = in ? raw[e] * kQueryLift<PAGE, ELEM> : 0.0f;
        u32x4 pieces[NQ];
        split_8<PAGE, NQ>(x, pieces);
#pragma unroll
        for (int n = 0; n < NQ; ++n) store(n, pieces[n]);
    } else {
        store(0, in ? raw : u32x4{0, 0, 0, 0});
    }
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

// A capped score relative to `shift`: c tanh(y) - shift, y = a ln 2 / 2, in the log2 domain (softcap_of_exp2_arg). Where a small score is
// to be as exact as one without a cap (SERIES), and 1 - 2 / (2^a + 1) leaves some 2^-23 of the cap: up to |y| = 0.45 the
// series y (1 - y^2 / 3 + 2 y^4 / 15 - ..) to y^13, whose next term is below 2^-25 of the value. That is for f32 tensors, and of 16 bits for
// caps beyond kPagedCapShort, below which the short form's error is a tenth of what a weight's rounding to f16 takes. STRAIGHT: both are
// worked out, where the compiler would make a branch of the choice, which turns lanes off amid the fullest registers.
template <bool SERIES, bool STRAIGHT = false>
__device__ __forceinline__ float softcapped(float a, float c, float shift) {
    if constexpr (!SERIES) return softcap_of_exp2_arg(a, c, shift);
    const float y = a * 0.34657359f, z = y * y;
    float p = __builtin_fmaf(z, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
    p = __builtin_fmaf(z, p, 62.0f / 2835.0f);
    p = __builtin_fmaf(z, p, -17.0f / 315.0f);
    p = __builtin_fmaf(z, p, 2.0f / 15.0f);
    p = __builtin_fmaf(z, p, -1.0f / 3.0f);
    float small = __builtin_fmaf(__builtin_fmaf(y * z, p, y), c, -shift);
    if constexpr (STRAIGHT) {
        float large = softcap_of_exp2_arg(a, c, shift);
        asm("" : "+v"(small), "+v"(large));
        return __builtin_fabsf(y) < 0.45f ? small : large;
    }
    return __builtin_fabsf(y) < 0.45f ? small : softcap_of_exp2_arg(a, c, shift);
}

}  // namespace itak
