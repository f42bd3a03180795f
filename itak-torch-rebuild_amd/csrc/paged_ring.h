// What the kernels of tiles over pages share: the wide products, and loads that travel from the pages to LDS.
#pragma once

#include "paged_mfma.h"

namespace itak {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

template <int PAGE>
__device__ __forceinline__ floatx16 mfma_32x32x16(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (PAGE == ITAK_ELEM_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
}

// Issued from assembly: the compiler then neither waits for such a load at every LDS read nor needs to, because its only
// consumer is ordered by the wait and the barrier at the top of each block. It does not look for hazards in there either: a scalar
// register that vector code wrote (readlane: the address) takes five wait states before a load may read it, m0 one.
__device__ __forceinline__ void page_to_lds(uint64_t base, uint32_t offset, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ void lane_to_lds(uint64_t address, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(address), "s"(lds_addr) : "memory");
}
template <int n>
__device__ __forceinline__ void wait_loads() {  // s_waitcnt vmcnt(n), other counters untouched
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | ((n >> 4) << 14));
}

}  // namespace

}  // namespace itak
