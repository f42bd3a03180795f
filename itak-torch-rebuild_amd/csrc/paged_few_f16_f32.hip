// The kernel of few rows over f16 pages, f32 tensors.
// Queries and weights as two halves each: 22 bits of them.
#include "paged_few_kernel.h"

namespace itak {

hipError_t launch_paged_few_f16_f32(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    return launch_few<ITAK_ELEM_F16, ITAK_ELEM_F32, 2, 2>(sets, a, stream);
}

}  // namespace itak
