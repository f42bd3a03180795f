// The kernel of few rows over f16 pages, f32 tensors, of a batch whose rows may be trees.
// Queries and weights as two halves each: 22 bits of them.
#include "paged_few_kernel.h"

namespace itak {

hipError_t launch_paged_few_tree_f16_f32(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    return launch_few<ITAK_ELEM_F16, ITAK_ELEM_F32, 2, 2, true>(sets, a, stream);
}

}  // namespace itak
