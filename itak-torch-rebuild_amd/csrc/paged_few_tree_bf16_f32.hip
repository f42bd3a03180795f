// The kernel of few rows over bf16 pages, f32 tensors, of a batch whose rows may be trees.
// Queries and weights as three pieces each: 24 bits of them.
#include "paged_few_kernel.h"

namespace itak {

hipError_t launch_paged_few_tree_bf16_f32(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    return launch_few<ITAK_ELEM_BF16, ITAK_ELEM_F32, 3, 3, true>(sets, a, stream);
}

}  // namespace itak
