// The kernel of few rows over bf16 pages, bf16 tensors, of a batch whose rows may be trees.
#include "paged_few_kernel.h"

namespace itak {

hipError_t launch_paged_few_tree_bf16(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    return launch_few<ITAK_ELEM_BF16, ITAK_ELEM_BF16, 1, 1, true>(sets, a, stream);
}

}  // namespace itak
