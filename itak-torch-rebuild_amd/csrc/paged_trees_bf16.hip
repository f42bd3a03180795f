// The kernel of trees over bf16 pages, bf16 tensors.
#include "paged_trees_kernel.h"

namespace itak {

hipError_t launch_paged_trees_bf16(const PagedAttn &a, hipStream_t stream) {
    return launch_trees<ITAK_ELEM_BF16, ITAK_ELEM_BF16, 1, 1>(a, stream);
}

}  // namespace itak
