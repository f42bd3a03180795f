// The kernel of many rows over bf16 pages, bf16 tensors, of a batch whose rows may be trees.
#include "paged_chunk_kernel.h"

namespace itak {

hipError_t launch_paged_chunk_tree_bf16(const PagedAttn &a, hipStream_t stream) {
    return launch_chunk<ITAK_ELEM_BF16, ITAK_ELEM_BF16, 1, 1, true>(a, stream);
}

}  // namespace itak
