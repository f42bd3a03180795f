// The kernel of trees over bf16 pages, f32 tensors.
#include "paged_trees_kernel.h"

namespace itak {

hipError_t launch_paged_trees_bf16_f32(const PagedAttn &a, hipStream_t stream) {
    return launch_trees<ITAK_ELEM_BF16, ITAK_ELEM_F32, 3, 3>(a, stream);
}

}  // namespace itak
