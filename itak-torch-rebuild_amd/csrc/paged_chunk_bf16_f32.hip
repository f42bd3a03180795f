// The kernel of many rows over bf16 pages, f32 tensors.
#include "paged_chunk_kernel.h"

namespace itak {

hipError_t launch_paged_chunk_bf16_f32(const PagedAttn &a, hipStream_t stream) {
    return launch_chunk<ITAK_ELEM_BF16, ITAK_ELEM_F32, 3, 3>(a, stream);
}

}  // namespace itak
