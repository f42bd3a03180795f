// The kernel of many rows over f16 pages, f16 tensors.
#include "paged_chunk_kernel.h"

namespace itak {

hipError_t launch_paged_chunk_f16(const PagedAttn &a, hipStream_t stream) {
    return launch_chunk<ITAK_ELEM_F16, ITAK_ELEM_F16, 1, 1>(a, stream);
}

}  // namespace itak
