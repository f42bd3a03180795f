// The kernel of few rows over f16 pages, f16 tensors.
#include "paged_few_kernel.h"

namespace itak {

hipError_t launch_paged_few_f16(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    return launch_few<ITAK_ELEM_F16, ITAK_ELEM_F16, 1, 1>(sets, a, stream);
}

}  // namespace itak
