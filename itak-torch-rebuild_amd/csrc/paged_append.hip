// New rows into pages, keys turned by their positions on the way; of a step its queries too, into a buffer beside.
//
// A workgroup serves one row of the batch or a part of its heads: one trip to memory for the batch's items, one for the page
// id, during which the row's cosines and sines are worked out once into LDS; then every thread moves pieces of eight
// channels, 16 bytes a load and store. Bytes bound it where rows are many, the two trips and the launch where they are few: 2,048 rows
// of 4 heads by 128, 8.4 MB, 5.1 us; 16 rows 2.7 us; a launch that does nothing takes 1.3.
#include "paged.h"

namespace itak {

namespace {

constexpr int kThreads = 256;

template <int PAGE, int ELEM, int W>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedAppend a) {
    typedef typename Elem<ELEM>::type T;
    typedef typename Elem<PAGE>::type P;
    __shared__ float2 cs[kMostPairs];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    uint4 item;
    if (!paged_item_of_row(a.g, a.batch, row, item)) return;  // (the same for the whole workgroup)
    const uint32_t position = item.x + (row - item.z);
    // (A row of a tree is turned by its depth.)
    const uint32_t turned_by = a.tree && a.batch[2] ? item.x + tree_depth(a.tree[uint64_t(row) * kTreeStride]) : position;
    const uint32_t page = a.batch[item.w + (position >> a.g.page_shift)];
    if (tid < a.r.half) cs[tid] = turn_of(a.r, double(turned_by), tid);
    __syncthreads();
    P *const base = reinterpret_cast<P *>(a.layer_base) + page * a.g.page_stride +
                    uint64_t(position & ((1u << a.g.page_shift) - 1)) * a.g.head_dim;
    const HeadPieces turned = head_pieces(a.g.head_dim, a.r.half, a.r.interleaved, W);
    const HeadPieces plain = head_pieces(a.g.head_dim, 0, 0, W);
    const uint32_t q_pieces = a.q_heads * turned.all, k_pieces = a.g.kv_heads * turned.all;
    const uint32_t first = blockIdx.y * a.per_group, end = min(first + a.per_group, a.pieces);
    for (uint32_t p = first + tid; p < end; p += kThreads) {
        if (p < q_pieces) {
            const uint32_t head = p / turned.all;
            move_piece<ELEM, ELEM, W>(static_cast<const T *>(a.q.data) + row * a.q.row_stride + head * a.q.head_stride,
                                      static_cast<T *>(a.q_out.data) + row * a.q_out.row_stride + head * a.q_out.head_stride,
                                      p - head * turned.all, turned, a.r.half, a.r.interleaved, cs, 1.0f);
        } else if (p - q_pieces < k_pieces) {
            const uint32_t at = p - q_pieces, head = at / turned.all;
            move_piece<ELEM, PAGE, W>(static_cast<const T *>(a.k.data) + row * a.k.row_stride + head * a.k.head_stride,
                                      base + head * a.g.head_stride, at - head * turned.all, turned, a.r.half, a.r.interleaved, cs,
                                      1.0f);
        } else {
            const uint32_t at = p - q_pieces - k_pieces, head = at / plain.all;
            move_piece<ELEM, PAGE, W>(static_cast<const T *>(a.v.data) + row * a.v.row_stride + head * a.v.head_stride,
                                      base + a.g.side_stride + head * a.g.head_stride, at - head * plain.all, plain, 0, 0, cs, 1.0f);
        }
    }
}

template <int PAGE, int ELEM>
void launch(bool by_8, const PagedAppend &a, dim3 grid, hipStream_t stream) {
    if (by_8)
        launch_kernel(paged_append_kernel<PAGE, ELEM, 8>, grid, kThreads, 0, stream, a);
    else
        launch_kernel(paged_append_kernel<PAGE, ELEM, 1>, grid, kThreads, 0, stream, a);
}

}  // namespace

hipError_t launch_paged_append(uint32_t page_elem, uint32_t elem, bool by_8, const PagedAppend &args, uint32_t rows,
                               hipStream_t stream) {
    PagedAppend a = args;
    const uint32_t w = by_8 ? 8 : 1;
    const uint32_t turned = head_pieces(a.g.head_dim, a.r.half, a.r.interleaved, w).all;
    a.pieces = (a.q_heads + a.g.kv_heads) * turned + a.g.kv_heads * head_pieces(a.g.head_dim, 0, 0, w).all;
    // Few rows are cut into parts of their heads until the device has two workgroups a compute unit.
    const uint32_t whole = (a.pieces + kThreads - 1) / kThreads;
    const uint32_t parts = std::min(whole, std::max(1u, 512u / rows));
    a.per_group = (whole + parts - 1) / parts * kThreads;
    const dim3 grid(rows, (a.pieces + a.per_group - 1) / a.per_group);
    if (page_elem == ITAK_ELEM_F16) {
        if (elem == ITAK_ELEM_F16)
            launch<ITAK_ELEM_F16, ITAK_ELEM_F16>(by_8, a, grid, stream);
        else
            launch<ITAK_ELEM_F16, ITAK_ELEM_F32>(by_8, a, grid, stream);
    } else {
        if (elem == ITAK_ELEM_BF16)
            launch<ITAK_ELEM_BF16, ITAK_ELEM_BF16>(by_8, a, grid, stream);
        else
            launch<ITAK_ELEM_BF16, ITAK_ELEM_F32>(by_8, a, grid, stream);
    }
    return hipGetLastError();
}

}  // namespace itak
