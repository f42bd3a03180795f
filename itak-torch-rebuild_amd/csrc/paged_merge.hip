// Joins the partials of units that several workgroups shared: out = sum_w 2^(m_w - m) acc_w / sum_w 2^(m_w - m) l_w.
//
// A workgroup serves one query head's row. Its unit's place in the line of blocks gives the workgroups that had a part of it, and so
// their slots. Eight lanes of a quarter of the channels' float4s each take every eighth partial, all loads of a partial's
// accumulators in flight beside the maxima, and meet in LDS. Two trips to memory and a launch are what it costs.
#include "paged.h"

#include "mfma_common.h"

namespace itak {

namespace {

constexpr int kThreads = 256;

template <int ELEM, int DP>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr int kQuads = DP / 4;               // float4s of a partial
    constexpr int kLanes = kThreads / kQuads;    // partials taken at once
    __shared__ floatx4 lds[kLanes][kQuads];
    __shared__ float lds_l[kLanes], lds_m[kLanes];
    const uint32_t tid = threadIdx.x, row = blockIdx.x, hq = blockIdx.y;
    const PagedLine line(a);
    const uint32_t share = a.parts ? 0 : paged_share(a, line.total());
    PagedSpan span;
    if (!line.find(span, [=](const PagedSpan &s, uint32_t) { return row >= s.row0 && row - s.row0 < s.rows; })) return;
    const uint32_t head = hq / a.group, v = (row - span.row0) * a.group + (hq - head * a.group);
    // (The kernel of many rows counts an item's tiles from the last.)
    const uint32_t tile = v / a.tile, local = (a.parts ? span.tiles - 1 - tile : tile) * a.g.kv_heads + head;
    const uint32_t unit = span.unit0 + local;
    // Slots first .. last of the unit's partials, from slot `base` on.
    uint32_t first = 0, last = a.parts - 1;
    uint64_t base = uint64_t(unit) * a.parts;
    if (a.parts) {
        if (unit >= a.units) return;
    } else {
        const uint32_t from = span.start + local * span.blocks;
        first = from / share, last = (from + span.blocks - 1) / share, base = unit;
        if (first == last || last + unit >= a.groups + a.units) return;  // written whole
    }
    const uint32_t quad = tid % kQuads, part = tid / kQuads;
    float m = -INFINITY, l = 0.0f;
    floatx4 acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t w = first + part; w <= last; w += kLanes) {
        const uint64_t slot = (base + w) * a.tile + (v - tile * a.tile);
        const float2 ml = a.ws_ml[slot];
        const floatx4 x = *reinterpret_cast<const floatx4 *>(a.ws_acc + slot * DP + quad * 4);
        if (ml.x == -INFINITY) {
            l += ml.y;  // nothing visible (0), or scores that are no numbers
            continue;
        }
        const float next = fmaxf(m, ml.x), old = m == -INFINITY ? 0.0f : fast_exp2(m - next), now = fast_exp2(ml.x - next);
        l = l * (m == -INFINITY ? 1.0f : old) + now * ml.y;
        acc = acc * old + x * now;
        m = next;
    }
    lds[part][quad] = acc;
    if (quad == 0) lds_l[part] = l, lds_m[part] = m;
    __syncthreads();
    if (tid >= kQuads) return;
    float most = -INFINITY;
#pragma unroll
    for (int p = 0; p < kLanes; ++p) most = fmaxf(most, lds_m[p]);
    float total = 0.0f;
    floatx4 sum = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < kLanes; ++p) {
        const float weight = lds_m[p] == -INFINITY ? 0.0f : fast_exp2(lds_m[p] - most);
        total += lds_m[p] == -INFINITY ? lds_l[p] : weight * lds_l[p];
        sum += lds[p][tid] * weight;
    }
    const float inv = 1.0f / total;
    const uint32_t c = tid * 4;
    if (c >= a.g.head_dim) return;
    T *dst = static_cast<T *>(a.out.data) + uint64_t(row) * a.out.row_stride + hq * a.out.head_stride + c;
    Piece<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(sum[e] * inv);
    if (a.out_on_16) {
        *reinterpret_cast<Piece<T, 4> *>(dst) = y;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[e] = y.v[e];
    }
}

template <int ELEM>
void launch(const PagedAttn &a, hipStream_t stream) {
    const dim3 grid(a.rows, a.g.kv_heads * a.group);
    const uint32_t dp = paged_padded(a.g.head_dim);
    if (dp == 64)
        launch_kernel(paged_merge_kernel<ELEM, 64>, grid, kThreads, 0, stream, a);
    else if (dp == 128)
        launch_kernel(paged_merge_kernel<ELEM, 128>, grid, kThreads, 0, stream, a);
    else
        launch_kernel(paged_merge_kernel<ELEM, 256>, grid, kThreads, 0, stream, a);
}

}  // namespace

hipError_t launch_paged_merge(uint32_t elem, const PagedAttn &a, hipStream_t stream) {
    if (elem == ITAK_ELEM_F32)
        launch<ITAK_ELEM_F32>(a, stream);
    else if (elem == ITAK_ELEM_F16)
        launch<ITAK_ELEM_F16>(a, stream);
    else
        launch<ITAK_ELEM_BF16>(a, stream);
    return hipGetLastError();
}

}  // namespace itak
