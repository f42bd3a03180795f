// Joins the partials of units that several workgroups shared: out = sum_w 2^(m_w - m) acc_w / sum_w 2^(m_w - m) l_w. Weights are divided by the
// sum before they meet the accumulators: acc_w / l_w is a mean of values, and no sum of the parts leaves f32's range if they do not.
//
// A workgroup serves one query head's row. Its unit's place in the line of blocks gives the workgroups that had a part of it, and so
// their slots. All loads go out before anything waits: maxima and sums a lane each, accumulators (a float4 a thread and
// partial) up to eight of a thread's at once. Up to 64 partials every wavefront works out the weights for itself; of more they
// meet in LDS. One trip to memory and a launch are what it costs: 33 partials of one token's 32 heads 3.3 us.
#include "paged.h"

#include "paged_mfma.h"

namespace itak {

namespace {

constexpr int kThreads = 256;

template <int ELEM, int DP>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr int kQuads = DP / 4;               // float4s of a partial
    constexpr int kLanes = kThreads / kQuads;    // partials taken at once
    constexpr int kAtOnce = 8;
    __shared__ floatx4 lds[kLanes][kQuads];
    __shared__ float weights[kPagedMostParts], lds_m[kThreads / 64], lds_l[kThreads / 64];
    paged_fetch_arguments(a);
    const uint32_t tid = threadIdx.x, row = blockIdx.x, hq = blockIdx.y;
    PagedLine line(a);
    if (!a.parts) line.cut();
    PagedSpan span;
    if (!line.find<PagedLine::kRow>(span, row)) return;
    const uint32_t head = paged_row_of(a, hq), v = (row - span.row0) * a.group + (hq - head * a.group);
    // (The kernel of many rows counts an item's tiles from the last.)
    const uint32_t tile = v >> a.tile_shift, local = (a.parts ? span.tiles - 1 - tile : tile) * a.g.kv_heads + head;
    const uint32_t unit = span.unit0 + local;
    // Slots first .. last of the unit's partials, from slot `base` on.
    uint32_t first = 0, last = a.parts - 1;
    uint64_t base = uint64_t(unit) * a.parts;
    if (a.parts) {
        if (unit >= a.units) return;
    } else {
        const uint32_t from = span.start + local * span.run;
        first = from / line.share, last = (from + span.blocks - 1) / line.share, base = unit;
        if (first == last || last + unit >= a.groups + a.units) return;  // written whole
    }
    const uint32_t quad = tid % kQuads, part = tid / kQuads, parts = last - first + 1;
    base = (base + first) * a.tile + (v - (tile << a.tile_shift));
    const float *const acc_at = a.ws_acc + base * DP + quad * 4;
    auto acc_of = [&](uint32_t w) { return *reinterpret_cast<const floatx4 *>(acc_at + uint64_t(w) * a.tile * DP); };
    floatx4 early[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) early[u] = acc_of(min(part + u * kLanes, parts - 1));
    // (A maximum of minus infinity: nothing visible, a sum of 0, or scores that are no numbers, which the sum then is.)
    auto weight_of = [](float2 x, float m) { return x.x == -INFINITY ? 0.0f : fast_exp2(x.x - m) * (x.y < 0.0f ? kPagedMergeLift : 1.0f); };
    auto sum_of = [](float2 x, float weight) { return x.x == -INFINITY ? x.y : weight * __builtin_fabsf(x.y); };
    floatx4 acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    if (parts <= 64) {
        // Every wavefront has all of them, one a lane.
        const uint32_t lane = __lane_id();
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < parts) ml = a.ws_ml[base + uint64_t(lane) * a.tile];
        float m = ml.x;
        m = fmaxf(m, dpp_lane<0xB1>(m));   // quad_perm [1,0,3,2]
        m = fmaxf(m, dpp_lane<0x4E>(m));   // quad_perm [2,3,0,1]
        m = fmaxf(m, dpp_lane<0x141>(m));  // row_half_mirror
        m = fmaxf(m, dpp_lane<0x140>(m));  // row_mirror
        m = max_over_groups(m);
        const float weight = weight_of(ml, m);
        float l = sum_of(ml, weight);
        l += dpp_lane<0xB1>(l);
        l += dpp_lane<0x4E>(l);
        l += dpp_lane<0x141>(l);
        l += dpp_lane<0x140>(l);
        const float share = weight * (1.0f / sum_over_groups(l));
        const uint32_t most = 64 / kLanes;  // of a thread's
#pragma unroll
        for (uint32_t u = 0; u < most; ++u) {
            const float w = __shfl(share, part + u * kLanes);
            if (u >= kAtOnce && u * kLanes >= parts) break;
            const floatx4 x = u < kAtOnce ? early[u] : acc_of(min(part + u * kLanes, parts - 1));
            if (part + u * kLanes < parts) acc += x * w;
        }
    } else {
        float2 ml[kPagedMostParts / kThreads];
        float m = -INFINITY;
#pragma unroll
        for (uint32_t u = 0; u < kPagedMostParts / kThreads; ++u) {
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (tid + u * kThreads < parts) ml[u] = a.ws_ml[base + uint64_t(tid + u * kThreads) * a.tile];
            m = fmaxf(m, ml[u].x);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if ((tid & 63) == 0) lds_m[tid >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
        float l = 0.0f;
#pragma unroll
        for (uint32_t u = 0; u < kPagedMostParts / kThreads; ++u) {
            const float weight = weight_of(ml[u], m);
            l += sum_of(ml[u], weight);
            if (tid + u * kThreads < parts) weights[tid + u * kThreads] = weight;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
        if ((tid & 63) == 0) lds_l[tid >> 6] = l;
        __syncthreads();
        const float inv = 1.0f / ((lds_l[0] + lds_l[1]) + (lds_l[2] + lds_l[3]));
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            if (part + u * kLanes < parts) acc += early[u] * (weights[part + u * kLanes] * inv);
        for (uint32_t w = part + kAtOnce * kLanes; w < parts; w += kLanes) acc += acc_of(w) * (weights[w] * inv);
    }
    lds[part][quad] = acc;
    __syncthreads();
    if (tid >= kQuads) return;
    floatx4 sum = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < kLanes; ++p) sum += lds[p][tid];
    const uint32_t c = tid * 4;
    if (c >= a.g.head_dim) return;
    T *dst = static_cast<T *>(a.out.data) + uint64_t(row) * a.out.row_stride + hq * a.out.head_stride + c;
    Piece<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(sum[e]);
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
