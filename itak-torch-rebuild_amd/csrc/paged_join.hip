// Joins the partials of the kernel of trees: out = sum_w 2^(m_w - m) acc_w / sum_w 2^(m_w - m) l_w, the weights divided by the sum before they meet
// the accumulators (paged_merge.hip says why).
//
// A unit's parts lie in consecutive slots, each a tile's accumulators as registers held them: 16 bytes of four channels, 32 vectors side by side. A
// wavefront serves four vectors, which share their 64 bytes, and has four channels of each in a lane; where parts are many and vectors few the four
// wavefronts of a workgroup share the parts. Bytes bound it, and below some megabytes the trips: item, maxima and sums, accumulators (4.4 MB 4.0 us, 13.6 MB
// 5.4, 33 MB 9.0: 3.7 TB/s).
#include "paged_mfma.h"

namespace itak {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kJoined = 4;  // vectors of a wavefront

// SHARED: wavefronts that share the parts of their vectors, 1 or 4.
template <int ELEM, int DP, uint32_t SHARED>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr uint32_t kOfLane = DP / 64, kQuads = DP / 8, kAtOnce = (SHARED > 1 ? 16 : 8) / kOfLane;  // quads of a lane; of a lane of the tile; parts at once
    constexpr uint32_t kWaves = kThreads / 64;
    const uint32_t of_tile = a.tile / kJoined;  // (a power of two)
    __shared__ float lds_weight[SHARED > 1 ? 1 : kWaves][kPagedTreesGroups][kJoined];
    __shared__ floatx4 lds_acc[SHARED > 1 ? SHARED - 1 : 1][SHARED > 1 ? kOfLane : 1][64];
    paged_fetch_arguments<true>(a);
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    // (Eight vectors share their lines of memory: workgroups on the same compute die, eight apart, have them; side by side, on two dies, the lines came
    // twice: 13.6 MB 7.2 us for 5.4. A head's workgroups are a multiple of sixteen.)
    const uint32_t beside = (blockIdx.x & ~15u) | (blockIdx.x & 7) << 1 | (blockIdx.x >> 3 & 1);
    const uint32_t joined = SHARED > 1 ? beside : blockIdx.x * kWaves + wave, unit = joined >> (a.tile_shift - 2);
    static_assert(kJoined == 4, "a tile is 2^(tile_shift - 2) times that");
    PagedTreeLine line(a);
    line.cut_apart();
    PagedSpan span;
    if (!line.find<PagedTreeLine::kUnit>(span, unit)) return;
    const uint32_t parts = (span.blocks + line.share - 1) / line.share;
    if (parts <= 1) return;  // written whole
    const uint32_t turn = unit - span.unit0, tile = span.tiles - 1 - turn, head = blockIdx.y;
    const uint32_t vectors = span.rows * a.group, of0 = (joined - unit * of_tile) * kJoined, v0 = tile * a.tile + of0;
    const uint32_t first_slot = (span.start + turn * span.run) / line.share;
    if (v0 >= vectors || first_slot + parts > a.groups) return;
    const uint32_t slot = head * a.groups + first_slot;
    const uint32_t mine = lane % kJoined, of = of0 + mine;
    const float2 *const ml_at = a.ws_ml + uint64_t(slot) * a.tile + of;
    // (Quad q of the vector: registers 4 q of a lane of the half h of its column's set, q = 2 * that + h.)
    const floatx4 *const acc_at = reinterpret_cast<const floatx4 *>(a.ws_acc) + uint64_t(slot) * a.tile * (DP / 4) +
                                  (of / 32 * kQuads) * 64 + of % 32;
    auto acc_of = [&](uint32_t part, uint32_t i) {
        const uint32_t q = lane / kJoined + 16 * i;
        return acc_at[uint64_t(part) * a.tile * (DP / 4) + (q / 2) * 64 + (q % 2) * 32];
    };
    // The first accumulators are asked for before the maxima are there.
    const uint32_t first = SHARED > 1 ? wave : 0;
    floatx4 early[kAtOnce][kOfLane];
    // (The second half of them where there are as many.)
    auto ask = [&](uint32_t p0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            if (u >= kAtOnce / 2 && p0 + kAtOnce / 2 * SHARED >= parts) break;
#pragma unroll
            for (uint32_t i = 0; i < kOfLane; ++i) early[u][i] = acc_of(min(p0 + u * SHARED, parts - 1), i);
        }
    };
    ask(first);
    // A lane has every sixteenth part's maximum and sum of its vector. The first 64 parts' stay in registers.
    constexpr uint32_t kKept = 4;
    float2 ml[kKept];
    float m = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < kKept; ++u) {
        const uint32_t p = lane / kJoined + 16 * u;
        ml[u] = make_float2(-INFINITY, 0.0f);
        if (p < parts) ml[u] = ml_at[uint64_t(p) * a.tile];
        m = fmaxf(m, ml[u].x);
    }
    for (uint32_t p = lane / kJoined + 16 * kKept; p < parts; p += 16) m = fmaxf(m, ml_at[uint64_t(p) * a.tile].x);
#pragma unroll
    for (uint32_t o = kJoined; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    // (A maximum of minus infinity: nothing visible, a sum of 0, or scores that are no numbers, which the sum then is.)
    auto weight_of = [&](float2 x) { return x.x == -INFINITY ? 0.0f : fast_exp2(x.x - m) * (x.y < 0.0f ? kPagedMergeLift : 1.0f); };
    auto sum_of = [&](float2 x) { return x.x == -INFINITY ? x.y : weight_of(x) * __builtin_fabsf(x.y); };
    float l = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < kKept; ++u) l += sum_of(ml[u]);
    for (uint32_t p = lane / kJoined + 16 * kKept; p < parts; p += 16) l += sum_of(ml_at[uint64_t(p) * a.tile]);
#pragma unroll
    for (uint32_t o = kJoined; o < 64; o *= 2) l += __shfl_xor(l, o);
    const float inv = 1.0f / l;
    // (Wavefronts that share their vectors write the same weights to the same places.)
    auto weights = lds_weight[SHARED > 1 ? 0 : wave];
#pragma unroll
    for (uint32_t u = 0; u < kKept; ++u)
        if (lane / kJoined + 16 * u < parts) weights[lane / kJoined + 16 * u][mine] = weight_of(ml[u]) * inv;
    for (uint32_t p = lane / kJoined + 16 * kKept; p < parts; p += 16) weights[p][mine] = weight_of(ml_at[uint64_t(p) * a.tile]) * inv;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    floatx4 acc[kOfLane];
#pragma unroll
    for (uint32_t i = 0; i < kOfLane; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t p0 = first; p0 < parts; p0 += kAtOnce * SHARED) {
        if (p0 != first) ask(p0);
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            const uint32_t p = p0 + u * SHARED;
            if (p >= parts) break;
            const float weight = weights[p][mine];
#pragma unroll
            for (uint32_t i = 0; i < kOfLane; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = __builtin_fmaf(weight, early[u][i][e], acc[i][e]);
        }
    }
    if constexpr (SHARED > 1) {
        if (wave)
#pragma unroll
            for (uint32_t i = 0; i < kOfLane; ++i) lds_acc[wave - 1][i][lane] = acc[i];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (uint32_t w = 0; w + 1 < SHARED; ++w)
#pragma unroll
            for (uint32_t i = 0; i < kOfLane; ++i) acc[i] += lds_acc[w][i][lane];
    }
    const uint32_t v = v0 + mine;
    if (v >= vectors) return;
    const uint32_t row = paged_row_of(a, v), hq = head * a.group + v - row * a.group;
    T *const dst = static_cast<T *>(a.out.data) + uint64_t(span.row0 + row) * a.out.row_stride + hq * a.out.head_stride;
#pragma unroll
    for (uint32_t i = 0; i < kOfLane; ++i) {
        const uint32_t c = (lane / kJoined + 16 * i) * 4;
        if (c >= a.g.head_dim) break;
        Piece<T, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(acc[i][e]);
        if (a.out_on_16) {
            *reinterpret_cast<Piece<T, 4> *>(dst + c) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[c + e] = y.v[e];
        }
    }
}

template <int ELEM, int DP>
void launch_as(const PagedAttn &a, hipStream_t stream) {
    // The wavefronts of a workgroup share their vectors' parts where those are many and the vectors do not fill the device: 16 sequences' 4,096 wavefronts
    // of up to 8 parts 13.6 us shared and 6.8 each for itself.
    const uint32_t waves = a.units * (a.tile / kJoined);
    if (a.units * a.g.kv_heads * 8 <= kPagedTreesGroups && waves * a.g.kv_heads <= 1024)
        launch_kernel(paged_join_kernel<ELEM, DP, 4>, dim3(waves, a.g.kv_heads), kThreads, 0, stream, a);
    else
        launch_kernel(paged_join_kernel<ELEM, DP, 1>, dim3(waves / (kThreads / 64), a.g.kv_heads), kThreads, 0, stream, a);
}
template <int ELEM>
void launch(const PagedAttn &a, hipStream_t stream) {
    const uint32_t dp = paged_padded(a.g.head_dim);
    if (dp == 64)
        launch_as<ELEM, 64>(a, stream);
    else if (dp == 128)
        launch_as<ELEM, 128>(a, stream);
    else
        launch_as<ELEM, 256>(a, stream);
}

// The partials of the kernel of few rows, which lie vector by vector, where rows are drafted trees: some vectors for every compute unit, of a few
// parts each. A wavefront serves a vector (paged_merge.hip gives a workgroup to each: 85 rows of 32 heads of 64 10.8 us, and so 4.6).
template <int ELEM, int DP>
__global__ __launch_bounds__(kThreads) void paged_few_join_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr uint32_t kQuads = DP / 4, kParts = 64 / kQuads, kAtOnce = 8;  // float4s of a partial, and partials that a wavefront takes at once
    paged_fetch_arguments(a);
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    // (Four rows of a head: vectors of all rows and heads would be more threads than a launch has in one dimension, 2^26 vectors on.)
    const uint32_t row = blockIdx.x * (kThreads / 64) + wave, hq = blockIdx.y;
    PagedLine line(a);
    line.cut();
    PagedSpan span;
    if (row >= a.rows || !line.find<PagedLine::kRow>(span, row)) return;
    const uint32_t head = paged_row_of(a, hq), v = (row - span.row0) * a.group + (hq - head * a.group);
    const uint32_t tile = v >> a.tile_shift, local = tile * a.g.kv_heads + head, unit = span.unit0 + local;
    // Slots first .. last of the unit's partials, from slot `unit` on.
    const uint32_t from = span.start + local * span.run, first = from / line.share, last = (from + span.blocks - 1) / line.share;
    if (first == last || last + unit >= a.groups + a.units) return;  // written whole
    const uint32_t parts = last - first + 1;
    const uint64_t base = uint64_t(unit + first) * a.tile + (v - (tile << a.tile_shift));
    const uint32_t quad = lane % kQuads, part = lane / kQuads;
    auto acc_of = [&](uint32_t w) { return *reinterpret_cast<const floatx4 *>(a.ws_acc + (base + uint64_t(w) * a.tile) * DP + quad * 4); };
    floatx4 early[kAtOnce];
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) early[u] = acc_of(min(part + u * kParts, parts - 1));
    // Every lane has every 64th part's maximum and sum; the first ones' stay.
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < parts) ml = a.ws_ml[base + uint64_t(lane) * a.tile];
    float m = ml.x;
    for (uint32_t p = lane + 64; p < parts; p += 64) m = fmaxf(m, a.ws_ml[base + uint64_t(p) * a.tile].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    // (A maximum of minus infinity: nothing visible, a sum of 0, or scores that are no numbers, which the sum then is.)
    auto weight_of = [&](float2 x) { return x.x == -INFINITY ? 0.0f : fast_exp2(x.x - m) * (x.y < 0.0f ? kPagedMergeLift : 1.0f); };
    auto sum_of = [&](float2 x) { return x.x == -INFINITY ? x.y : weight_of(x) * __builtin_fabsf(x.y); };
    float l = sum_of(ml);
    for (uint32_t p = lane + 64; p < parts; p += 64) l += sum_of(a.ws_ml[base + uint64_t(p) * a.tile]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    const float inv = 1.0f / l;
    floatx4 acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t run = 0; run < parts; run += 64) {
        if (run) {
            ml = make_float2(-INFINITY, 0.0f);
            if (run + lane < parts) ml = a.ws_ml[base + uint64_t(run + lane) * a.tile];
        }
        const float share = weight_of(ml) * inv;
        for (uint32_t first_of = 0; first_of < min(64u, parts - run); first_of += kAtOnce * kParts) {
            if (run + first_of) {
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; ++u) early[u] = acc_of(min(run + first_of + part + u * kParts, parts - 1));
            }
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u) {
                const uint32_t w = first_of + part + u * kParts;  // of the run: below 64, or behind the last part
                const float x = __shfl(share, w & 63);
                if (w < 64 && run + w < parts) acc += early[u] * x;
            }
        }
    }
#pragma unroll
    for (uint32_t o = kQuads; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    const uint32_t c = quad * 4;
    if (part || c >= a.g.head_dim) return;
    T *dst = static_cast<T *>(a.out.data) + uint64_t(row) * a.out.row_stride + hq * a.out.head_stride + c;
    Piece<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(acc[e]);
    if (a.out_on_16) {
        *reinterpret_cast<Piece<T, 4> *>(dst) = y;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[e] = y.v[e];
    }
}

template <int ELEM>
void launch_few(const PagedAttn &a, hipStream_t stream) {
    const uint32_t dp = paged_padded(a.g.head_dim), waves = kThreads / 64;
    const dim3 groups((a.rows + waves - 1) / waves, a.g.kv_heads * a.group);
    if (dp == 64)
        launch_kernel(paged_few_join_kernel<ELEM, 64>, groups, kThreads, 0, stream, a);
    else if (dp == 128)
        launch_kernel(paged_few_join_kernel<ELEM, 128>, groups, kThreads, 0, stream, a);
    else
        launch_kernel(paged_few_join_kernel<ELEM, 256>, groups, kThreads, 0, stream, a);
}

}  // namespace

hipError_t launch_paged_few_join(uint32_t elem, const PagedAttn &a, hipStream_t stream) {
    // (One row's or two's vectors would leave most of the device without: a workgroup each.)
    if (uint64_t(a.rows) * a.g.kv_heads * a.group <= 256) return launch_paged_merge(elem, a, stream);
    if (elem == ITAK_ELEM_F32)
        launch_few<ITAK_ELEM_F32>(a, stream);
    else if (elem == ITAK_ELEM_F16)
        launch_few<ITAK_ELEM_F16>(a, stream);
    else
        launch_few<ITAK_ELEM_BF16>(a, stream);
    return hipGetLastError();
}

hipError_t launch_paged_join(uint32_t elem, const PagedAttn &a, hipStream_t stream) {
    if (elem == ITAK_ELEM_F32)
        launch<ITAK_ELEM_F32>(a, stream);
    else if (elem == ITAK_ELEM_F16)
        launch<ITAK_ELEM_F16>(a, stream);
    else
        launch<ITAK_ELEM_BF16>(a, stream);
    return hipGetLastError();
}

}  // namespace itak
