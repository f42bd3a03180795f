// A unit's attention where something in it is not finite.
//
// The kernels multiply whole tiles: a masked key's zero weight meets the key's value row, a query's pieces meet every key, and
// 0 x inf is NaN where the row of a masked key is never read by the definition. That is looked for once, in a unit's result:
// without an infinity or a NaN in its inputs none is NaN. Over f16 pages no infinity comes out other than as it should either: 2^31
// values up to 2^16 with weights up to 2^15 are 2^62. Values of bf16 end where f32 does, and a sum of them with weights up to 2^15
// may pass that though the mean does not, so infinities are looked for as well. A unit that holds
// one is computed again here, row by row and key by key in f32, with nothing read that the row does not see, and
// so scaled that no sum leaves f32's range.
#pragma once

#include "paged_mfma.h"

namespace itak {

namespace {

__device__ __forceinline__ float lane_of(float x, uint32_t lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}

// Whether a unit is to be computed here: by a sum over what it gave.
template <int PAGE>
__device__ __forceinline__ bool to_be_done_over(float check) {
    return PAGE == ITAK_ELEM_F16 ? check != check : !(__builtin_fabsf(check) < INFINITY);
}

// What comes out is scaled by this: 2^31 values below 2^128 with weights up to 2^-32 stay below 2^127. The factor goes to the values: a
// weight that it made zero would make an infinite value NaN. (Over f16 pages there is no need.)
template <int PAGE>
constexpr float kCarefulScale = PAGE == ITAK_ELEM_F16 ? 1.0f : 1.0f / kPagedMergeLift;

// A wavefront's vectors of v0 .. v_end over the keys [key0, key1): WRITE(vector, accumulators of channels 64 c + lane, maximum in
// the log2 domain, sum), accumulators and sum scaled. kCareful vectors at once, so that a row is fetched once for them, and 64 keys: a lane has the scores
// of one key; then the lanes are channels.
constexpr uint32_t kCareful = 4;
template <int PAGE, int ELEM, int DP, typename W>
__device__ __forceinline__ void paged_careful(const PagedAttn &a, const PagedSpan &span, uint32_t head, uint32_t v0, uint32_t v_end,
                                           uint32_t wave, uint32_t waves, uint32_t key0, uint32_t key1, W write) {
    typedef typename Elem<ELEM>::type T;
    typedef typename Elem<PAGE>::type P;
    constexpr int kRuns = DP / 64;
    constexpr uint32_t kAtOnce = 8;
    const uint32_t lane = __lane_id(), d = a.g.head_dim, page_mask = (1u << a.g.page_shift) - 1;
    const P *const base = reinterpret_cast<const P *>(a.layer_base) + head * a.g.head_stride;
    const uint32_t *ids = a.batch + span.table;
    for (uint32_t v = v0 + wave * kCareful; v < v_end; v += waves * kCareful) {
        uint32_t lo[kCareful], hi[kCareful], from = key1, to = key0;
        float q[kCareful][kRuns], acc[kCareful][kRuns], m[kCareful], sum[kCareful];
#pragma unroll
        for (uint32_t u = 0; u < kCareful; ++u) {
            const uint32_t mine = min(v + u, v_end - 1), row = paged_row_of(a, mine), pos = span.position + row;
            lo[u] = max(lowest_visible(pos, a.window, 0), key0), hi[u] = min(pos + 1, key1);
            if (lo[u] < hi[u]) from = min(from, lo[u]), to = max(to, hi[u]);
            const T *src = static_cast<const T *>(a.q.data) + uint64_t(span.row0 + row) * a.q.row_stride +
                           (head * a.group + mine - row * a.group) * a.q.head_stride;
            m[u] = -INFINITY, sum[u] = 0.0f;
#pragma unroll
            for (int c = 0; c < kRuns; ++c) {
                q[u][c] = 64 * c + lane < d ? Elem<ELEM>::to_f32(src[64 * c + lane]) : 0.0f;
                acc[u][c] = 0.0f;
            }
        }
        for (uint32_t at = from; at < to; at += 64) {
            const uint32_t n = min(to - at, 64u), key = at + min(lane, n - 1);
            const P *const k = base + ids[key >> a.g.page_shift] * a.g.page_stride + uint64_t(key & page_mask) * d;
            float x[kCareful], p[kCareful];
#pragma unroll
            for (uint32_t u = 0; u < kCareful; ++u) x[u] = 0.0f;
#pragma unroll
            for (int c = 0; c < kRuns; ++c)
                for (uint32_t o = 0; o < min(64u, d - min(d, 64u * c)); o += 8) {
                    const Piece<P, 8> y = *reinterpret_cast<const Piece<P, 8> *>(k + 64 * c + o);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (uint32_t u = 0; u < kCareful; ++u)
                            x[u] = __builtin_fmaf(lane_of(q[u][c], o + e), Elem<PAGE>::to_f32(y.v[e]), x[u]);
                }
            bool every = true;  // (vector sees every key of these)
#pragma unroll
            for (uint32_t u = 0; u < kCareful; ++u) {
                every = every && at >= lo[u] && at + n <= hi[u];
                x[u] *= a.scale_log2 * kQueryLift<PAGE, ELEM>;
                if (a.cap_log2 != 0.0f) x[u] = softcapped<true>(x[u], a.cap_log2, 0.0f);
                const bool seen = lane < n && key >= lo[u] && key < hi[u];
                float most = seen ? fmaxf(m[u], x[u]) : m[u];
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
                const float ref = most == -INFINITY ? 0.0f : most;
                const float alpha = m[u] == -INFINITY ? 1.0f : fast_exp2(m[u] - ref);
                p[u] = seen ? fast_exp2(x[u] - ref) : 0.0f;
                m[u] = most;
                sum[u] = __builtin_fmaf(sum[u], alpha, p[u]);
#pragma unroll
                for (int c = 0; c < kRuns; ++c) acc[u][c] *= alpha;
            }
            const uint64_t row_at = reinterpret_cast<uint64_t>(k + a.g.side_stride);
            auto add = [&](uint32_t j, auto keys) {
                constexpr uint32_t kKeys = keys.value;
                float y[kKeys][kRuns];
#pragma unroll
                for (uint32_t t = 0; t < kKeys; ++t) {
                    const uint64_t low = uint32_t(__builtin_amdgcn_readlane(uint32_t(row_at), j + t));
                    const uint64_t high = uint32_t(__builtin_amdgcn_readlane(uint32_t(row_at >> 32), j + t));
                    const P *value = reinterpret_cast<const P *>(high << 32 | low);
#pragma unroll
                    for (int c = 0; c < kRuns; ++c) y[t][c] = 64 * c + lane < d ? Elem<PAGE>::to_f32(value[64 * c + lane]) * kCarefulScale<PAGE> : 0.0f;
                }
#pragma unroll
                for (uint32_t t = 0; t < kKeys; ++t)
#pragma unroll
                    for (uint32_t u = 0; u < kCareful; ++u)
                        if (kKeys > 1 || (at + j >= lo[u] && at + j < hi[u]))
#pragma unroll
                            for (int c = 0; c < kRuns; ++c) acc[u][c] = __builtin_fmaf(lane_of(p[u], j + t), y[t][c], acc[u][c]);
            };
            uint32_t j = 0;
            if (every)
                for (; j + kAtOnce <= n; j += kAtOnce) add(j, std::integral_constant<uint32_t, kAtOnce>{});
            for (; j < n; ++j) add(j, std::integral_constant<uint32_t, 1>{});
        }
#pragma unroll
        for (uint32_t u = 0; u < kCareful; ++u) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum[u] += __shfl_xor(sum[u], o);
            if (v + u < v_end) write(v + u, acc[u], m[u], sum[u] * kCarefulScale<PAGE>);
        }
    }
}

// What it gives for a vector: out, or its slot of the workspace, where a negative sum says that the part is scaled. (The maximum cannot say so: raised
// by 32 it would lose bits, of scores from 2^29 on all of the 32.)
template <int PAGE, int ELEM, int DP>
__device__ __forceinline__ void paged_write_careful(const PagedAttn &a, const PagedSpan &span, uint32_t head, uint32_t v, bool whole,
                                                    uint64_t slot, bool has_slot, const float (&acc)[DP / 64], float m, float l) {
    typedef typename Elem<ELEM>::type T;
    const uint32_t lane = __lane_id(), row = paged_row_of(a, v);
    T *dst = static_cast<T *>(a.out.data) + uint64_t(span.row0 + row) * a.out.row_stride +
             (head * a.group + v - row * a.group) * a.out.head_stride;
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
        if (64 * c + lane >= a.g.head_dim) continue;
        if (whole)
            dst[64 * c + lane] = Elem<ELEM>::from_f32(acc[c] / l);
        else if (has_slot)
            a.ws_acc[slot * DP + 64 * c + lane] = acc[c];
    }
    if (!whole && has_slot && lane == 0) a.ws_ml[slot] = make_float2(m, kCarefulScale<PAGE> == 1.0f ? l : -l);
}

// Whether any of a workgroup's threads says so; all of them ask.
__device__ __forceinline__ bool any_of_group(bool mine, uint32_t *lds_word) {
    if (threadIdx.x == 0) *lds_word = 0;
    __syncthreads();
    if (mine) *lds_word = 1;
    __syncthreads();
    return *lds_word != 0;
}

}  // namespace

}  // namespace itak
