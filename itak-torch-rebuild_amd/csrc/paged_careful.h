// A unit's attention where something in it is not finite.
//
// The kernels multiply whole tiles: a masked key's zero weight meets the key's value row, a query's pieces meet every key, and
// 0 x inf is NaN where the row of a masked key is never read by the definition. That is looked for once, in a unit's result:
// without an infinity or a NaN in its inputs none is NaN, and no infinity comes out other than as it should. A unit that holds
// one is computed again here, row by row and key by key in f32, with nothing read that the row does not see. No speed is asked of it.
#pragma once

#include "paged_mfma.h"

namespace itak {

namespace {

// Vectors v0 + wave, v0 + wave + waves, .. below v_end over the keys [key0, key1): WRITE(vector, run, accumulators of channels
// 64 c + lane, maximum in the log2 domain, sum).
template <int PAGE, int ELEM, int DP, typename W>
__device__ __forceinline__ void paged_careful(const PagedAttn &a, const PagedSpan &span, uint32_t head, uint32_t v0, uint32_t v_end,
                                           uint32_t wave, uint32_t waves, uint32_t key0, uint32_t key1, W write) {
    typedef typename Elem<ELEM>::type T;
    typedef typename Elem<PAGE>::type P;
    constexpr int kRuns = DP / 64;
    const uint32_t lane = __lane_id(), d = a.g.head_dim, page_mask = (1u << a.g.page_shift) - 1;
    const P *const base = reinterpret_cast<const P *>(a.layer_base) + head * a.g.head_stride;
    const uint32_t *ids = a.batch + span.table;
    auto row_of = [&](uint32_t key) { return base + ids[key >> a.g.page_shift] * a.g.page_stride + uint64_t(key & page_mask) * d; };
    for (uint32_t v = v0 + wave; v < v_end; v += waves) {
        const uint32_t row = paged_row_of(a, v), pos = span.position + row;
        const uint32_t lo = max(lowest_visible(pos, a.window, 0), key0), hi = min(pos + 1, key1);
        const T *q = static_cast<const T *>(a.q.data) + uint64_t(span.row0 + row) * a.q.row_stride +
                     (head * a.group + v - row * a.group) * a.q.head_stride;
        auto score = [&](uint32_t key) {
            const P *k = row_of(key);
            float s = 0.0f;
            for (uint32_t c = 0; c < d; ++c) s = __builtin_fmaf(Elem<ELEM>::to_f32(q[c]), Elem<PAGE>::to_f32(k[c]), s);
            return a.cap_log2 != 0.0f ? softcap_of_exp2_arg(s * a.scale_log2, a.cap_log2, 0.0f) : s * a.scale_log2;
        };
        float m = -INFINITY;
        for (uint32_t key = lo + lane; key < hi; key += 64) m = fmaxf(m, score(key));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f, acc[kRuns];
#pragma unroll
        for (int c = 0; c < kRuns; ++c) acc[c] = 0.0f;
        for (uint32_t at = lo; at < hi; at += 64) {
            const float p = at + lane < hi ? fast_exp2(score(at + lane) - ref) : 0.0f;
            sum += p;
            for (uint32_t j = 0; j < min(hi - at, 64u); ++j) {
                const float w = __shfl(p, j);
                const P *value = row_of(at + j) + a.g.side_stride;
#pragma unroll
                for (int c = 0; c < kRuns; ++c)
                    if (64 * c + lane < d) acc[c] = __builtin_fmaf(w, Elem<PAGE>::to_f32(value[64 * c + lane]), acc[c]);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        write(v, acc, m, sum);
    }
}

// What it gives for a vector: out, or its slot of the workspace.
template <int ELEM, int DP>
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
    if (!whole && has_slot && lane == 0) a.ws_ml[slot] = make_float2(m, l);
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
