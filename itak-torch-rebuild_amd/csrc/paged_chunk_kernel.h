// Attention of many rows over pages: prompt chunks and long blocks, tiles of 128 or 256 query vectors.
//
// 4 d operations a pair of vector and position on the matrix pipe against an exponential, a multiply-add, half a maximum and a
// conversion of it: the two are of one length, and what bounds the kernel is how far they run beside each other.
//
// A workgroup of four wavefronts owns a tile of one KV head; each wavefront keeps 32 * COLS of its vectors, queries and
// accumulators in registers, and all four walk the tile's keys together in blocks of 32 that lie in LDS. Per block
//   S^T = K . Q^T, softmax in the lane's own column, O^T += V^T . P^T       (v_mfma_f32_32x32x16)
// with S^T's rows dealt so that P stays in the registers the scores came in: a lane holds keys 16m + 8u + 4h + e (h = lane / 32) and
// so must the product's other operand. That one is V row by row as the page has it, turned over on the way out of LDS
// (ds_read_b64_tr_b16: sixteen lanes read four rows of sixteen channels and each gets four keys of one channel).
// 64 vectors a wavefront read each block from LDS for 32 bytes a MFMA; with 32, LDS would be as busy as the matrix pipe.
//
// Blocks travel from the pages to LDS without passing through registers (global_load_lds_dwordx4: lane i's 16 bytes go to
// M0 + 16 i) into a ring of stages, whole rows at a time; the 16-byte pieces of a row are shuffled by the row's number on the way (the source
// address is free per lane), so that neither the operand reads of K nor the turning reads of V meet a bank twice. A
// load covers rows of one half of a block only, and pages hold at least 16 rows: its page is one scalar load, a block ahead.
//
// The maximum is a reference that moves only when a score passes it by 2^8 (see the kernel of few rows).
#pragma once

#include "paged_careful.h"

namespace itak {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

constexpr int kChunkWaves = 4;
constexpr float kChunkSlack = 8.0f;

template <int PAGE>
__device__ __forceinline__ floatx16 mfma_32x32x16(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (PAGE == ITAK_ELEM_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
}

// Issued from assembly: the compiler then neither waits for such a load at every LDS read nor needs to, because its only
// consumer is ordered by the wait and the barrier at the top of each block.
__device__ __forceinline__ void page_to_lds(uint64_t base, uint32_t offset, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ void lane_to_lds(uint64_t address, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(address), "s"(lds_addr) : "memory");
}
template <int n>
__device__ __forceinline__ void wait_loads() {  // s_waitcnt vmcnt(n), other counters untouched
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | ((n >> 4) << 14));
}

// Sub-blocks of 32 keys a stage of the ring holds, and stages.
constexpr int chunk_subs(int dp) { return dp <= 128 ? 2 : 1; }
constexpr int chunk_stages(int dp) { return dp == 256 ? 4 : 4; }
constexpr size_t chunk_lds(int dp) { return size_t(chunk_stages(dp)) * chunk_subs(dp) * 2 * 32 * 2 * dp; }

template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP, int COLS, int GROUPS, bool CAP>
__global__ __launch_bounds__(kChunkWaves * 64, GROUPS) void paged_chunk_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr int kTile = kChunkWaves * 32 * COLS;
    constexpr int kSteps = DP / 16;               // products of a score tile
    constexpr int kOut = DP / 32;                 // output tiles of 32 channels
    constexpr int kRowBytes = 2 * DP;
    constexpr int kBlockBytes = 32 * kRowBytes;   // of one side of a sub-block
    constexpr int kSubBytes = 2 * kBlockBytes;
    constexpr int kSubs = chunk_subs(DP), kStages = chunk_stages(DP), kStageBytes = kSubs * kSubBytes;
    constexpr int kRowPieces = DP / 8;            // 16-byte pieces of a row
    constexpr int kLoadRows = 512 / DP;           // rows a load of one wavefront moves
    constexpr int kLoads = DP / 64;               // loads a wavefront issues for a side of a sub-block
    constexpr int kStageLoads = 2 * kLoads * kSubs;
    extern __shared__ __attribute__((aligned(16))) unsigned char ring[];
    __shared__ uint32_t lds_flag;

    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t h = lane >> 5, j = lane & 31;
    const uint32_t d = EXACT ? DP : a.g.head_dim;

    // Which tile of which head of which item, and which part of its keys. Parts come slowest and heads fastest: workgroup w runs on
    // compute die w mod 8, so a die keeps to the keys of few heads, and the tiles that run at a time read them together. Longest first.
    const uint32_t units = gridDim.x / a.parts;
    const uint32_t part = blockIdx.x / units, unit = blockIdx.x - part * units;
    const PagedLine line(a);
    PagedSpan span;
    if (!line.find(span, [=](const PagedSpan &s, uint32_t) { return unit >= s.unit0 && unit - s.unit0 < s.tiles * a.g.kv_heads; })) return;
    const uint32_t local = unit - span.unit0, turn = local / a.g.kv_heads, head = local - turn * a.g.kv_heads;
    const uint32_t tile = span.tiles - 1 - turn;
    const uint32_t length = span.position + span.rows;
    const uint32_t vectors = span.rows * a.group, v0 = tile * kTile;
    // Keys the tile's rows see, and this workgroup's blocks of them.
    const uint32_t first_row = v0 / a.group, last_row = min((v0 + kTile - 1) / a.group, span.rows - 1);
    const uint32_t tile_lo = lowest_visible(span.position + first_row, a.window, 0), tile_hi = span.position + last_row + 1;
    const uint32_t b_first = tile_lo / 32, b_all = (tile_hi + 31) / 32 - b_first, b_part = (b_all + a.parts - 1) / a.parts;
    const uint32_t kb0 = b_first + min(b_all, part * b_part), kb_end = b_first + min(b_all, part * b_part + b_part);
    const uint64_t slot0 = uint64_t(unit * a.parts + part) * kTile;

    // Of this wavefront's vectors: positions some, and positions all of its rows see.
    const uint32_t wv0 = v0 + wave * 32 * COLS;
    const uint32_t w_first = min(wv0 / a.group, span.rows - 1), w_last = min((wv0 + 32 * COLS - 1) / a.group, span.rows - 1);
    const bool active = wv0 < vectors;
    const uint32_t some_lo = lowest_visible(span.position + w_first, a.window, 0), some_hi = active ? span.position + w_last + 1 : 0;
    const uint32_t every_lo = lowest_visible(span.position + w_last, a.window, 0), every_hi = span.position + w_first + 1;

    // Loads: piece `lane` of a load is row lane / kRowPieces of its rows, 16-byte place lane % kRowPieces. The place holds the piece
    // place ^ (the row's shuffle): of keys, so that 16 rows' pieces of one number lie in 16 different places modulo 256 bytes;
    // of values, so that four rows' 64 bytes of one number lie in four.
    const uint32_t l_row = lane / kRowPieces, l_place = lane % kRowPieces;
    auto k_shuffle = [](uint32_t row) { return DP == 64 ? (row >> 1) & 7 : row & 15; };
    auto v_shuffle = [](uint32_t row) { return DP == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); };
    uint32_t k_src[kLoads], v_src[kLoads];  // bytes from the half block's first row
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t row = (wave + 4 * i) * kLoadRows + l_row;
        const uint32_t kp = l_place ^ k_shuffle(row), vp = l_place ^ v_shuffle(row);
        k_src[i] = (row & 15) * d * 2 + kp * 16;
        v_src[i] = (row & 15) * d * 2 + vp * 16;
        if (!EXACT && kp * 8 >= d) k_src[i] = ~0u;  // (zeros)
        if (!EXACT && vp * 8 >= d) v_src[i] = ~0u;
    }
    const uint32_t ring_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)ring;
    typedef const __attribute__((address_space(4))) uint32_t *ScalarIds;
    const ScalarIds ids = (ScalarIds)(uintptr_t)(a.batch + span.table);
    const uint32_t last_page = (length - 1) >> a.g.page_shift, page_mask = (1u << a.g.page_shift) - 1;
    const uint64_t head_base = reinterpret_cast<uint64_t>(a.layer_base + head * a.g.head_stride);
    const uint64_t side_bytes = 2 * a.g.side_stride;
    struct Pages {
        uint32_t id[2];
    };
    auto pages_of = [&](uint32_t kb) {
        Pages p;
        p.id[0] = ids[min((32 * kb) >> a.g.page_shift, last_page)];
        p.id[1] = ids[min((32 * kb + 16) >> a.g.page_shift, last_page)];
        return p;
    };
    // Block kb to its place in the ring. Past the end the last block comes once more: the loads in flight stay the same.
    auto issue = [&](uint32_t kb, uint32_t place, const Pages &pages) {
        const uint32_t at = min(kb, max(kb_end, kb0 + 1) - 1);
        uint64_t base[2];
#pragma unroll
        for (int half = 0; half < 2; ++half)
            base[half] = head_base + pages.id[half] * a.g.page_stride * 2 + uint64_t((32 * at + 16 * half) & page_mask) * (d * 2);
        const uint32_t dst = ring_base + place + wave * 1024;
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                // (The half a load's rows lie in, the same for all of its lanes.)
                const uint32_t half = DP == 64 ? wave >> 1 : DP == 128 ? uint32_t(i) : uint32_t(i) >> 1;
                const uint64_t from = (half ? base[1] : base[0]) + (side ? side_bytes : 0);
                const uint32_t off = side ? v_src[i] : k_src[i];
                const uint32_t to = dst + side * kBlockBytes + i * 4096;
                if constexpr (EXACT)
                    page_to_lds(from, off, to);
                else
                    lane_to_lds(off == ~0u ? reinterpret_cast<uint64_t>(a.zeros) : from + off, to);
            }
    };

    // The queries as B operands: column j, channels 16 s + 8 h .. + 7.
    u32x4 q[COLS][NQ][kSteps];
    uint32_t my_pos[COLS], my_lo[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const uint32_t v = wv0 + 32 * c + j;
        const uint32_t row = min(v / a.group, span.rows - 1);
        const uint32_t hq = head * a.group + (v < vectors ? v - row * a.group : 0);
        my_pos[c] = span.position + row;
        my_lo[c] = lowest_visible(my_pos[c], a.window, 0);
        const T *src = static_cast<const T *>(a.q.data) + uint64_t(span.row0 + row) * a.q.row_stride + hq * a.q.head_stride;
        typename QueryRaw<ELEM>::type raw[kSteps];
        if (a.q_on_16) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                raw[s] = load_query<ELEM, true>(src + (EXACT || 16 * s + 8 * h < d ? 16 * s + 8 * h : 0));
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                raw[s] = load_query<ELEM, false>(src + (EXACT || 16 * s + 8 * h < d ? 16 * s + 8 * h : 0));
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
            split_query<PAGE, ELEM, NQ>(raw[s], v < vectors && (EXACT || 16 * s + 8 * h < d),
                                        [&](int n, u32x4 x) { q[c][n][s] = x; });
    }
    // (The compiler cannot count the ring's loads: every load of its own has to be in before the first of them.)
    wait_loads<0>();

    // Where the operands lie in a stage: K row j, piece 2 s + h at ((2 s + h) ^ shuffle) = place0 ^ 2 s; V row 4 h + (lane & 15) / 4
    // (of the four of 16 m + 8 u + ..), channels 32 t + 16 (lane / 16 % 2) + 4 (lane % 4) on.
    const uint32_t k_at = j * kRowBytes + ((h ^ k_shuffle(j)) * 16);
    const uint32_t tr_row = 4 * h + ((lane & 15) >> 2);
    const uint32_t v_at = kBlockBytes + tr_row * kRowBytes + ((v_shuffle(tr_row) * 16) ^ (((lane >> 4) & 1) * 32 + (lane & 3) * 8));

    float ref[COLS], threshold[COLS], sum[COLS];
    floatx16 o[COLS][kOut];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        ref[c] = 0.0f, threshold[c] = -INFINITY, sum[c] = 0.0f;
#pragma unroll
        for (int t = 0; t < kOut; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][t][r] = 0.0f;
    }

    // Operands out of a sub-block at LDS address `at`.
    auto k_operand = [&](uint32_t at, int i) {
        return *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>((uintptr_t)(at + (k_at ^ (i * 32))));
    };
    auto v_operand = [&](uint32_t at, int t, int m) {
        u32x4 v;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4 *)(uintptr_t)(at + (v_at ^ (t * 64)) + (16 * m + 8 * u) * kRowBytes));
            const uint2 y = __builtin_bit_cast(uint2, x);
            v[2 * u] = y.x, v[2 * u + 1] = y.y;
        }
        return v;
    };
    // A lane's scores of a block, relative to the reference, and the largest of a column.
    float x[COLS][16];
    auto scaled = [&](float s, int c) {
        if constexpr (CAP)
            return softcap_of_exp2_arg(s * a.scale_log2, a.cap_log2, ref[c]);
        else
            return __builtin_fmaf(s, a.scale_log2, -ref[c]);
    };
    // Masks the scores of block kb where a row does not see all of it, and moves references that they pass.
    auto settle = [&](uint32_t kb, float (&most)[COLS]) {
        if (32 * kb < every_lo || 32 * kb + 32 > every_hi) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                most[c] = -INFINITY;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t key = 32 * kb + 8 * (r / 4) + 4 * h + r % 4;
                    if (key > my_pos[c] || key < my_lo[c]) x[c][r] = -INFINITY;
                    most[c] = fmaxf(most[c], x[c][r]);
                }
            }
        }
        bool over = false;
#pragma unroll
        for (int c = 0; c < COLS; ++c) over = over || most[c] > threshold[c];
        if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(most[c]), __float_as_uint(most[c]), false, false);
                const float m = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                const bool live = threshold[c] != -INFINITY;
                float delta = live ? fmaxf(m, 0.0f) : m;
                if (m == -INFINITY) delta = 0.0f;
                const float alpha = live ? fast_exp2(-delta) : 1.0f;
                ref[c] += delta;
                if (m != -INFINITY) threshold[c] = kChunkSlack;
                sum[c] *= alpha;
#pragma unroll
                for (int t = 0; t < kOut; ++t) o[c][t] *= alpha;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[c][r] -= delta;
            }
        }
    };
    // Rows of block kb no query of the tile sees may hold anything: their values are zeroed in LDS, where the block lies at `at`.
    auto clear = [&](uint32_t kb, uint32_t at) {
        for (uint32_t p = tid; p < 32 * kRowPieces; p += kChunkWaves * 64) {
            const uint32_t key = 32 * kb + p / kRowPieces;
            if (key < tile_lo || key >= tile_hi)
                *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(at + kBlockBytes + p * 16)) = u32x4{0, 0, 0, 0};
        }
    };
    // The blocks of a stage that have such rows: at most the tile's first and last, and what comes past the end in their stage.
    auto clear_stage = [&](uint32_t kb, uint32_t at) {
        bool any = false;
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
            if (32 * (kb + u) < tile_lo || 32 * (kb + u) + 32 > tile_hi) clear(kb + u, at + u * kSubBytes), any = true;
        if (any) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        }
    };

    // Stages of the ring fill ahead of the one at hand; its last places are never read where the blocks end inside one.
    const uint32_t stages = (kb_end - kb0 + kSubs - 1) / kSubs;
    Pages ahead[kSubs];
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
#pragma unroll
        for (int u = 0; u < kSubs; ++u) issue(kb0 + s * kSubs + u, s * kStageBytes + u * kSubBytes, pages_of(kb0 + s * kSubs + u));
#pragma unroll
    for (int u = 0; u < kSubs; ++u) ahead[u] = pages_of(kb0 + (kStages - 1) * kSubs + u);
    u32x4 k[kSteps];
    if (stages) {
        // The first block's scores by themselves, and the operands of the second block's.
        wait_loads<kStageLoads * (kStages - 2)>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        clear_stage(kb0, ring_base);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) k[i] = k_operand(ring_base, i);
        float most[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            floatx16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int n = 0; n < NQ; ++n) s = mfma_32x32x16<PAGE>(k[i], q[c][n][i], s);
            most[c] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[c][r] = scaled(s[r], c), most[c] = fmaxf(most[c], x[c][r]);
        }
        settle(kb0, most);
        if constexpr (kSubs > 1) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) k[i] = k_operand(ring_base + kSubBytes, i);
        }
    }
    uint32_t at = ring_base, next = ring_base + kStageBytes, free_at = (kStages - 1) * kStageBytes;
    for (uint32_t g = 0; g < stages; ++g) {
        // This wavefront's loads of the next stage have landed (those of the stages behind it may still fly); behind the barrier
        // everybody's have, and everybody is done with the stage before this one, which the loads that go out now overwrite.
        wait_loads<kStageLoads * (kStages - 3)>();
        __builtin_amdgcn_s_barrier();
        const uint32_t kb = kb0 + g * kSubs;
#pragma unroll
        for (int u = 0; u < kSubs; ++u) issue(kb + (kStages - 1) * kSubs + u, free_at + u * kSubBytes, ahead[u]);
#pragma unroll
        for (int u = 0; u < kSubs; ++u) ahead[u] = pages_of(kb + kStages * kSubs + u);
        clear_stage(kb + kSubs, next);
        if constexpr (kSubs == 1) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) k[i] = k_operand(next, i);
        }
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
            const uint32_t here = at + u * kSubBytes;
            // Where the operands of the scores after the next lie.
            const uint32_t k_next = u + 2 < kSubs ? at + (u + 2) * kSubBytes : next + (u + 2 - kSubs) * kSubBytes;
            // Three stretches, each of products beside vector work of about their length: the next block's scores beside three quarters
            // of this block's exponentials, the first half of P.V beside the rest, the second half beside the next scores' scaling.
            constexpr int kAll = 16 * COLS, kFirst = kAll * 3 / 4;
            floatx16 s[COLS];
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[c][r] = 0.0f;
            u32x4 p[COLS][NP][2];
            u32x4 v[kOut][2];
            auto weigh = [&](int e) {  // exponential e: halves of the keys, columns, keys
                const int m = e / (8 * COLS), c = e / 8 % COLS, r = 8 * m + e % 8;
                x[c][r] = fast_exp2(x[c][r]);
                if (e % 8 == 7) {
                    float w[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) w[y] = x[c][8 * m + y];
                    sum[c] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                    u32x4 pieces[NP];
                    split_8<PAGE, NP>(w, pieces);
#pragma unroll
                    for (int n = 0; n < NP; ++n) p[c][n][m] = pieces[n];
                }
            };
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int c = 0; c < COLS; ++c)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) s[c] = mfma_32x32x16<PAGE>(k[i], q[c][n][i], s[c]);
#pragma unroll
                for (int e = i * kFirst / kSteps; e < (i + 1) * kFirst / kSteps; ++e) weigh(e);
                if (i >= kSteps - 2 * kOut) v[(i - (kSteps - 2 * kOut)) % kOut][(i - (kSteps - 2 * kOut)) / kOut] =
                    v_operand(here, (i - (kSteps - 2 * kOut)) % kOut, (i - (kSteps - 2 * kOut)) / kOut);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
#pragma unroll
                for (int c = 0; c < COLS; ++c)
#pragma unroll
                    for (int n = 0; n < NP; ++n) o[c][t] = mfma_32x32x16<PAGE>(v[t][0], p[c][n][0], o[c][t]);
#pragma unroll
                for (int e = kFirst + t * (kAll - kFirst) / kOut; e < kFirst + (t + 1) * (kAll - kFirst) / kOut; ++e) weigh(e);
                if (kSubs > 1) {
                    k[2 * t] = k_operand(k_next, 2 * t);
                    k[2 * t + 1] = k_operand(k_next, 2 * t + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            float most[COLS];
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
#pragma unroll
                for (int c = 0; c < COLS; ++c)
#pragma unroll
                    for (int n = 0; n < NP; ++n) o[c][t] = mfma_32x32x16<PAGE>(v[t][1], p[c][n][1], o[c][t]);
#pragma unroll
                for (int e = t * kAll / kOut; e < (t + 1) * kAll / kOut; ++e) {
                    const int c = e / 16, r = e % 16;
                    x[c][r] = scaled(s[c][r], c);
                    if (r == 0)
                        most[c] = x[c][0];
                    else if (r % 2 == 0)
                        most[c] = max3(most[c], x[c][r - 1], x[c][r]);
                    else if (r == 15)
                        most[c] = fmaxf(most[c], x[c][15]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (kb + u + 1 < kb_end) settle(kb + u + 1, most);
            if (kb + u + 1 >= kb_end) break;
        }
        const uint32_t was = at;
        at = next;
        free_at = was - ring_base;
        next = next + kStageBytes == ring_base + kStages * kStageBytes ? ring_base : next + kStageBytes;
    }
    wait_loads<0>();  // (the surplus loads)

    // A lane holds of its column channels 32 t + 8 (r / 4) + 4 h + r % 4.
    const bool whole = a.parts == 1;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[c]), __float_as_uint(sum[c]), false, false);
        const float l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
        const uint32_t v = wv0 + 32 * c + j;
        if (v >= vectors) continue;
        float check = l;
#pragma unroll
        for (int t = 0; t < kOut; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) check += EXACT || 32u * t + 8 * (r / 4) + 4 * h < d ? o[c][t][r] : 0.0f;
        bad = bad || check != check;
        if (whole) {
            const float inv = 1.0f / l;
            const uint32_t row = v / a.group, hq = head * a.group + v - row * a.group;
            T *dst = static_cast<T *>(a.out.data) + uint64_t(span.row0 + row) * a.out.row_stride + hq * a.out.head_stride;
            typedef Piece<T, 4> Four;
#pragma unroll
            for (int t = 0; t < kOut; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const uint32_t ch = 32 * t + 2 * r + 4 * h;
                    if (!EXACT && ch >= d) continue;
                    Four y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(o[c][t][r + e] * inv);
                    if (a.out_on_16) {
                        *reinterpret_cast<Four *>(dst + ch) = y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) dst[ch + e] = y.v[e];
                    }
                }
        } else {
            const uint64_t slot = slot0 + (v - v0);
#pragma unroll
            for (int t = 0; t < kOut; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<floatx4 *>(a.ws_acc + slot * DP + 32 * t + 2 * r + 4 * h) =
                        floatx4{o[c][t][r], o[c][t][r + 1], o[c][t][r + 2], o[c][t][r + 3]};
            if (h == 0) a.ws_ml[slot] = make_float2(threshold[c] == -INFINITY ? -INFINITY : ref[c], l);
        }
    }
    if (any_of_group(bad, &lds_flag))
        paged_careful<PAGE, ELEM, DP>(a, span, head, v0, min(v0 + kTile, vectors), wave, kChunkWaves, 32 * kb0, 32 * kb_end,
                                      [&](uint32_t v, const float (&acc)[DP / 64], float m, float l) {
                                          paged_write_careful<ELEM, DP>(a, span, head, v, whole, slot0 + v - v0, true, acc, m, l);
                                      });
}

template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP>
hipError_t launch_chunk_as(const PagedAttn &a, hipStream_t stream) {
    if constexpr (!paged_chunk_takes(DP, PAGE, ELEM)) return hipErrorInvalidValue;
    else {
    constexpr int kCols = int(paged_chunk_tile(DP, ELEM)) / (kChunkWaves * 32);
    constexpr int kGroups = DP == 64 ? 2 : 1;
    auto run = [&](auto kernel) {
        static const hipError_t granted =
            hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(chunk_lds(DP)));
        if (granted != hipSuccess) return granted;
        launch_kernel(kernel, a.units * a.parts, kChunkWaves * 64, chunk_lds(DP), stream, a);
        return hipGetLastError();
    };
    return a.cap_log2 != 0.0f ? run(paged_chunk_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, kCols, kGroups, true>)
                              : run(paged_chunk_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, kCols, kGroups, false>);
    }
}
template <int PAGE, int ELEM, int NQ, int NP>
hipError_t launch_chunk(const PagedAttn &a, hipStream_t stream) {
    const uint32_t d = a.g.head_dim;
    return d == 64    ? launch_chunk_as<PAGE, ELEM, 64, true, NQ, NP>(a, stream)
           : d < 64   ? launch_chunk_as<PAGE, ELEM, 64, false, NQ, NP>(a, stream)
           : d == 128 ? launch_chunk_as<PAGE, ELEM, 128, true, NQ, NP>(a, stream)
           : d < 128  ? launch_chunk_as<PAGE, ELEM, 128, false, NQ, NP>(a, stream)
           : d == 256 ? launch_chunk_as<PAGE, ELEM, 256, true, NQ, NP>(a, stream)
                      : launch_chunk_as<PAGE, ELEM, 256, false, NQ, NP>(a, stream);
}

}  // namespace

}  // namespace itak
