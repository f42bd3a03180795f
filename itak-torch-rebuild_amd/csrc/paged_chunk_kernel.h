// Attention of many rows over pages: prompt chunks and long blocks, tiles of 128 or 256 query vectors.
//
// 4 d operations a pair of vector and position on the matrix pipe against an exponential, a multiply-add, half a maximum and a
// conversion of it: the two are of one length, and what bounds the kernel is how far they run beside each other.
//
// A workgroup of eight wavefronts (four of f32 tensors and of 256 channels) owns a tile of one KV head; each wavefront keeps 32 of its
// vectors, queries and accumulators in registers, and all walk the tile's keys together in blocks of 32 that lie in LDS. Per block
//   S^T = K . Q^T, softmax in the lane's own column, O^T += V^T . P^T       (v_mfma_f32_32x32x16)
// with S^T's rows dealt so that P stays in the registers the scores came in: a lane holds keys 16m + 8u + 4h + e (h = lane / 32) and
// so must the product's other operand. That one is V row by row as the page has it, turned over on the way out of LDS
// (ds_read_b64_tr_b16: sixteen lanes read four rows of sixteen channels and each gets four keys of one channel).
// The next block's scores are multiplied beside this block's exponentials, and this block's P.V beside the next one's maximum.
// 32 vectors a wavefront and two wavefronts a SIMD, which fill each other's gaps: 64 vectors and one wavefront read half as much from LDS
// and took 1,035 us where these took 959 to 980 on the same devices and take up to 1,000 on others (2,048 rows by 32 heads over 30,720 and
// themselves, 128 channels, f16: 1.07 TFLOP, 1.07 to 1.11 PFLOP/s, where a library product of 8,192 cubed reaches 1.14). The matrix pipe is busy 64 % of the time at the 1.77 GHz that the
// power leaves it; without its LDS reads and loads the loop would take some 800 us. f32 tensors are products times pieces: over f16 two by two,
// 1,865 us (two times a library product's time are 1,880), over bf16 three by three, 2,510 us.
//
// Blocks travel from the pages to LDS without passing through registers (global_load_lds_dwordx4: lane i's 16 bytes go to
// M0 + 16 i) into a ring of stages, whole rows at a time; the 16-byte pieces of a row are shuffled by the row's number on the way (the source
// address is free per lane), so that neither the operand reads of K nor the turning reads of V meet a bank twice. A
// load covers rows of one half of a block only, and pages hold at least 16 rows: it has one page, looked up 64 blocks at a time.
//
// The maximum is a reference that moves only when a score passes it by far (kWeightMost).
#pragma once

#include "lds_grant.h"
#include "paged_careful.h"

namespace itak {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

template <int PAGE>
__device__ __forceinline__ floatx16 mfma_32x32x16(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (PAGE == ITAK_ELEM_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
}

// Issued from assembly: the compiler then neither waits for such a load at every LDS read nor needs to, because its only
// consumer is ordered by the wait and the barrier at the top of each block. It does not look for hazards in there either: a scalar
// register that vector code wrote (readlane: the address) takes five wait states before a load may read it, m0 one.
__device__ __forceinline__ void page_to_lds(uint64_t base, uint32_t offset, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_addr) : "memory");
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
constexpr int kChunkStages = 4;
constexpr size_t chunk_lds(int dp) { return size_t(kChunkStages) * chunk_subs(dp) * 2 * 32 * 2 * dp; }

// Scores without a cap, capped by the short form, capped by the series (paged_cap_by_series).
enum ChunkCap { kNoCap, kShortCap, kSeriesCap };
template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP, ChunkCap CAP>
__global__ __launch_bounds__(paged_chunk_waves(DP, ELEM) * 64) void paged_chunk_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr int kWaves = paged_chunk_waves(DP, ELEM);
    constexpr int kTile = kWaves * 32;
    constexpr int kSteps = DP / 16;               // products of a score tile
    constexpr int kOut = DP / 32;                 // output tiles of 32 channels
    constexpr int kRowBytes = 2 * DP;
    constexpr int kBlockBytes = 32 * kRowBytes;   // of one side of a sub-block
    constexpr int kSubBytes = 2 * kBlockBytes;
    constexpr int kSubs = chunk_subs(DP), kStages = kChunkStages, kStageBytes = kSubs * kSubBytes;
    constexpr int kRowPieces = DP / 8;            // 16-byte pieces of a row
    constexpr int kLoadRows = 512 / DP;           // rows a load of one wavefront moves
    constexpr int kSideLoads = DP / 16;           // loads of a side of a sub-block, dealt to the wavefronts in turn
    constexpr int kLoads = 2 * kSideLoads / kWaves; // loads of a wavefront for a sub-block, both sides
    constexpr int kStageLoads = kLoads * kSubs;
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
    if (!line.find<PagedLine::kUnit>(span, unit)) return;
    const uint32_t local = unit - span.unit0, turn = local / a.g.kv_heads, head = local - turn * a.g.kv_heads;
    const uint32_t tile = span.tiles - 1 - turn;
    const uint32_t length = span.position + span.rows;
    const uint32_t vectors = span.rows * a.group, v0 = tile * kTile;
    // Keys the tile's rows see, and this workgroup's blocks of them.
    const uint32_t first_row = paged_row_of(a, v0), last_row = min(paged_row_of(a, v0 + kTile - 1), span.rows - 1);
    const uint32_t tile_lo = lowest_visible(span.position + first_row, a.window, 0), tile_hi = span.position + last_row + 1;
    const uint32_t b_first = tile_lo / 32, b_all = (tile_hi + 31) / 32 - b_first, b_part = (b_all + a.parts - 1) / a.parts;
    const uint32_t kb0 = b_first + min(b_all, part * b_part), kb_end = b_first + min(b_all, part * b_part + b_part);
    const uint64_t slot0 = uint64_t(unit * a.parts + part) * kTile;

    // Positions all of this wavefront's rows see.
    const uint32_t wv0 = v0 + wave * 32;
    const uint32_t w_first = min(paged_row_of(a, wv0), span.rows - 1), w_last = min(paged_row_of(a, wv0 + 31), span.rows - 1);
    const uint32_t every_lo = lowest_visible(span.position + w_last, a.window, 0), every_hi = span.position + w_first + 1;
    // Blocks all of which they all see: from inner0 on, `inner` of them.
    const uint32_t inner0 = __builtin_amdgcn_readfirstlane((every_lo + 31) / 32);
    const uint32_t inner = __builtin_amdgcn_readfirstlane(every_hi / 32 > inner0 ? every_hi / 32 - inner0 : 0);

    // Loads: piece `lane` of a load is row lane / kRowPieces of its rows, 16-byte place lane % kRowPieces. The place holds the piece
    // place ^ (the row's shuffle): of keys, so that 16 rows' pieces of one number lie in 16 different places modulo 256 bytes;
    // of values, so that four rows' 64 bytes of one number lie in four.
    const uint32_t l_row = lane / kRowPieces, l_place = lane % kRowPieces;
    auto k_shuffle = [](uint32_t row) { return DP == 64 ? (row >> 1) & 7 : row & 15; };
    auto v_shuffle = [](uint32_t row) { return DP == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); };
    // Load i of this wavefront: which side, and which of its loads. (The rows of a load lie in one half of the block.)
    auto side_of = [&](int i) { return kSideLoads >= kWaves ? uint32_t(i / (kSideLoads / kWaves)) : wave / kSideLoads; };
    auto load_of = [&](int i) { return kSideLoads >= kWaves ? wave + kWaves * (i % (kSideLoads / kWaves)) : wave % kSideLoads; };
    auto half_of = [&](int i) {
        constexpr int kHalf = 16 / kLoadRows;  // loads of a half of a side
        return kSideLoads > kWaves || kWaves == 4 ? uint32_t(kWaves * (i % (kSideLoads / kWaves)) / kHalf) : load_of(i) / kHalf;
    };
    uint32_t src[kLoads];  // bytes from the half block's first row
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t row = load_of(i) * kLoadRows + l_row;
        const uint32_t piece = l_place ^ (side_of(i) ? v_shuffle(row) : k_shuffle(row));
        src[i] = (row & 15) * d * 2 + piece * 16;
        if (!EXACT && piece * 8 >= d) src[i] = ~0u;  // (zeros)
    }
    const uint32_t ring_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)ring;
    const uint32_t last_page = (length - 1) >> a.g.page_shift, page_mask = (1u << a.g.page_shift) - 1;
    const uint64_t head_base = reinterpret_cast<uint64_t>(a.layer_base + head * a.g.head_stride);
    const uint32_t page_bytes = uint32_t(2 * a.g.page_stride), side_bytes = uint32_t(2 * a.g.side_stride);
    // Where the next 64 blocks' halves begin, a block a lane: worked out by vector code every 64 blocks and read lane by lane, where a
    // scalar load and some sixteen scalar instructions a block would each cost the wavefront an issue slot. A wavefront's loads lie in
    // one half of a block where it has one or two of them, else in both. (Positions past the end are clamped to the last page: any row of it may be read.)
    constexpr bool kBothHalves = kLoads > 2;
    uint64_t begins[kBothHalves ? 2 : 1];
    auto look_up = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < (kBothHalves ? 2 : 1); ++i) {
            const uint32_t key = 32 * (kb + lane) + 16 * (kBothHalves ? uint32_t(i) : half_of(0));
            const uint32_t id = a.batch[span.table + min(key >> a.g.page_shift, last_page)];
            begins[i] = head_base + uint64_t(id) * page_bytes + (key & page_mask) * (d * 2);
        }
    };
    // Block number n (from kb0 on) to its place in the ring.
    auto issue = [&](uint32_t n, uint32_t place) {
        uint64_t begin[kBothHalves ? 2 : 1];
#pragma unroll
        for (int i = 0; i < (kBothHalves ? 2 : 1); ++i)
            begin[i] = uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(begins[i] >> 32), n & 63))) << 32 |
                       uint32_t(__builtin_amdgcn_readlane(uint32_t(begins[i]), n & 63));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint64_t from = begin[kBothHalves ? half_of(i) : 0] + (side_of(i) ? side_bytes : 0);
            const uint32_t to = ring_base + place + side_of(i) * kBlockBytes + load_of(i) * 1024;
            if constexpr (EXACT)
                page_to_lds(from, src[i], to);
            else
                lane_to_lds(src[i] == ~0u ? reinterpret_cast<uint64_t>(a.zeros) : from + src[i], to);
        }
    };

    // The queries as B operands: column j, channels 16 s + 8 h .. + 7.
    u32x4 q[NQ][kSteps];
    uint32_t my_pos, my_lo;
    {
        const uint32_t v = wv0 + j;
        const uint32_t row = min(paged_row_of(a, v), span.rows - 1);
        const uint32_t hq = head * a.group + (v < vectors ? v - row * a.group : 0);
        my_pos = span.position + row;
        my_lo = lowest_visible(my_pos, a.window, 0);
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
                                        [&](int n, u32x4 x) { q[n][s] = x; });
    }
    // Of 256 channels queries go to the accumulation registers, which products read as well: there are 256 vector registers, and
    // what vector code works on fills them. (Left to itself the compiler moves the queries out and back in every block.)
    if constexpr (DP == 256) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) asm volatile("" : "+a"(q[n][s]));
    }

    // Where the operands lie in a stage: K row j, piece 2 s + h at ((2 s + h) ^ shuffle) = place0 ^ 2 s; V row 4 h + (lane & 15) / 4
    // (of the four of 16 m + 8 u + ..), channels 32 t + 16 (lane / 16 % 2) + 4 (lane % 4) on.
    const uint32_t k_at = j * kRowBytes + ((h ^ k_shuffle(j)) * 16);
    const uint32_t tr_row = 4 * h + ((lane & 15) >> 2);
    const uint32_t v_at = kBlockBytes + tr_row * kRowBytes + ((v_shuffle(tr_row) * 16) ^ (((lane >> 4) & 1) * 32 + (lane & 3) * 8));

    float ref = 0.0f, threshold = -INFINITY, sum = 0.0f;
    floatx16 o[kOut];
#pragma unroll
    for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.0f;

    // Operands out of LDS: a lane's address for each of a row's places, from which the rest is a constant.
    auto k_operand = [&](uint32_t lane_at) { return *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>((uintptr_t)lane_at); };
    auto v_operand = [&](uint32_t lane_at, int m) {
        u32x4 v;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4 *)(uintptr_t)(lane_at + (16 * m + 8 * u) * kRowBytes));
            const uint2 y = __builtin_bit_cast(uint2, x);
            v[2 * u] = y.x, v[2 * u + 1] = y.y;
        }
        return v;
    };
    // A lane's scores of a block, relative to the reference.
    floatx16 x;
    auto scaled = [&](float s) {
        if constexpr (CAP != kNoCap)
            return softcapped<CAP == kSeriesCap>(s * a.scale_log2, a.cap_log2, ref);
        else
            return __builtin_fmaf(s, a.scale_log2, -ref);
    };
    // Masks the scores of block kb where a row does not see all of it, and moves the references that they pass; `most`: the
    // largest of a lane's.
    auto settle = [&](uint32_t kb, float most) {
        if (kb - inner0 >= inner) {
            most = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t key = 32 * kb + 8 * (r / 4) + 4 * h + r % 4;
                if (key > my_pos || key < my_lo) x[r] = -INFINITY;
                most = fmaxf(most, x[r]);
            }
        }
        if (__builtin_amdgcn_ballot_w64(most > threshold) != 0) {
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
            const float m = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
            const bool live = threshold != -INFINITY;
            float delta = live ? fmaxf(m - kWeightLift<PAGE>, 0.0f) : m - kWeightLift<PAGE>;
            if (m == -INFINITY) delta = 0.0f;
            const float alpha = live ? fast_exp2(-delta) : 1.0f;
            ref += delta;
            if (m != -INFINITY) threshold = kWeightMost;
            sum *= alpha;
#pragma unroll
            for (int t = 0; t < kOut; ++t) o[t] *= alpha;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] -= delta;
        }
    };
    // Rows of block kb no query of the tile sees may hold anything: their values are zeroed in LDS, where the block lies at `at`.
    // (Every lane reads and writes: a branch that turns lanes off would stand amid the fullest registers there are.)
    auto clear = [&](uint32_t kb, uint32_t at) {
        constexpr uint32_t kPieces = 32 * kRowPieces, kStep = kWaves * 64;  // (where lanes are more, two do the same)
#pragma unroll 1
        for (uint32_t first = 0; first < kPieces; first += kStep) {
            const uint32_t p = (first + tid) % kPieces;
            const uint32_t key = 32 * kb + p / kRowPieces, keep = key < tile_lo || key >= tile_hi ? 0 : ~0u;
            auto *const piece = reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(at + kBlockBytes + p * 16));
            u32x4 x = *piece;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= keep;
            *piece = x;
        }
    };
    // The blocks of a stage that have such rows: at most the tile's first and last.
    auto clear_stage = [&](uint32_t kb, uint32_t at) {
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
            if (32 * (kb + u) < tile_lo || 32 * (kb + u) + 32 > tile_hi) clear(kb + u, at + u * kSubBytes);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // Stages of the ring fill ahead of the one at hand; the last one's places are never read where the blocks end inside it. Behind
    // the last stage nothing is asked for, and the waits there are for all that flies.
    const uint32_t stages = (kb_end - kb0 + kSubs - 1) / kSubs;
    look_up(kb0);
    wait_loads<0>();  // (the compiler cannot count the ring's loads: every load of its own has to be in before the first of them)
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (uint32_t(s) >= stages) break;
#pragma unroll
        for (int u = 0; u < kSubs; ++u) issue(s * kSubs + u, s * kStageBytes + u * kSubBytes);
    }
    u32x4 k[kSteps];
    if (stages) {
        // The first block's scores by themselves, and the operands of the second block's.
        if (stages >= kStages - 1)
            wait_loads<kStageLoads * (kStages - 2)>();
        else
            wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        clear_stage(kb0, ring_base);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) k[i] = k_operand(ring_base + (k_at ^ (i * 32)));
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int n = 0; n < NQ; ++n) s = mfma_32x32x16<PAGE>(k[i], q[n][i], s);
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = scaled(s[r]), most = fmaxf(most, x[r]);
        settle(kb0, most);
        if constexpr (kSubs > 1) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) k[i] = k_operand(ring_base + (k_at ^ (i * 32)) + kSubBytes);
        }
    }
    uint32_t at = ring_base, next = ring_base + kStageBytes, free_at = (kStages - 1) * kStageBytes;
    for (uint32_t g = 0; g < stages; ++g) {
        const uint32_t kb = kb0 + g * kSubs;
        // This wavefront's loads of the next stage have landed (those of the stages behind it may still fly); behind the barrier
        // everybody's have, and everybody is done with the stage before this one, which the loads that go out now overwrite.
        if (g + kStages - 1 <= stages)
            wait_loads<kStageLoads * (kStages - 3)>();
        else
            wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        if (g + kStages - 1 < stages) {
            const uint32_t n = (g + kStages - 1) * kSubs;
            if ((n & 63) == 0) look_up(kb0 + n);
#pragma unroll
            for (int u = 0; u < kSubs; ++u) issue(n + u, free_at + u * kSubBytes);
        }
        if (g + 2 == stages) clear_stage(kb + kSubs, next);
        uint32_t k_lane[kSteps], v_lane[kOut];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) k_lane[i] = next + (k_at ^ (i * 32));
#pragma unroll
        for (int t = 0; t < kOut; ++t) v_lane[t] = at + (v_at ^ (t * 64));
        if constexpr (kSubs == 1) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) k[i] = k_operand(k_lane[i]);
        }
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
            // Two stretches of products: the next block's scores beside this block's exponentials, then P.V beside the next scores'
            // scaling and maximum, which are done when the products are: nothing waits at the border of two blocks.
            floatx16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.0f;
            u32x4 p[NP][2], v[kOut][2];
            // The wavefront of a SIMD that is behind goes first: left to itself the SIMD prefers the older one, which then waits at the
            // barrier while the younger runs alone.
            if (u == 0)
                __builtin_amdgcn_s_setprio(3);
            else
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) s = mfma_32x32x16<PAGE>(k[i], q[n][i], s);
                v[i % kOut][i / kOut] = v_operand(v_lane[i % kOut] + u * kSubBytes, i / kOut);
#pragma unroll
                for (int e = i * 16 / kSteps; e < (i + 1) * 16 / kSteps; ++e) {
                    x[e] = fast_exp2(x[e]);
                    if (e % 8 == 7) {
                        float w[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) w[y] = x[e - 7 + y];
                        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                        u32x4 pieces[NP];
                        split_8<PAGE, NP>(w, pieces);
#pragma unroll
                        for (int n = 0; n < NP; ++n) p[n][e / 8] = pieces[n];
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            float most = 0.0f;
            if (u == 0 && kSubs > 1)
                __builtin_amdgcn_s_setprio(2);
            else
                __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int i = 0; i < 2 * kOut; ++i) {
                const int t = i % kOut, m = i / kOut;
#pragma unroll
                for (int n = 0; n < NP; ++n) o[t] = mfma_32x32x16<PAGE>(v[t][m], p[n][m], o[t]);
                // (The scores' last product is on its way for the time of two others.)
                constexpr int kSlots = 2 * kOut > 4 ? 2 * kOut - 3 : 2, kSkip = 2 * kOut > 4 ? 2 : 1;
#pragma unroll
                for (int r = (i - kSkip) * 16 / kSlots; r < (i - kSkip + 1) * 16 / kSlots; ++r) {
                    if (r < 0 || r >= 16) continue;
                    s[r] = scaled(s[r]);
                    if (r == 2)
                        most = max3(s[0], s[1], s[2]);
                    else if (r > 2 && r % 2 == 0)
                        most = max3(most, s[r - 1], s[r]);
                    else if (r == 15)
                        most = max3(most, s[15], s[15]);
                }
                if (kSubs > 1) k[i] = k_operand(k_lane[i] + u * kSubBytes);
                __builtin_amdgcn_sched_barrier(0);
            }
            x = s;
            if (kb + u + 1 >= kb_end) break;
            settle(kb + u + 1, most);
        }
        const uint32_t was = at;
        at = next;
        free_at = was - ring_base;
        next = next + kStageBytes == ring_base + kStages * kStageBytes ? ring_base : next + kStageBytes;
    }
    // A lane holds of its column channels 32 t + 8 (r / 4) + 4 h + r % 4.
    // (The check comes before the stores: the barriers it takes would wait for them.)
    const bool whole = a.parts == 1, mine = wv0 + j < vectors;
    const uint32_t v = wv0 + j;
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    const float l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    float check[4] = {l, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) check[r % 4] += EXACT || 32u * t + 8 * (r / 4) + 4 * h < d ? o[t][r] : 0.0f;
    const float all = (check[0] + check[1]) + (check[2] + check[3]);
    if (any_of_group(mine && to_be_done_over<PAGE>(all), &lds_flag)) {
        paged_careful<PAGE, ELEM, DP>(a, span, head, v0, min(v0 + kTile, vectors), wave, kWaves, 32 * kb0, 32 * kb_end,
                                      [&](uint32_t v, const float (&acc)[DP / 64], float m, float l) {
                                          paged_write_careful<PAGE, ELEM, DP>(a, span, head, v, whole, slot0 + v - v0, true, acc, m, l);
                                      });
    } else if (mine) {
        if (whole) {
            const float inv = 1.0f / l;
            const uint32_t row = paged_row_of(a, v), hq = head * a.group + v - row * a.group;
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
                    for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(o[t][r + e] * inv);
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
                        floatx4{o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]};
            if (h == 0) a.ws_ml[slot] = make_float2(threshold == -INFINITY ? -INFINITY : ref, l);
        }
    }
}

template <auto Kernel, int ELEM, int DP>
hipError_t launch_chunk_kernel(const PagedAttn &a, hipStream_t stream) {
    int device = -1;
    (void)hipGetDevice(&device);
    const hipError_t granted = granted_once<Kernel>(device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(chunk_lds(DP)));
    });
    if (granted != hipSuccess) return granted;
    launch_kernel(Kernel, a.units * a.parts, paged_chunk_waves(DP, ELEM) * 64, chunk_lds(DP), stream, a);
    return hipGetLastError();
}
template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP>
hipError_t launch_chunk_as(const PagedAttn &a, hipStream_t stream) {
    if constexpr (!paged_chunk_takes(DP, PAGE, ELEM)) {
        return hipErrorInvalidValue;
    } else {
        if (a.cap_log2 == 0.0f) return launch_chunk_kernel<&paged_chunk_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, kNoCap>, ELEM, DP>(a, stream);
        if constexpr (ELEM != ITAK_ELEM_F32)
            if (!paged_cap_by_series(ELEM, a.cap_log2))
                return launch_chunk_kernel<&paged_chunk_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, kShortCap>, ELEM, DP>(a, stream);
        return launch_chunk_kernel<&paged_chunk_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, kSeriesCap>, ELEM, DP>(a, stream);
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
