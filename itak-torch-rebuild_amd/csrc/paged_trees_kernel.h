// Attention of drafted trees over pages: some tens of rows over a long context.
//
// What a row sees behind the held positions is in its record (paged_tree.h), a bit a key; in front of them every row sees all of its window. 4 d
// operations a pair of vector and key, some 250 a byte of keys at 128 vectors: between the matrix pipe and the memory, and where the context is
// short neither bounds it but the chain of trips, the code that is fetched to be run once, and the partials.
//
// A workgroup has one part of one tile (the cut is such that all parts are about of one length). Each of its wavefronts has a set of 32 of the
// tile's vectors and, as one of `groups` that have the same set, every groups-th block of 32 keys: two wavefronts a SIMD, which fill each other's gaps,
// whether the tile is two sets or eight. The loop is one block long: the products of the scores, the softmax, those of the values. Blocks
// travel from the pages to LDS without passing through registers, into a ring that is full at the start; layout and operands are those of the
// kernel of many rows (paged_chunk_kernel.h), whose loop is longer and faster: it takes batches of tiles of 256 vectors. At the end the groups meet in LDS.
//
// A small tile makes small partials and reads the keys once a set: the host weighs the two (trees_plan). Partials are written as the registers hold
// them, 1 KiB a store (a vector's row at a time they took 1.6 us of a part).
//
// Measured, 32 query heads over 4 of 128 channels, f16: 16 rows at 4,096 12.2 us (8.4 MB of keys and values), 64 rows at 8,192 22.9 (16.8 MB, 8.6 GFLOP), 4
// trees of 61 rows in a window of 2,048 26.4 (21 MB, 8.2 GFLOP). Of a part's clocks some 16,000 are its start and end: arguments and item 1,350, page ids
// and queries 2,900, sending the ring's loads 2,600, the first blocks' way 2,600, the groups' meeting 4,200, the stores 2,000; a step of two blocks takes
// 2,700, some 850 of them products and softmax, where LDS reads and writes take some 1,900; with all keys in the L2 it takes 2,550.
#pragma once

#include "lds_grant.h"
#include "paged_careful.h"
#include "paged_ring.h"

namespace itak {

namespace {

// Blocks of 32 keys in the ring, 16 bytes from one register quad of a wavefront to the next where the groups meet (a quad's 64 lanes, and one
// that moves the next quad to other banks), and bytes of LDS for either.
constexpr int trees_blocks(int dp, int waves) { return dp == 256 ? 4 : waves; }
constexpr uint32_t kTreesQuad = 65;
constexpr size_t trees_lds(int dp, int waves) {
    const size_t ring = size_t(trees_blocks(dp, waves)) * 2 * 32 * 2 * dp, met = size_t(waves) * (dp / 8) * kTreesQuad * 16;
    return ring > met ? ring : met;
}

template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP>
__global__ __launch_bounds__(paged_trees_waves(DP, PAGE, ELEM) * 64) void paged_trees_kernel(PagedAttn a) {
    typedef typename Elem<ELEM>::type T;
    constexpr int kWaves = paged_trees_waves(DP, PAGE, ELEM), kTile = kWaves * 32;
    constexpr uint32_t kBlocks = trees_blocks(DP, kWaves), kWavesShift = kWaves == 8 ? 3 : 2;
    static_assert(kBlocks >= kWaves);  // two steps of the most groups
    constexpr int kSteps = DP / 16;               // products of a score tile
    constexpr int kOut = DP / 32;                 // output tiles of 32 channels
    constexpr int kRowBytes = 2 * DP, kBlockBytes = 32 * kRowBytes, kStageBytes = 2 * kBlockBytes;
    constexpr int kRowPieces = DP / 8;            // 16-byte pieces of a row
    constexpr int kLoadRows = 512 / DP;           // rows a load of one wavefront moves
    constexpr int kSideLoads = DP / 16;           // loads of a side of a block, dealt to the wavefronts in turn
    constexpr int kLoads = 2 * kSideLoads / kWaves;
    extern __shared__ __attribute__((aligned(16))) unsigned char ring[];
    __shared__ uint32_t lds_sees[kTreeBlocks][kTile];
    __shared__ float2 lds_ml[kWaves][32];
    __shared__ uint32_t lds_flag;

    paged_fetch_arguments<true>(a);
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t h = lane >> 5, j = lane & 31;
    const uint32_t d = EXACT ? DP : a.g.head_dim;
    PagedTreeLine line(a);
    line.cut_apart();
    uint32_t nth, head;
    if (!paged_part_of(line, nth, head)) return;
    const uint32_t at = nth * line.share;
    PagedSpan span;
    if (at >= line.total || !line.find<PagedTreeLine::kBlock>(span, at)) return;
    const bool trees = paged_has_trees(a);
    const uint32_t turn = span.tiles == 1 ? 0 : (at - span.start) / span.run, from = (at - span.start) - turn * span.run;
    const uint32_t tile = span.tiles - 1 - turn;  // (the longest first, of a chain)
    const bool whole = span.blocks <= line.share;
    const uint32_t vectors = span.rows * a.group, v0 = tile << a.tile_shift, v_end = min(v0 + a.tile, vectors);
    const uint32_t first_row = paged_row_of(a, v0), last_row = min(paged_row_of(a, v_end - 1), span.rows - 1);
    // Keys that some of the tile's rows see, and this part's blocks of them.
    const uint32_t tile_lo = lowest_visible(span.position + (trees ? 0 : first_row), a.window, 0), tile_hi = span.position + last_row + 1;
    // (One for all lanes, which the compiler does not see.)
    const uint32_t kb0 = __builtin_amdgcn_readfirstlane(max(span.first + from, tile_lo / 32));
    const uint32_t kb_end = min(span.first + min(from + line.share, span.blocks), (tile_hi + 31) / 32);
    const uint32_t blocks = __builtin_amdgcn_readfirstlane(kb_end > kb0 ? kb_end - kb0 : 0);
    // The wavefront's vectors, and which of every `groups` blocks are its own.
    const uint32_t sets_shift = a.tile_shift - 5, sets = 1u << sets_shift, groups_shift = kWavesShift - sets_shift, groups = 1u << groups_shift;
    const uint32_t set = wave & (sets - 1), group = wave >> sets_shift;
    const uint32_t wv0 = v0 + set * 32;
    // Keys that all of its rows see.
    const uint32_t w_first = min(paged_row_of(a, wv0), span.rows - 1), w_last = min(paged_row_of(a, wv0 + 31), span.rows - 1);
    const uint32_t every_lo = lowest_visible(span.position + w_last, a.window, 0), every_hi = span.position + (trees ? 0 : w_first + 1);

    // Where the next 64 blocks' halves begin, a block a lane. (Positions past the end are clamped to the last page: any row of it may be read.)
    const uint32_t last_page = (span.position + span.rows - 1) >> a.g.page_shift, page_mask = (1u << a.g.page_shift) - 1;
    const uint64_t head_base = reinterpret_cast<uint64_t>(a.layer_base + head * a.g.head_stride);
    const uint32_t page_bytes = uint32_t(2 * a.g.page_stride), side_bytes = uint32_t(2 * a.g.side_stride);
    // (A wavefront's loads lie in one half of a block where it has one or two of them.)
    constexpr int kHalves = kLoads > 2 ? 2 : 1;
    auto load_of = [&](int i) { return kSideLoads >= kWaves ? wave + kWaves * (i % (kSideLoads / kWaves)) : wave % kSideLoads; };
    auto half_of = [&](int i) { return load_of(i) * kLoadRows / 16; };
    auto key_of = [&](uint32_t kb, int i) { return 32 * (kb + lane) + 16 * (kHalves == 2 ? uint32_t(i) : half_of(0)); };
    uint32_t ids[kHalves];
    auto ask = [&](uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kHalves; ++i) ids[i] = a.batch[span.table + min(key_of(kb, i) >> a.g.page_shift, last_page)];
    };
    uint64_t begins[kHalves];
    auto answer = [&](uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kHalves; ++i)
            begins[i] = head_base + uint64_t(ids[i]) * page_bytes + (key_of(kb, i) & page_mask) * (d * 2);
    };
    ask(kb0);

    // A lane's column: its query, and what it sees.
    const uint32_t v = wv0 + j, row = min(paged_row_of(a, v), span.rows - 1);
    const uint32_t hq = head * a.group + (v < vectors ? v - row * a.group : 0);
    const uint32_t *const record = a.tree + tree_record_at(trees, span.row0 + row);
    typename QueryRaw<ELEM>::type raw[kSteps];
    {
        const T *src = static_cast<const T *>(a.q.data) + uint64_t(span.row0 + row) * a.q.row_stride + hq * a.q.head_stride;
        if (a.q_on_16) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) raw[s] = load_query<ELEM, true>(src + (EXACT || 16 * s + 8 * h < d ? 16 * s + 8 * h : 0));
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) raw[s] = load_query<ELEM, false>(src + (EXACT || 16 * s + 8 * h < d ? 16 * s + 8 * h : 0));
        }
    }
    // Its record, where the part's keys reach behind the held positions, or a window is counted from its depth. (A lane of each half has the column:
    // each brings every other word. No lane is turned off.)
    const bool reaches = trees && 32 * kb_end > span.position;
    uint32_t word = kTreeChain | row, sees[kTreeBlocks / 2 + 1];
    if (trees && (reaches || a.window)) word = record[kTreeDepth];
    if (reaches) {
#pragma unroll
        for (uint32_t w = 0; w < kTreeBlocks / 2 + 1; ++w) sees[w] = record[kTreeSees + min(2 * w + h, kTreeBlocks - 1)];
    }

    // Loads: piece `lane` of a load is row lane / kRowPieces of its rows, 16-byte place lane % kRowPieces, which holds the piece place ^
    // (the row's shuffle): so that neither the operand reads of K nor the turning reads of V meet a bank twice.
    const uint32_t l_row = lane / kRowPieces, l_place = lane % kRowPieces;
    auto k_shuffle = [](uint32_t r) { return DP == 64 ? (r >> 1) & 7 : r & 15; };
    auto v_shuffle = [](uint32_t r) { return DP == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
    // Load i of this wavefront: which side.
    auto side_of = [&](int i) { return kSideLoads >= kWaves ? uint32_t(i / (kSideLoads / kWaves)) : wave / kSideLoads; };
    uint32_t src[kLoads];  // bytes from the half block's first row
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t r = load_of(i) * kLoadRows + l_row;
        const uint32_t piece = l_place ^ (side_of(i) ? v_shuffle(r) : k_shuffle(r));
        src[i] = (r & 15) * d * 2 + piece * 16;
        if (!EXACT && piece * 8 >= d) src[i] = ~0u;  // (zeros)
    }
    const uint32_t ring_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)ring;
    // Block n (of the part's) to its place in the ring.
    auto issue = [&](uint32_t block) __attribute__((always_inline)) {
        const uint32_t n = block, place = n % kBlocks;
        uint64_t begin[kHalves];
#pragma unroll
        for (int i = 0; i < kHalves; ++i)
            begin[i] = uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(begins[i] >> 32), n & 63))) << 32 |
                       uint32_t(__builtin_amdgcn_readlane(uint32_t(begins[i]), n & 63));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint64_t first = begin[kHalves == 2 ? half_of(i) : 0] + (side_of(i) ? side_bytes : 0);
            const uint32_t to = ring_base + place * kStageBytes + side_of(i) * kBlockBytes + load_of(i) * 1024;
            if constexpr (EXACT)
                page_to_lds(first, src[i], to);
            else
                lane_to_lds(src[i] == ~0u ? reinterpret_cast<uint64_t>(a.zeros) : first + src[i], to);
        }
    };

    // The compiler cannot count the ring's loads: every load of its own has to be in before the first of them.
    wait_loads<0>();
    answer(kb0);
    uint32_t issued = min(blocks, kBlocks);
    for (uint32_t n = 0; n < issued; ++n) issue(n);
    // Waits until at most `most` blocks' loads of this wavefront's are on their way, or fewer.
    auto wait_for = [&](uint32_t most) __attribute__((always_inline)) {
        if (most >= 7)
            wait_loads<7 * kLoads>();
        else if (most >= 6)
            wait_loads<6 * kLoads>();
        else if (most >= 4)
            wait_loads<4 * kLoads>();
        else if (most >= 2)
            wait_loads<2 * kLoads>();
        else
            wait_loads<0>();
    };

    // Queries as B operands: column j, channels 16 s + 8 h .. + 7.
    u32x4 q[NQ][kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
        split_query<PAGE, ELEM, NQ>(raw[s], v < vectors && (EXACT || 16 * s + 8 * h < d), [&](int n, u32x4 x) { q[n][s] = x; });
    const uint32_t tree_block = span.position / 32;
    const uint32_t my_pos = span.position + row, my_lo = lowest_visible(span.position + tree_depth(word), a.window, 0);
    if (reaches) {
#pragma unroll
        for (uint32_t w = 0; w < kTreeBlocks / 2 + 1; ++w)
            lds_sees[min(2 * w + h, kTreeBlocks - 1)][set * 32 + j] = word & kTreeChain ? ~0u : sees[w];
    }
    if (tid == 0) lds_flag = 0;

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

    const uint32_t steps = (blocks + groups - 1) >> groups_shift;
#pragma unroll 1
    for (uint32_t n = 0; n < steps; ++n) {
        // This wavefront's loads of the step's blocks have landed; behind the barrier everybody's have, and everybody is done with the step before,
        // whose places the loads that go out now take. (The ring holds two steps or more.)
        const uint32_t upto = min(blocks, (n + 1) << groups_shift);
        wait_for(issued > upto ? issued - upto : 0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (n)
            for (const uint32_t more = min(blocks, issued + groups); issued < more; ++issued) {
                if ((issued & 63) == 0) ask(kb0 + issued), answer(kb0 + issued);
                issue(issued);
            }
        // Rows no query of the tile sees may hold anything: their values are zeroed. (Every lane reads and writes.)
        const uint32_t k0 = 32 * (kb0 + (n << groups_shift)), k1 = 32 * (kb0 + upto);
        if (k0 < tile_lo || k1 > tile_hi) {
            constexpr uint32_t kPieces = 32 * kRowPieces;
            for (uint32_t b = 0; b < (k1 - k0) / 32; ++b) {
                if (k0 + 32 * b >= tile_lo && k0 + 32 * b + 32 <= tile_hi) continue;
                const uint32_t values = ring_base + (((n << groups_shift) + b) % kBlocks) * kStageBytes + kBlockBytes;
#pragma unroll 1
                for (uint32_t at = 0; at < kPieces; at += kWaves * 64) {
                    const uint32_t p = (at + tid) % kPieces;  // (where threads are more, two do the same)
                    const uint32_t key = k0 + 32 * b + p / kRowPieces, keep = key < tile_lo || key >= tile_hi ? 0 : ~0u;
                    auto *const piece = reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(values + p * 16));
                    u32x4 x = *piece;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] &= keep;
                    *piece = x;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        }
        const uint32_t mine = (n << groups_shift) + group, kb = kb0 + mine, stage = ring_base + (mine % kBlocks) * kStageBytes;
        if (mine >= blocks) continue;
        floatx16 x;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const u32x4 k = *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>((uintptr_t)(stage + (k_at ^ (s * 32))));
#pragma unroll
            for (int m = 0; m < NQ; ++m) x = mfma_32x32x16<PAGE>(k, q[m][s], x);
        }
        if (a.cap_log2 != 0.0f) {
            if (paged_cap_by_series(ELEM, a.cap_log2)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = softcapped<true, true>(x[r] * a.scale_log2, a.cap_log2, ref);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = softcapped<false>(x[r] * a.scale_log2, a.cap_log2, ref);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], a.scale_log2, -ref);
        }
        // A lane holds of its column the keys 8 (r / 4) + 4 h + r % 4.
        if (32 * kb < every_lo || 32 * kb + 32 > every_hi) {
            uint32_t bits = kb < tree_block || !reaches ? ~0u : lds_sees[min(kb - tree_block, kTreeBlocks - 1)][set * 32 + j];
            // (Of the keys from my_lo to my_pos: a shift by 32 or more leaves nothing.)
            const uint32_t below = my_lo > 32 * kb ? my_lo - 32 * kb : 0, upto = my_pos >= 32 * kb ? my_pos - 32 * kb + 1 : 0;
            bits &= below < 32 ? ~0u << below : 0u;
            bits &= upto < 32 ? (1u << upto) - 1 : ~0u;
            bits >>= 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = bits >> (8 * (r / 4) + r % 4) & 1 ? x[r] : -INFINITY;
        }
        float most = max3(x[0], x[1], x[2]);
#pragma unroll
        for (int r = 3; r < 15; r += 2) most = max3(most, x[r], x[r + 1]);
        most = fmaxf(most, x[15]);
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
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = fast_exp2(x[8 * m + e]);
            sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            u32x4 p[NP];
            split_8<PAGE, NP>(w, p);
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
                u32x4 y;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const shortx4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) shortx4 *)(uintptr_t)(stage + (v_at ^ (t * 64)) + (16 * m + 8 * u) * kRowBytes));
                    const uint2 pair = __builtin_bit_cast(uint2, z);
                    y[2 * u] = pair.x, y[2 * u + 1] = pair.y;
                }
#pragma unroll
                for (int i = 0; i < NP; ++i) o[t] = mfma_32x32x16<PAGE>(y, p[i], o[t]);
            }
        }
    }
    // The groups meet in the ring's place, where a wavefront has 1 KiB for each of its register quads: a lane holds of its column the channels
    // 32 t + 8 (r / 4) + 4 h + r % 4, quad 4 t + r / 4. Maxima and sums lie beside.
    constexpr uint32_t kQuads = DP / 8;
    floatx4 *const met = reinterpret_cast<floatx4 *>(ring);
    {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        if (h == 0)
            lds_ml[wave][j] = make_float2(threshold == -INFINITY ? -INFINITY : ref, __uint_as_float(both[0]) + __uint_as_float(both[1]));
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();  // (everybody is done with the ring)
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }
    // Column c of a set over all its groups: the maximum and sum, and the groups' weights. (A maximum of minus infinity: nothing visible, a sum of 0, or
    // scores that are no numbers, which the sum then is.)
    auto all_of = [&](uint32_t c, auto &weights) __attribute__((always_inline)) {
        constexpr uint32_t kGroups = sizeof(weights) / sizeof(float);
        float2 ml[kGroups];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) ml[g] = lds_ml[(g << sets_shift) + set][c];
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) m = fmaxf(m, ml[g].x);
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) {
            weights[g] = ml[g].x == -INFINITY ? 0.0f : fast_exp2(ml[g].x - m);
            l += ml[g].x == -INFINITY ? ml[g].y : weights[g] * ml[g].y;
        }
        return make_float2(m, l);
    };
    // A part's place: its workgroup's (a head's side by side); of a vector's channels as the registers of its column hold them.
    const uint64_t slot0 = uint64_t(head * a.groups + nth) * a.tile;
    floatx4 *const part = reinterpret_cast<floatx4 *>(a.ws_acc + slot0 * DP);
    float2 *const part_ml = a.ws_ml + slot0;
    // Whether the part is to be done over.
    auto asked_over = [&](bool bad) __attribute__((always_inline)) {
        if (bad) lds_flag = 1;
        __syncthreads();
        return lds_flag != 0;
    };
    // What a lane finishes, where 2^GROUPS groups share a set: of a split unit quads of its own column, stored as they are; of a whole one, whose outputs
    // are stored as rows, pairs of quads: eight channels of a vector, sixteen lanes a row of 128.
    auto finish = [&](auto GROUPS) __attribute__((always_inline)) {
        constexpr uint32_t kGroups = 1u << GROUPS.value, kMine = kQuads / kGroups, kOfRow = DP / 8;
        floatx4 acc[kMine];
        float weights[kGroups];
        // (Of a split unit a group's own quads stay in its registers.)
        auto own = [&](uint32_t q) { return floatx4{o[q / 4][4 * (q % 4)], o[q / 4][4 * (q % 4) + 1], o[q / 4][4 * (q % 4) + 2], o[q / 4][4 * (q % 4) + 3]}; };
#pragma unroll
        for (uint32_t q = 0; q < kQuads; ++q)
            if (whole || q / kMine != group) met[(wave * kQuads + q) * kTreesQuad + lane] = own(q);
        __syncthreads();
        if (!whole) {
            const float2 ml = all_of(j, weights);
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g)
                if (g == group) {
#pragma unroll
                    for (uint32_t u = 0; u < kMine; ++u) acc[u] = own(g * kMine + u) * weights[g];
                }
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g) {
                if (g == group) continue;
                const uint32_t w = (g << sets_shift) + set;
                const float weight = weights[g];
#pragma unroll
                for (uint32_t u = 0; u < kMine; ++u) {
                    const floatx4 y = met[(w * kQuads + group * kMine + u) * kTreesQuad + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[u][e] = __builtin_fmaf(weight, y[e], acc[u][e]);
                }
            }
            float check[4] = {ml.y, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t u = 0; u < kMine; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) check[e] += EXACT || 8 * (group * kMine + u) + 4 * h < d ? acc[u][e] : 0.0f;
            if (asked_over(wv0 + j < v_end && to_be_done_over<PAGE>((check[0] + check[1]) + (check[2] + check[3])))) return true;
#pragma unroll
            for (uint32_t u = 0; u < kMine; ++u)
                if (wv0 < v_end) store_part(part, (set * kQuads + group * kMine + u) * 64 + lane, acc[u]);
            if (group == 0 && h == 0) part_ml[set * 32 + j] = ml;
        } else {
            const uint32_t ch = lane % kOfRow;
            auto column = [&](uint32_t u) { return (lane + 64 * (group * (kMine / 2) + u)) / kOfRow; };
            bool bad = false;
#pragma unroll
            for (uint32_t u = 0; u < kMine / 2; ++u) {
                const uint32_t c = column(u);
                const float2 ml = all_of(c, weights);
                acc[2 * u] = acc[2 * u + 1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t g = 0; g < kGroups; ++g) {
                    const uint32_t w = (g << sets_shift) + set;
                    const float weight = weights[g];
#pragma unroll
                    for (uint32_t x = 0; x < 2; ++x) {
                        const floatx4 y = met[(w * kQuads + ch) * kTreesQuad + x * 32 + c];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[2 * u + x][e] = __builtin_fmaf(weight, y[e], acc[2 * u + x][e]);
                    }
                }
                float check = ml.y;
                const float inv = 1.0f / ml.y;
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) check += EXACT || 8 * ch < d ? acc[2 * u + x][e] : 0.0f, acc[2 * u + x][e] *= inv;
                bad = bad || (wv0 + c < v_end && to_be_done_over<PAGE>(check));
            }
            if (asked_over(bad)) return true;
#pragma unroll
            for (uint32_t u = 0; u < kMine / 2; ++u) {
                const uint32_t v = wv0 + column(u);
                if (v >= v_end || (!EXACT && 8 * ch >= d)) continue;
                const uint32_t row = paged_row_of(a, v), hq = head * a.group + v - row * a.group;
                T *dst = static_cast<T *>(a.out.data) + uint64_t(span.row0 + row) * a.out.row_stride + hq * a.out.head_stride + 8 * ch;
                Piece<T, 8> y;
#pragma unroll
                for (int e = 0; e < 8; ++e) y.v[e] = Elem<ELEM>::from_f32(acc[2 * u + e / 4][e % 4]);
                if (a.out_on_16) {
                    *reinterpret_cast<Piece<T, 8> *>(dst) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = y.v[e];
                }
            }
        }
        return false;
    };
    bool over = false;
    if (groups == 1)
        over = finish(std::integral_constant<int, 0>{});
    else if (groups == 2)
        over = finish(std::integral_constant<int, 1>{});
    else if constexpr (kWaves == 8)
        over = finish(std::integral_constant<int, 2>{});
    if (!over) return;
    paged_careful<PAGE, ELEM, DP, true>(a, span, head, v0, v_end, wave, kWaves, 32 * kb0, 32 * max(kb0, kb_end),
                                        [&](uint32_t u, const float (&sums)[DP / 64], float most, float s) {
                                            if (whole)
                                                paged_write_careful<PAGE, ELEM, DP>(a, span, head, u, true, 0, false, sums, most, s);
                                            else
                                                paged_part_careful<PAGE, DP>(a, slot0, u - v0, sums, most, s);
                                        });
}

template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP>
hipError_t launch_trees_as(const PagedAttn &a, hipStream_t stream) {
    constexpr int kWaves = paged_trees_waves(DP, PAGE, ELEM);
    constexpr auto kernel = &paged_trees_kernel<PAGE, ELEM, DP, EXACT, NQ, NP>;
    int device = -1;
    (void)hipGetDevice(&device);
    const hipError_t granted = granted_once<kernel>(device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(trees_lds(DP, kWaves)));
    });
    if (granted != hipSuccess) return granted;
    launch_kernel(kernel, dim3(a.across, a.g.kv_heads), kWaves * 64, trees_lds(DP, kWaves), stream, a);
    return hipGetLastError();
}
template <int PAGE, int ELEM, int NQ, int NP>
hipError_t launch_trees(const PagedAttn &a, hipStream_t stream) {
    const uint32_t d = a.g.head_dim;
    return d == 64    ? launch_trees_as<PAGE, ELEM, 64, true, NQ, NP>(a, stream)
           : d < 64   ? launch_trees_as<PAGE, ELEM, 64, false, NQ, NP>(a, stream)
           : d == 128 ? launch_trees_as<PAGE, ELEM, 128, true, NQ, NP>(a, stream)
           : d < 128  ? launch_trees_as<PAGE, ELEM, 128, false, NQ, NP>(a, stream)
           : d == 256 ? launch_trees_as<PAGE, ELEM, 256, true, NQ, NP>(a, stream)
                      : launch_trees_as<PAGE, ELEM, 256, false, NQ, NP>(a, stream);
}

}  // namespace

}  // namespace itak
