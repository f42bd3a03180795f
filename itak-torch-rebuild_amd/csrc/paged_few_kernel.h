// Attention of few rows over pages: single tokens and short blocks, 16 or 32 query vectors a tile.
//
//   o_j = sum_p 2^(s_jp - m_j) v_p / sum_p 2^(s_jp - m_j),  s = log2(e) * (scale q.k, capped), m_j the running maximum
//
// Every visible key and value row is read once a tile and multiplied into its columns: 32 or 64 operations a byte, below
// what the matrix pipe does beside the memory, so the bytes bound it, and where they are few the chain of trips to memory: the
// batch's items, page ids, rows, and the merge.
//
// A wavefront takes 32-key blocks of its workgroup's run in turn with three others, keeps a softmax of its own, and meets them
// once at the end of a unit, through LDS. Per block: S^T = K . Q^T, with K's rows read from the page as the operand wants them
// (a lane's 16 bytes are 8 channels of its row; the rows are dealt to the two tiles so that a lane receives the scores of 8
// consecutive keys), then O^T += V^T . P^T with P in the registers the scores came in. V lies row by row, and the product
// wants 8 keys of one channel in a lane: a lane reads 8 rows' 16 bytes (a page row of 128 channels is one run of 16 lanes) and
// turns the 8 x 8 block over in its registers, 32 permutes a block; it then holds channels 8i .. 8i + 7 where tile t of the output is
// the channels 8i + t, which costs nothing as the output is put in order when it is stored.
// The next block's rows are asked for before the block at hand is multiplied, and its page ids a block earlier.
//
// Measured, 32 heads over 4 of 128 channels: 16 tokens at up to 16,384 in bf16, 315 MB, 54.5 us, 5.8 TB/s, where a kernel that only reads
// gets 6.2; one token at 4,096 6.0 to 6.4 us, of which the arguments and the item's place take 1.3, page ids and rows 1, 32 keys' products 0.7
// and the meeting of the wavefronts 1.
#pragma once

#include "paged_careful.h"

namespace itak {

namespace {

constexpr int kFewWaves = 4;
constexpr int kSet = kPagedSet;  // vectors of one column tile

// Rows and channels of a 32-key block as a lane holds them: DP = head_dim padded to 64, 128 or 256.
template <int DP>
struct FewShape {
    static constexpr int kSteps = DP / 32;                 // products of a score tile
    static constexpr int kHalves = DP == 256 ? 2 : 1;      // runs of up to 128 channels
    static constexpr int kWide = DP == 64 ? 4 : 8;         // channels a lane reads of a value row in a run
    static constexpr int kTiles = DP / 16;                 // output tiles of 16 channels
};

template <int DP>
struct FewBlock {
    typedef FewShape<DP> S;
    u32x4 k[2][S::kSteps];
    uint32_t v[S::kHalves][8][S::kWide / 2];
};

// NQ, NP: pieces of the pages' type that a query and a weight enter the products as. EXACT: head_dim == DP. SETS of 16 vectors.
template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP, int SETS>
__global__ __launch_bounds__(kFewWaves * 64, paged_few_groups_per_cu(DP, PAGE, ELEM, SETS)) void paged_few_kernel(PagedAttn a) {
    typedef FewShape<DP> S;
    typedef typename Elem<ELEM>::type T;
    // (Two blocks of 256 channels beside the accumulators are more than 512 registers.)
    constexpr bool kAhead = DP <= 128;
    constexpr int kTile = SETS * kSet;
    constexpr int kStride = DP + 4;  // floats from one vector to the next in LDS
    // Queries in several pieces, and those of a large tile, lie in LDS, where the four wavefronts share them, and not in
    // registers that the rows need.
    constexpr bool kQInLds = NQ > 1 || SETS * DP > 256;
    constexpr uint32_t kQBytes = kQInLds ? SETS * NQ * S::kSteps * 64 * sizeof(u32x4) : 0;
    constexpr uint32_t kOBytes = kFewWaves * kTile * kStride * sizeof(float);
    // (The queries' place is the wavefronts' results' in the end.)
    __shared__ __attribute__((aligned(16))) unsigned char lds[kQBytes > kOBytes ? kQBytes : kOBytes];
    __shared__ float2 lds_ml[kFewWaves][kTile];
    __shared__ uint32_t lds_flag;
    u32x4 *const lds_q = reinterpret_cast<u32x4 *>(lds);
    auto lds_o = reinterpret_cast<float (*)[kTile][kStride]>(lds);

    paged_fetch_arguments(a);
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t g = lane >> 4, i = lane & 15;
    const uint32_t d = EXACT ? DP : a.g.head_dim;
    PagedLine line(a);
    line.cut();
    uint32_t at = blockIdx.x * line.share;
    const uint32_t end = min(line.total, at + line.share);

    // Where a lane reads: of a key block the rows 8 (i / 4) + i % 4 (+ 4 for the second tile), channels 8g of every 32; of a value
    // block the rows 8g .. 8g + 7, channels kWide * i of every run. Channels past head_dim are read from channel 0.
    const uint32_t k_group = i >> 2, k_row = i & 3;
    uint32_t k_chan[S::kSteps], v_chan[S::kHalves];
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) k_chan[s] = EXACT || 32 * s + 8 * g < d ? 32 * s + 8 * g : 0;
#pragma unroll
    for (int h = 0; h < S::kHalves; ++h) {
        const uint32_t c = 128 * h + S::kWide * i;
        v_chan[h] = EXACT || c < d ? c : 0;
    }
    const uint32_t page_mask = (1u << a.g.page_shift) - 1;

    while (at < end) {
        PagedSpan span;
        if (!line.find<PagedLine::kBlock>(span, at)) break;
        const uint32_t local = (at - span.start) / span.run, from = (at - span.start) - local * span.run;
        const uint32_t count = min(span.blocks - from, end - at);
        const uint32_t tile = local / a.g.kv_heads, head = local - tile * a.g.kv_heads;
        const uint32_t unit = span.unit0 + local;
        const uint32_t length = span.position + span.rows;
        const uint32_t vectors = span.rows * a.group, v0 = tile * kTile;
        const uint32_t first_row = paged_row_of(a, v0), last_row = min(paged_row_of(a, v0 + kTile - 1), span.rows - 1);
        // Positions some, and positions every row of the tile sees.
        const uint32_t some_lo = lowest_visible(span.position + first_row, a.window, 0), some_hi = span.position + last_row + 1;
        const uint32_t every_lo = lowest_visible(span.position + last_row, a.window, 0), every_hi = span.position + first_row + 1;
        // A lane's columns.
        uint32_t my_row[SETS], my_head[SETS];
#pragma unroll
        for (int n = 0; n < SETS; ++n) {
            const uint32_t v = v0 + n * kSet + i;
            my_row[n] = min(paged_row_of(a, v), span.rows - 1);
            my_head[n] = head * a.group + (v < vectors ? v - my_row[n] * a.group : 0);
        }

        const uint32_t *ids = a.batch + span.table;
        const uint32_t last_page = (length - 1) >> a.g.page_shift;
        const uint64_t head_off = head * a.g.head_stride;
        auto page_of = [&](uint32_t key) { return ids[min(key >> a.g.page_shift, last_page)]; };
        auto load = [&](uint32_t kb, uint32_t k_page, uint32_t v_page, FewBlock<DP> &b) {
            const uint16_t *kp = a.layer_base + k_page * a.g.page_stride + head_off +
                                 (((32 * kb + 8 * k_group) & page_mask) + k_row) * d;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < S::kSteps; ++s)
                    b.k[t][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kp + 4 * t * d + k_chan[s]));
            const uint16_t *vp = a.layer_base + v_page * a.g.page_stride + head_off + a.g.side_stride +
                                 ((32 * kb + 8 * g) & page_mask) * d;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const uint16_t *p = vp + r * d + v_chan[h];
                    if constexpr (S::kWide == 8) {
                        const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
#pragma unroll
                        for (int c = 0; c < 4; ++c) b.v[h][r][c] = x[c];
                    } else {
                        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p));
                        b.v[h][r][0] = x[0], b.v[h][r][1] = x[1];
                    }
                }
        };

        // What the first block takes is asked for in the order of the trips: page ids, the queries, keys and values.
        const uint32_t kb_end = span.first + from + count;
        uint32_t kb = span.first + from + wave;
        uint32_t kp = page_of(32 * kb + 8 * k_group), vp = page_of(32 * kb + 8 * g);
        u32x4 q[SETS][kQInLds ? 1 : S::kSteps];
        // (Of queries in LDS every wavefront brings its share of the steps.)
        constexpr int kMine = kQInLds ? (S::kSteps + kFewWaves - 1) / kFewWaves : S::kSteps;
        typename QueryRaw<ELEM>::type raw[SETS][kMine];
        auto step = [&](int m) { return kQInLds ? m * kFewWaves + wave : uint32_t(m); };
        auto load_queries = [&](auto on_16) {
#pragma unroll
            for (int n = 0; n < SETS; ++n) {
                const T *src = static_cast<const T *>(a.q.data) + uint64_t(span.row0 + my_row[n]) * a.q.row_stride +
                               my_head[n] * a.q.head_stride;
#pragma unroll
                for (int m = 0; m < kMine; ++m)
                    raw[n][m] = load_query<ELEM, on_16.value>(src + (EXACT || 32 * step(m) + 8 * g < d ? min(32 * step(m) + 8 * g, uint32_t(DP) - 8) : 0u));
            }
        };
        if (a.q_on_16)
            load_queries(std::true_type{});
        else
            load_queries(std::false_type{});
        FewBlock<DP> block;
        load(kb, kp, vp, block);  // (of a wavefront without a block whatever the last page holds)
        kp = page_of(32 * (kb + kFewWaves) + 8 * k_group), vp = page_of(32 * (kb + kFewWaves) + 8 * g);
        // The queries as B operands.
#pragma unroll
        for (int n = 0; n < SETS; ++n)
#pragma unroll
            for (int m = 0; m < kMine; ++m) {
                if (kQInLds && step(m) >= uint32_t(S::kSteps)) continue;
                split_query<PAGE, ELEM, NQ>(raw[n][m], v0 + n * kSet + i < vectors && (EXACT || 32 * step(m) + 8 * g < d), [&](int piece, u32x4 x) {
                    if constexpr (kQInLds)
                        lds_q[((n * NQ + piece) * S::kSteps + step(m)) * 64 + lane] = x;
                    else
                        q[n][m] = x;
                });
            }
        if constexpr (kQInLds) __syncthreads();

        float ref[SETS], threshold[SETS], sum[SETS];
        floatx4 o[SETS][S::kTiles];
#pragma unroll
        for (int n = 0; n < SETS; ++n) {
            ref[n] = 0.0f, threshold[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) o[n][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        auto multiply = [&](uint32_t kb, FewBlock<DP> &b) {
            const uint32_t key = 32 * kb + 8 * g;  // the lane's first
            if constexpr (!EXACT) {
#pragma unroll
                for (int c = 0; c < S::kSteps; ++c)
                    if (32 * c + 32 > d && 32 * c + 8 * g >= d) b.k[0][c] = b.k[1][c] = u32x4{0, 0, 0, 0};
            }
            const bool edge = 32 * kb < every_lo || 32 * kb + 32 > every_hi;  // some row does not see some key
            if (edge) {  // Rows no query of the tile sees may hold anything: they stay out of the products.
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const uint32_t keep = key + r >= some_lo && key + r < some_hi ? ~0u : 0u;
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                        for (int c = 0; c < S::kWide / 2; ++c) b.v[h][r][c] &= keep;
                }
            }
            u32x4 pieces[SETS][NP];
#pragma unroll
            for (int n = 0; n < SETS; ++n) {
                float x[8];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    floatx4 s = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < S::kSteps; ++c) {
#pragma unroll
                        for (int m = 0; m < NQ; ++m)
                            s = mfma_16x16x32<PAGE>(b.k[t][c], kQInLds ? lds_q[((n * NQ + m) * S::kSteps + c) * 64 + lane] : q[n][kQInLds ? 0 : c], s);
                        if constexpr (DP == 256) __builtin_amdgcn_sched_barrier(0);  // (registers)
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[4 * t + r] = s[r];
                }
                if (a.cap_log2 != 0.0f) {
                    if (paged_cap_by_series(ELEM, a.cap_log2)) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = softcapped<true>(x[e] * a.scale_log2, a.cap_log2, ref[n]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = softcapped<false>(x[e] * a.scale_log2, a.cap_log2, ref[n]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(x[e], a.scale_log2, -ref[n]);
                }
                if (edge) {
                    const uint32_t pos = span.position + my_row[n], lo = lowest_visible(pos, a.window, 0);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (key + e > pos || key + e < lo) x[e] = -INFINITY;
                }
                float most = max3(x[0], x[1], x[2]);
                most = max3(most, x[3], x[4]);
                most = max3(most, x[5], x[6]);
                most = fmaxf(most, x[7]);
                if (__builtin_amdgcn_ballot_w64(most > threshold[n]) != 0) {
                    const float m = max_over_groups(most);
                    const bool live = threshold[n] != -INFINITY;
                    float delta = live ? fmaxf(m - kWeightLift<PAGE>, 0.0f) : m - kWeightLift<PAGE>;
                    if (m == -INFINITY) delta = 0.0f;
                    const float alpha = live ? fast_exp2(-delta) : 1.0f;
                    ref[n] += delta;
                    if (m != -INFINITY) threshold[n] = kWeightMost;
                    sum[n] *= alpha;
#pragma unroll
                    for (int t = 0; t < S::kTiles; ++t) o[n][t] *= alpha;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] -= delta;
                }
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = fast_exp2(x[e]);
                sum[n] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                split_8<PAGE, NP>(p, pieces[n]);
            }
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (int c = 0; c < S::kWide / 2; ++c) {
                    u32x4 even, odd;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        even[r] = __builtin_amdgcn_perm(b.v[h][2 * r + 1][c], b.v[h][2 * r][c], 0x05040100u);
                        odd[r] = __builtin_amdgcn_perm(b.v[h][2 * r + 1][c], b.v[h][2 * r][c], 0x07060302u);
                    }
                    const int t = h * 8 + 2 * c;
#pragma unroll
                    for (int n = 0; n < SETS; ++n)
#pragma unroll
                        for (int m = 0; m < NP; ++m) {
                            o[n][t] = mfma_16x16x32<PAGE>(even, pieces[n][m], o[n][t]);
                            o[n][t + 1] = mfma_16x16x32<PAGE>(odd, pieces[n][m], o[n][t + 1]);
                        }
                    if constexpr (DP == 256 || SETS > 1) __builtin_amdgcn_sched_barrier(0);  // (registers)
                }
        };

        if (kb < kb_end) {
            if constexpr (kAhead) {
                for (; kb + kFewWaves < kb_end; kb += kFewWaves) {
                    FewBlock<DP> next;
                    load(kb + kFewWaves, kp, vp, next);
                    kp = page_of(32 * (kb + 2 * kFewWaves) + 8 * k_group), vp = page_of(32 * (kb + 2 * kFewWaves) + 8 * g);
                    multiply(kb, block);
                    block = next;
                }
                multiply(kb, block);
            } else {
                while (true) {
                    multiply(kb, block);
                    kb += kFewWaves;
                    if (kb >= kb_end) break;
                    load(kb, kp, vp, block);
                    kp = page_of(32 * (kb + kFewWaves) + 8 * k_group), vp = page_of(32 * (kb + kFewWaves) + 8 * g);
                }
            }
        }

        // The four wavefronts' softmaxes meet. A lane holds of its column, for r = 0 .. 3, the channels
        // kWide * (4g + r) + t of every run.
        const bool whole = count == span.blocks;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < SETS; ++n) {
            const float l = sum_over_groups(sum[n]);
            if (n == 0) __syncthreads();  // (what was there has been read)
            if (g == 0) lds_ml[wave][n * kSet + i] = make_float2(threshold[n] == -INFINITY ? -INFINITY : ref[n], l);
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < S::kWide; c += 4)
                        *reinterpret_cast<floatx4 *>(&lds_o[wave][n * kSet + i][128 * h + S::kWide * (4 * g + r) + c]) = floatx4{
                            o[n][8 * h + c][r], o[n][8 * h + c + 1][r], o[n][8 * h + c + 2][r], o[n][8 * h + c + 3][r]};
        }
        __syncthreads();
        // (A loop: code that runs once is fetched as slowly as it is long.)
#pragma unroll 1
        for (int n = 0; n < SETS; ++n) {
            constexpr int kChunk = DP / 16;  // channels a thread writes
            const uint32_t j = tid >> 4, c0 = (tid & 15) * kChunk;
            const uint32_t v = v0 + n * kSet + j;
            float2 ml[kFewWaves];
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w) ml[w] = lds_ml[w][n * kSet + j], m = fmaxf(m, ml[w].x);
            float all = 0.0f, weight[kFewWaves];
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w) {
                weight[w] = ml[w].x == -INFINITY ? 0.0f : fast_exp2(ml[w].x - m);
                all += ml[w].x == -INFINITY ? ml[w].y : weight[w] * ml[w].y;
            }
            float acc[kChunk];
#pragma unroll
            for (int c = 0; c < kChunk; ++c) acc[c] = 0.0f;
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w)
#pragma unroll
                for (int c = 0; c < kChunk; c += 4) {
                    const floatx4 x = *reinterpret_cast<const floatx4 *>(&lds_o[w][n * kSet + j][c0 + c]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[c + e] = __builtin_fmaf(weight[w], x[e], acc[c + e]);
                }
            if (v < vectors) {
                float check = all;
#pragma unroll
                for (int c = 0; c < kChunk; ++c) check += EXACT || c0 + c < d ? acc[c] : 0.0f;
                bad = bad || to_be_done_over<PAGE>(check);
                if (whole) {
                    const float inv = 1.0f / all;
                    const uint32_t row = paged_row_of(a, v), hq = head * a.group + v - row * a.group;
                    T *dst = static_cast<T *>(a.out.data) + uint64_t(span.row0 + row) * a.out.row_stride + hq * a.out.head_stride + c0;
                    typedef Piece<T, 4> Four;
#pragma unroll
                    for (int c = 0; c < kChunk; c += 4) {
                        Four y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) y.v[e] = Elem<ELEM>::from_f32(acc[c + e] * inv);
                        if (!EXACT && c0 + c >= d) break;
                        if (a.out_on_16) {
                            *reinterpret_cast<Four *>(dst + c) = y;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) dst[c + e] = y.v[e];
                        }
                    }
                } else if (blockIdx.x + unit < a.groups + a.units) {
                    const uint64_t slot = uint64_t(blockIdx.x + unit) * kTile + n * kSet + j;
#pragma unroll
                    for (int c = 0; c < kChunk; c += 4)
                        *reinterpret_cast<floatx4 *>(a.ws_acc + slot * DP + c0 + c) = floatx4{acc[c], acc[c + 1], acc[c + 2], acc[c + 3]};
                    if ((tid & 15) == 0) a.ws_ml[slot] = make_float2(m, all);
                }
            }
        }
        if (any_of_group(bad, &lds_flag)) {
            const uint32_t kb0 = span.first + from;
            paged_careful<PAGE, ELEM, DP>(a, span, head, v0, min(v0 + kTile, vectors), wave, kFewWaves, 32 * kb0, 32 * (kb0 + count),
                                          [&](uint32_t v, const float (&acc)[DP / 64], float m, float l) {
                                              paged_write_careful<PAGE, ELEM, DP>(a, span, head, v, whole, uint64_t(blockIdx.x + unit) * kTile + v - v0,
                                                                            blockIdx.x + unit < a.groups + a.units, acc, m, l);
                                          });
        }
        at += line.pad ? line.share : count;
    }
}

template <int PAGE, int ELEM, int DP, bool EXACT, int NQ, int NP>
void launch_few_as(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    // (Workgroups that would find nothing are left out where the batch is known.)
    const uint32_t groups = a.inline_items ? (a.total + a.share - 1) / a.share : a.groups;
    if (sets == 1) {
        launch_kernel(paged_few_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, 1>, groups, kFewWaves * 64, 0, stream, a);
    } else {
        launch_kernel(paged_few_kernel<PAGE, ELEM, DP, EXACT, NQ, NP, 2>, groups, kFewWaves * 64, 0, stream, a);
    }
}
template <int PAGE, int ELEM, int NQ, int NP>
hipError_t launch_few(uint32_t sets, const PagedAttn &a, hipStream_t stream) {
    const uint32_t d = a.g.head_dim;
    if (d == 64)
        launch_few_as<PAGE, ELEM, 64, true, NQ, NP>(sets, a, stream);
    else if (d < 64)
        launch_few_as<PAGE, ELEM, 64, false, NQ, NP>(sets, a, stream);
    else if (d == 128)
        launch_few_as<PAGE, ELEM, 128, true, NQ, NP>(sets, a, stream);
    else if (d < 128)
        launch_few_as<PAGE, ELEM, 128, false, NQ, NP>(sets, a, stream);
    else if (d == 256)
        launch_few_as<PAGE, ELEM, 256, true, NQ, NP>(sets, a, stream);
    else
        launch_few_as<PAGE, ELEM, 256, false, NQ, NP>(sets, a, stream);
    return hipGetLastError();
}

}  // namespace

}  // namespace itak
