// What the kernels of a paged cache share: its geometry, the batch in device memory, and how attention cuts it.
#pragma once

#include "rotation.h"

#include "paged_table.h"

namespace itak {

constexpr float kPagedLog2e = 1.4426950408889634f;
constexpr float kPagedQueryLift = 16.0f;  // paged_mfma.h
constexpr float kPagedMergeLift = 0x1p32f;  // parts with a negative sum stand for that many times themselves (paged_careful.h)
constexpr float kPagedCapShort = 256.0f * kPagedLog2e;  // paged_mfma.h
// Whether capped scores are worked out by the series (`cap_log2` > 0).
__host__ __device__ constexpr bool paged_cap_by_series(uint32_t elem, float cap_log2) {
    return elem == ITAK_ELEM_F32 || cap_log2 > kPagedCapShort;
}

// Strides in elements; side = keys or values of a page, all its heads.
struct PagedGeom {
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t page_shift;  // log2(page_rows)
    uint32_t ids_at;      // first page id's word in the batch
    uint64_t head_stride; // page_rows * head_dim
    uint64_t side_stride;
    uint64_t page_stride;
};

struct PagedAppend {
    PagedGeom g;
    const uint32_t *batch;
    uint16_t *layer_base;
    RowsView k, v;
    RotationView r;
    uint32_t q_heads;      // 0: keys and values only
    RowsView q, q_out;
    uint32_t pieces;       // of a row: queries', keys', values'
    uint32_t per_group;
};
// `page_elem`, `elem`: ITAK_ELEM_* of the pages and the tensors; `by_8`: pieces of eight channels.
hipError_t launch_paged_append(uint32_t page_elem, uint32_t elem, bool by_8, const PagedAppend &a, uint32_t rows,
                               hipStream_t stream);

// Attention. A query vector is one query head's row; the `group` query heads of a KV head times an item's rows are that KV
// head's vectors, vector v being row v / group, head v % group. A tile is `kTile` of them, a unit a tile of one KV head of one
// item: its work is the 32-key blocks from the window of the item's first row to the item's last position. All units' blocks
// in one line (items in order, in an item tile by tile, in a tile head by head) are dealt out evenly: workgroup w takes blocks w * share
// .. (w + 1) * share of the line, so that a batch of any lengths keeps every compute unit busy to the end and the grid does not
// depend on the lengths. Where that makes a share little longer, every unit's run is rounded up to a multiple of the share, so that
// no workgroup has parts of two units one after the other: a part costs some 4 us beside its blocks (one token at 4,096:
// 3.4 us more over borders than the 6.0 to 6.4 that the launch takes). A unit that one workgroup has whole is written out by it; of the others every workgroup
// leaves its partial in slot w + (unit's index), which no two parts share, and the merge launch joins them.
// The cut is worked out on the device from the batch's lengths, so a captured launch is right for whatever batch is set when it runs.
// Items that travel with a launch: an eager call whose batch has at most this many hands them over by value, and its kernels do not
// go to memory for them; one that is being captured, or has more, leaves them to the batch in device memory.
constexpr uint32_t kPagedInline = 8;
struct PagedItemWords {
    uint32_t position, rows, row0, table;
};
struct PagedAttn {
    PagedGeom g;
    const uint32_t *batch;
    const uint16_t *layer_base;
    RowsView q, out;
    uint32_t rows;       // of the batch the launch was made for
    uint32_t items;
    uint32_t group;      // query heads a KV head
    uint32_t group_magic; // ceil(2^32 / group): v / group is the high word of v * magic for v below 2^26; group 1: 0
    uint32_t tile;       // vectors, a power of two
    uint32_t tile_shift;
    uint32_t groups;     // workgroups
    uint32_t least;      // blocks a workgroup takes at least
    uint32_t units;      // of the batch the launch was made for
    uint32_t v_from, v_to; // the launch takes the items of v_from .. v_to vectors a KV head
    uint32_t q_on_16;    // every 8 channels of q start on 16 bytes
    uint32_t out_on_16;
    float scale_log2;    // scale * log2(e); with a softcap 2 * log2(e) * scale / cap; of lifted queries divided by their lift
    float cap_log2;      // cap * log2(e), 0: none
    uint32_t window;
    uint32_t parts;      // kernel of many rows: workgroups a unit is dealt to; 0: the line above
    const void *zeros;   // 16 bytes of them
    uint32_t inline_items; // 0: the batch's are read from device memory
    uint32_t total;      // with inline items: the line's length, and its cut
    uint32_t share, pad;
    PagedItemWords item[kPagedInline];  // those behind the last: row0, start and unit0 are ~0
    uint32_t start[kPagedInline], unit0[kPagedInline];  // where an item's blocks and units begin in the line
    float *ws_acc;       // [slots][tile][padded head_dim]
    float2 *ws_ml;       // [slots][tile]: maximum (log2 domain), sum; negative: of a part that is scaled down by kPagedMergeLift
};
// Workgroups that may share a unit.
constexpr uint32_t kPagedMostParts = 1024;
// The kernel of few rows (paged_few_kernel.h): tiles of `sets` times 16 vectors, 1 or 2.
constexpr uint32_t kPagedSet = 16;
// Workgroups a compute unit holds: two where a lane does with 256 registers.
__host__ __device__ constexpr uint32_t paged_few_groups_per_cu(uint32_t padded, uint32_t page_elem, uint32_t elem, uint32_t sets) {
    return padded * sets <= (page_elem == ITAK_ELEM_BF16 && elem == ITAK_ELEM_F32 ? 64 : 128) ? 2 : 1;
}
hipError_t launch_paged_few_f16(uint32_t sets, const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_few_f16_f32(uint32_t sets, const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_few_bf16(uint32_t sets, const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_few_bf16_f32(uint32_t sets, const PagedAttn &a, hipStream_t stream);
// The kernel of many rows (paged_chunk_kernel.h): 32 vectors a wavefront, four or eight wavefronts a tile.
__host__ __device__ constexpr uint32_t paged_chunk_waves(uint32_t padded, uint32_t elem) {
    return padded == 64 || (padded == 128 && elem != ITAK_ELEM_F32) ? 8 : 4;
}
// Workgroups a compute unit holds (by LDS and registers).
constexpr uint32_t kPagedChunkGroupsPerCu = 1;
// (f32 queries of 256 channels in three bf16 pieces are more registers than there are: the kernel of few rows takes them, in tiles of 32 and
// slowly: 2,048 rows over 30,720 14.4 ms, where f16 pages take 3.6.)
__host__ __device__ constexpr bool paged_chunk_takes(uint32_t padded, uint32_t page_elem, uint32_t elem) {
    return !(padded == 256 && page_elem == ITAK_ELEM_BF16 && elem == ITAK_ELEM_F32);
}
hipError_t launch_paged_chunk_f16(const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_chunk_f16_f32(const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_chunk_bf16(const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_chunk_bf16_f32(const PagedAttn &a, hipStream_t stream);
hipError_t launch_paged_merge(uint32_t elem, const PagedAttn &a, hipStream_t stream);
// head_dim as the kernels hold it.
__host__ __device__ constexpr uint32_t paged_padded(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// ---- on the device ----------------------------------------------------------------------------

struct PagedSpan {
    uint32_t position, rows, row0, table;
    uint32_t first;   // first 32-key block its rows see
    uint32_t blocks;  // of a unit
    uint32_t run;     // and with the line's rounding
    uint32_t tiles;
    uint32_t start;   // of its blocks in the line of all units'
    uint32_t unit0;   // its first unit's index
};

__host__ __device__ inline uint32_t paged_first_block(uint32_t position, uint32_t window) {
    return window && position + 1 > window ? (position + 1 - window) / 32 : 0;
}

// How the line is cut: blocks a workgroup takes, and what the units' runs are multiples of (0: of nothing). With rounded runs
// the workgroups are at most total / share + units, which is why `groups` of them do; or they are the units, where a unit is
// not much longer than a share: then nothing is split, and an eager call leaves the merge out.
struct PagedCut {
    uint32_t share, pad;
};
// Blocks that a share may be longer for lying in one unit, and for being one (64 of one token at 600 28.6 us cut evenly and
// 16.8 whole, 100 at 400 37.3 and 21.0; 16 of 8 heads at 4,096, 33 blocks a share, 52.4 and with 43 in one unit 57.3).
constexpr uint32_t kPagedPart = 8, kPagedWhole = 24;
__host__ __device__ inline PagedCut paged_cut(uint32_t total, uint32_t units, uint32_t longest, uint32_t groups, uint32_t least) {
    const uint32_t even = (total + groups - 1) / groups, share = even > least ? even : least;
    if (units <= groups && longest <= share + kPagedWhole && units * 2 >= groups) return {longest, longest};
    if (units >= groups) return {share, 0};
    const uint32_t left = groups - units, apart = (total + left - 1) / left, own = apart > least ? apart : least;
    return own <= share + kPagedPart ? PagedCut{own, own} : PagedCut{share, 0};
}
__host__ __device__ inline uint32_t paged_run(uint32_t blocks, uint32_t pad) { return pad ? (blocks + pad - 1) / pad * pad : blocks; }

#if defined(__HIPCC__)

__device__ __forceinline__ uint32_t paged_row_of(const PagedAttn &a, uint32_t vector) {
    return a.group_magic ? __umulhi(vector, a.group_magic) : vector;
}

// Asks for all of the arguments at once: the compiler asks where it needs them, a trip to memory for every 64 bytes that come
// first there (of the few rows' kernel four in a row, some 3,000 clocks before the first page id).
__device__ __forceinline__ void paged_fetch_arguments(const PagedAttn &a) {
    static_assert(sizeof(PagedAttn) <= 9 * 64 && kPagedInline == 8, "a word of every 64 bytes is named");
    asm volatile("" ::"s"(a.batch), "s"(a.layer_base), "s"(a.q.data), "s"(a.out.data), "s"(a.rows), "s"(a.units), "s"(a.v_to), "s"(a.window),
                 "s"(a.zeros), "s"(a.total), "s"(a.item[1].row0), "s"(a.item[5].row0), "s"(a.start[1]), "s"(a.unit0[1]), "s"(a.ws_acc),
                 "s"(a.ws_ml));
}

// The items a launch takes, in order: where their blocks and units lie in the line. Those in memory are looked at 64 at a time, one
// a lane.
struct PagedLine {
    const PagedAttn &a;
    uint32_t share = 0, pad = 0, total = 0;

    __device__ __forceinline__ explicit PagedLine(const PagedAttn &args) : a(args) {}
    // An item's span, and blocks and units of all of it; none of an item that the launch does not take, and of one beyond the
    // launch's rows (a batch that is not what a captured launch was made for).
    __device__ __forceinline__ PagedSpan span_of(const PagedItemWords &w, bool there, uint32_t &work, uint32_t &units) const {
        PagedSpan s{};
        work = units = 0;
        const uint32_t vectors = w.rows * a.group;
        if (there && w.row0 + w.rows <= a.rows && w.rows && vectors >= a.v_from && vectors <= a.v_to) {
            s.position = w.position, s.rows = w.rows, s.row0 = w.row0, s.table = w.table;
            s.first = paged_first_block(w.position, a.window);
            s.blocks = (w.position + w.rows + 31) / 32 - s.first;
            s.tiles = (vectors + (1u << a.tile_shift) - 1) >> a.tile_shift;
            units = s.tiles * a.g.kv_heads;
            s.run = paged_run(s.blocks, pad);
            work = units * s.run;
        }
        return s;
    }
    __device__ __forceinline__ PagedSpan of_lane(uint32_t at, uint32_t n, uint32_t &work, uint32_t &units) const {
        PagedItemWords w{};
        const bool there = at + __lane_id() < n;
        if (there) {
            const uint4 x = *reinterpret_cast<const uint4 *>(a.batch + kPagedItem0 + 4 * (at + __lane_id()));
            w.position = x.x, w.rows = x.y, w.row0 = x.z, w.table = x.w;
        }
        return span_of(w, there, work, units);
    }
    static __device__ __forceinline__ uint32_t scan(uint32_t x) {  // inclusive, over the wavefront
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(x, d);
            x += (__lane_id() >= uint32_t(d)) ? y : 0;
        }
        return x;
    }
    static __device__ __forceinline__ uint32_t most_of(uint32_t x) {  // over the wavefront
#define ITAK_MOST(ctrl) x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), ctrl, 0xf, 0xf, true)))
        ITAK_MOST(0xB1), ITAK_MOST(0x4E), ITAK_MOST(0x141), ITAK_MOST(0x140);  // (of sixteen lanes)
#undef ITAK_MOST
        const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
        const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
        return max(max(a, b), max(c, d));
    }
    // The cut; before anything that counts blocks.
    __device__ __forceinline__ void cut() {
        if (a.inline_items) {
            share = a.share, pad = a.pad, total = a.total;
            return;
        }
        const uint32_t n = min(a.batch[0], a.items);
        uint32_t all = 0, all_units = 0, longest = 0;
        for (uint32_t at = 0; at < n; at += 64) {
            uint32_t work, units;
            const PagedSpan s = of_lane(at, n, work, units);
            all += __builtin_amdgcn_readlane(scan(work), 63);
            all_units += __builtin_amdgcn_readlane(scan(units), 63);
            longest = max(longest, s.blocks);
        }
        longest = most_of(longest);
        const PagedCut c = paged_cut(all, all_units, longest, a.groups, a.least);
        share = c.share, pad = c.pad, total = pad ? share * a.groups : all;  // (of rounded runs: what lies past the last is nobody's)
    }
    // The item that block, unit or row x of the line belongs to; none if it is no item's, or of one that the launch does not take.
    enum By { kBlock, kUnit, kRow };
    template <By BY>
    __device__ __forceinline__ bool find(PagedSpan &out, uint32_t x) const {
        auto holds = [&](const PagedSpan &s, uint32_t work, uint32_t units) {
            if (BY == kBlock) return x >= s.start && x - s.start < work;
            if (BY == kUnit) return x >= s.unit0 && x - s.unit0 < units;
            return work != 0 && x >= s.row0 && x - s.row0 < s.rows;
        };
        uint32_t before = 0, units_before = 0;
        if (a.inline_items) {
            uint32_t at = 0;  // (of several that begin there all but the last are empty)
#pragma unroll
            for (uint32_t i = 1; i < kPagedInline; ++i)
                at = x >= (BY == kBlock ? a.start[i] : BY == kUnit ? a.unit0[i] : a.item[i].row0) ? i : at;
            uint32_t work, units;
            out = span_of(a.item[at], true, work, units);
            out.start = a.start[at], out.unit0 = a.unit0[at];
            return holds(out, work, units);
        }
        const uint32_t n = min(a.batch[0], a.items);
        for (uint32_t at = 0; at < n; at += 64) {
            uint32_t work, units;
            PagedSpan s = of_lane(at, n, work, units);
            const uint32_t upto = scan(work), units_upto = scan(units);
            s.start = before + upto - work;
            s.unit0 = units_before + units_upto - units;
            const uint64_t mask = __builtin_amdgcn_ballot_w64(holds(s, work, units));
            if (mask) {
                const uint32_t l = __builtin_ctzll(mask);
#define ITAK_FIELD(f) out.f = __builtin_amdgcn_readlane(s.f, l)
                ITAK_FIELD(position), ITAK_FIELD(rows), ITAK_FIELD(row0), ITAK_FIELD(table), ITAK_FIELD(first);
                ITAK_FIELD(blocks), ITAK_FIELD(run), ITAK_FIELD(tiles), ITAK_FIELD(start), ITAK_FIELD(unit0);
#undef ITAK_FIELD
                return true;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
            units_before += __builtin_amdgcn_readlane(units_upto, 63);
        }
        return false;
    }
};

// The batch's item that holds row `row`: its position, first row and table. All lanes ask together.
__device__ __forceinline__ bool paged_item_of_row(const uint32_t *batch, uint32_t row, uint4 &item) {
    const uint32_t n = batch[0], lane = __lane_id();
    for (uint32_t at = 0; at < n; at += 64) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (at + lane < n) w = *reinterpret_cast<const uint4 *>(batch + kPagedItem0 + 4 * (at + lane));
        const uint64_t mask = __builtin_amdgcn_ballot_w64(row >= w.z && row - w.z < w.y);
        if (mask) {
            const uint32_t l = __builtin_ctzll(mask);
            item.x = __builtin_amdgcn_readlane(w.x, l), item.y = __builtin_amdgcn_readlane(w.y, l);
            item.z = __builtin_amdgcn_readlane(w.z, l), item.w = __builtin_amdgcn_readlane(w.w, l);
            return true;
        }
    }
    return false;
}

#endif

}  // namespace itak
