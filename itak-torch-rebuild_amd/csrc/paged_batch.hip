// A batch made on the device: the records of trees, items and page ids from lengths and page tables that lie there, and the tables
// themselves, which take their pages from a free list and give them back.
//
// All of it is a few words a sequence and a row; what it costs are launches and, inside one, the trips to memory that wait for one another.
// A workgroup serves a sequence and finds out for itself what stands before it (a sum over up to 1,024 lengths that lie in the cache),
// so that a batch is one launch; the free list is one workgroup's, which every sequence's place in it has to pass through.
#include "paged_handle.h"

#include <algorithm>

using namespace itak;

namespace itak {

namespace {

constexpr uint32_t kThreads = 256;

__device__ __forceinline__ uint64_t wave_sum(uint64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// An item's records from its parents; `up`: kTreeRows words of LDS. All of a workgroup's threads ask. False, and nothing written, where they are no tree's: a parent that is no
// row before and not -1, or more rows than a tree may have that are no chain.
__device__ __forceinline__ bool make_records(uint32_t *tree, const int32_t *parents, uint32_t rows, uint32_t position, int32_t *up) {
    const uint32_t tid = threadIdx.x;
    bool other = false, wrong = false;
    int32_t mine = 0;
    for (uint32_t r = tid; r < rows; r += kThreads) {
        const int32_t parent = parents[r];
        if (r == tid) mine = parent;
        other = other || parent != int32_t(r) - 1;
        wrong = wrong || parent < -1 || parent >= int32_t(r);
    }
    if (tid < kTreeRows) up[tid] = mine;
    if (__syncthreads_or(wrong)) return false;
    if (!__syncthreads_or(other)) {
        for (uint32_t r = tid; r < rows; r += kThreads) {
            tree[uint64_t(r) * kTreeStride + kTreeDepth] = kTreeChain | r;
            tree[uint64_t(r) * kTreeStride + kTreeParent] = r - 1;
        }
        return true;
    }
    if (rows > kTreeRows) return false;
    if (tid < rows) {
        // Upwards from the row: every step goes to a lower row, so there are at most as many steps as rows.
        const uint32_t held = position % 32;
        uint32_t word[kTreeBlocks], depth = 0;
#pragma unroll
        for (uint32_t w = 0; w < kTreeBlocks; ++w) word[w] = w == 0 ? (1u << held) - 1 : 0;
        for (int32_t at = int32_t(tid); at >= 0; at = up[at], ++depth) {
            const uint32_t bit = held + uint32_t(at);
#pragma unroll
            for (uint32_t w = 0; w < kTreeBlocks; ++w) word[w] |= bit / 32 == w ? 1u << bit % 32 : 0u;
        }
        uint32_t *const record = tree + uint64_t(tid) * kTreeStride;
        record[kTreeDepth] = depth - 1;
        record[kTreeParent] = uint32_t(up[tid]);
#pragma unroll
        for (uint32_t w = 0; w < kTreeBlocks; ++w) record[kTreeSees + w] = word[w];
    }
    return true;
}

__global__ __launch_bounds__(kThreads) void paged_records_kernel(const uint32_t *batch, const int32_t *parents, uint32_t *tree) {
    __shared__ int32_t up[kTreeRows];
    const uint4 item = *reinterpret_cast<const uint4 *>(batch + kPagedItem0 + 4 * blockIdx.x);
    (void)make_records(tree + uint64_t(item.z) * kTreeStride, parents + item.z, item.y, item.x, up);
}

// Rows of every sequence travel with the launch, or lie at rows_at where they are more.
constexpr uint32_t kRowsInline = 256;
struct DeviceBatch {
    uint32_t *batch;
    uint32_t *tree;
    const int32_t *parents;    // null: no trees
    const int32_t *positions;
    const uint32_t *table;
    uint64_t stride;
    const int32_t *held;       // pages of every sequence
    int32_t *status;           // null: not asked for
    const uint32_t *rows_at;
    uint32_t sequences, rows;
    uint32_t page_shift;
    uint32_t page_count;
    uint32_t most_positions;
    uint32_t ids_at;
    uint64_t ids_room;
    uint32_t inline_rows[kRowsInline];
};
__device__ __forceinline__ uint32_t rows_of(const DeviceBatch &a, uint32_t i) { return a.rows_at ? a.rows_at[i] : a.inline_rows[i]; }

__global__ __launch_bounds__(kThreads) void paged_device_batch_kernel(DeviceBatch a) {
    __shared__ uint64_t sums[2][kThreads / 64];
    __shared__ int32_t up[kTreeRows];
    const uint32_t i = blockIdx.x, tid = threadIdx.x;
    // What a sequence's positions are refused for, and the pages that they take otherwise.
    auto pages_of = [&](uint32_t s, uint32_t rows, uint32_t &pages) {
        pages = 0;
        if (!rows) return ITAK_TABLE_OK;
        const int32_t position = a.positions[s], held = a.held[s];
        if (position < 0 || uint32_t(position) > a.most_positions) return ITAK_TABLE_POSITION;
        const uint32_t need = (uint32_t(position) + rows + (1u << a.page_shift) - 1) >> a.page_shift;
        if (held < 0 || need > uint32_t(held) || uint32_t(held) > a.stride) return ITAK_TABLE_PAGES;
        pages = need;
        return ITAK_TABLE_OK;
    };
    uint64_t row0 = 0, id0 = 0;
    for (uint32_t s = tid; s < i; s += kThreads) {
        const uint32_t rows = rows_of(a, s);
        uint32_t pages;
        (void)pages_of(s, rows, pages);
        row0 += rows, id0 += pages;
    }
    row0 = wave_sum(row0), id0 = wave_sum(id0);
    if ((tid & 63) == 0) sums[0][tid / 64] = row0, sums[1][tid / 64] = id0;
    __syncthreads();
    row0 = id0 = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) row0 += sums[0][w], id0 += sums[1][w];
    const uint32_t rows = rows_of(a, i);
    uint32_t pages;
    int32_t status = pages_of(i, rows, pages);
    if (status == ITAK_TABLE_OK && id0 + pages > a.ids_room) status = ITAK_TABLE_ROOM;
    const uint32_t position = status == ITAK_TABLE_OK && rows ? uint32_t(a.positions[i]) : 0;
    uint32_t *const ids = a.batch + a.ids_at + id0;
    bool wrong = false;
    if (status == ITAK_TABLE_OK)
        for (uint32_t p = tid; p < pages; p += kThreads) {
            const uint32_t id = a.table[i * a.stride + p];
            wrong = wrong || id >= a.page_count;
            ids[p] = id;
        }
    if (__syncthreads_or(wrong)) status = ITAK_TABLE_ID;
    if (a.parents && status == ITAK_TABLE_OK &&
        !make_records(a.tree + row0 * kTreeStride, a.parents + row0, rows, position, up))
        status = ITAK_TABLE_PARENTS;
    if (tid == 0) {
        const bool in = status == ITAK_TABLE_OK;
        *reinterpret_cast<uint4 *>(a.batch + kPagedItem0 + 4 * i) =
            make_uint4(in ? position : 0, in ? rows : 0, uint32_t(row0), a.ids_at + uint32_t(in ? id0 : 0));
        if (a.status) a.status[i] = status;
        if (i == 0) a.batch[0] = a.sequences, a.batch[1] = a.rows, a.batch[2] = a.parents ? 1 : 0, a.batch[3] = 0;
    }
}

// Every row's position in the text and its row in the storage; -1 of rows that the batch does not take.
struct BatchRows {
    const uint32_t *batch;
    const uint32_t *tree;
    uint32_t page_shift;
    uint32_t rows;
    int64_t *positions, *slots;
};
__global__ __launch_bounds__(kThreads) void paged_batch_rows_kernel(BatchRows a) {
    const uint32_t n = min(a.batch[0], gridDim.x), i = blockIdx.x;
    if (i >= n) return;
    const uint4 item = *reinterpret_cast<const uint4 *>(a.batch + kPagedItem0 + 4 * i);
    const uint32_t end = min(a.rows, i + 1 < n ? a.batch[kPagedItem0 + 4 * (i + 1) + 2] : a.batch[1]);
    const bool trees = a.tree && a.batch[2];
    for (uint32_t row = item.z + threadIdx.x; row < end; row += kThreads) {
        const uint32_t r = row - item.z, place = item.x + r;
        int64_t position = -1, slot = -1;
        if (r < item.y) {
            position = item.x + (trees ? tree_depth(a.tree[uint64_t(row) * kTreeStride]) : r);
            slot = (int64_t(a.batch[item.w + (place >> a.page_shift)]) << a.page_shift) + (place & ((1u << a.page_shift) - 1));
        }
        if (a.positions) a.positions[row] = position;
        if (a.slots) a.slots[row] = slot;
    }
}

// Page tables that grow and shrink to lengths. Pages given back come onto the free list's end in the order in which taking them from
// there finds them again; then sequences take theirs from the end, the first ones first.
constexpr uint32_t kFitThreads = 1024;
struct FitTables {
    uint32_t *table;
    uint64_t stride;
    int32_t *held;
    uint32_t *free_ids;
    int32_t *free_count;
    const int32_t *lengths;
    int32_t *status;
    const uint32_t *rows_at;
    uint32_t sequences;
    uint32_t page_shift;
    uint32_t page_count;
    uint32_t plus_rows;        // whether rows come on top of the lengths
    uint32_t inline_rows[kRowsInline];
};
// Inclusive sums over the workgroup; `sums` is kFitThreads / 64 words of LDS, which the caller lets go of behind a barrier.
__device__ __forceinline__ uint64_t scan_all(uint64_t x, uint64_t *sums) {
    const uint32_t lane = __lane_id(), wave = threadIdx.x / 64;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up(x, d);
        x += lane >= uint32_t(d) ? y : 0;
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) x += sums[w];
    return x;
}
__global__ __launch_bounds__(kFitThreads) void paged_fit_kernel(FitTables a) {
    __shared__ uint64_t sums[2][kFitThreads / 64];
    __shared__ uint64_t ends[kFitThreads];   // of every sequence's pages among those that move
    __shared__ uint32_t from[kFitThreads];   // its first of them
    const uint32_t i = threadIdx.x, n = a.sequences;
    int32_t status = ITAK_TABLE_OK;
    uint32_t held = 0, need = 0;
    if (i < n) {
        const int32_t length = a.lengths[i], have = a.held[i];
        const uint64_t rows = !a.plus_rows ? 0 : a.rows_at ? a.rows_at[i] : a.inline_rows[i];
        const uint64_t want = (uint64_t(uint32_t(length)) + rows + (1u << a.page_shift) - 1) >> a.page_shift;
        if (have < 0 || uint64_t(have) > a.stride)
            status = ITAK_TABLE_PAGES;
        else if (length < 0 || want > a.stride)
            status = ITAK_TABLE_POSITION;
        else
            held = uint32_t(have), need = uint32_t(want);
    }
    const int32_t said = *a.free_count;
    const bool sound = said >= 0 && uint32_t(said) <= a.page_count;
    const uint64_t count = sound ? uint32_t(said) : 0;
    // Back: page `from + k` of a sequence is number `before + k` of all that go, and lies that far from the list's end when they have come.
    const uint64_t back = need < held ? held - need : 0, back_end = scan_all(back, sums[0]);
    ends[i] = back_end, from[i] = need;
    __syncthreads();
    const uint64_t all_back = ends[kFitThreads - 1];
    const bool room = sound && count + all_back <= a.page_count;
    // The sequence that has number x of the pages that move, and which of its own that is.
    auto owner = [&](uint64_t x, uint64_t &own) {
        uint32_t s = 0;
#pragma unroll
        for (uint32_t step = kFitThreads / 2; step; step /= 2)
            if (ends[s + step - 1] <= x) s += step;
        own = x - (s ? ends[s - 1] : 0) + from[s];
        return s;
    };
    if (room)
        for (uint64_t x = i; x < all_back; x += kFitThreads) {
            uint64_t own;
            const uint32_t s = owner(x, own);
            a.free_ids[count + all_back - 1 - x] = a.table[s * a.stride + own];
        }
    __syncthreads();  // (what was given back is there to be taken)
    const uint64_t have_free = count + all_back;
    uint64_t take = room && need > held ? need - held : 0;
    const uint64_t take_end = scan_all(take, sums[1]);
    const bool granted = take_end <= have_free;
    // (Sequences behind one that goes without do so too where they take any: what they would get depends on nobody else's being refused.)
    if (take && !granted) status = ITAK_TABLE_FREE;
    if (!room && status == ITAK_TABLE_OK && need != held) status = ITAK_TABLE_FREE;
    const uint64_t grant_end = granted ? take_end : 0;
    ends[i] = take_end, from[i] = held;
    __syncthreads();
    // Sequences are granted in order: all up to the last whose sum fits.
    uint64_t all_taken = grant_end;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor(all_taken, o);
        all_taken = y > all_taken ? y : all_taken;
    }
    if (__lane_id() == 0) sums[0][i / 64] = all_taken;
    __syncthreads();
    for (uint32_t w = 0; w < kFitThreads / 64; ++w) all_taken = sums[0][w] > all_taken ? sums[0][w] : all_taken;
    for (uint64_t x = i; x < all_taken; x += kFitThreads) {
        uint64_t own;
        const uint32_t s = owner(x, own);
        a.table[s * a.stride + own] = a.free_ids[have_free - 1 - x];
    }
    if (i < n) {
        if (room && status == ITAK_TABLE_OK) a.held[i] = int32_t(need);
        if (a.status) a.status[i] = status;
    }
    if (i == 0 && room) *a.free_count = int32_t(have_free - all_taken);
}

}  // namespace

hipError_t launch_paged_records(const uint32_t *batch, uint32_t items, const int32_t *parents, uint32_t *tree, hipStream_t stream) {
    launch_kernel(paged_records_kernel, items, kThreads, 0, stream, batch, parents, tree);
    return hipGetLastError();
}

}  // namespace itak

namespace {

itak_status check_tables(itak_paged *p, const itak_page_tables *t) {
    if (!t) return invalid_argument(p->err, "tables are null");
    if (t->sequences == 0) return zero_dimension(p->err, "sequences");
    if (t->sequences > p->cfg.max_sequences)
        return set_error(p->err, ITAK_CAPACITY_EXCEEDED, "sequences", t->sequences, p->cfg.max_sequences, 0, 0,
                         "page tables of %u sequences, the paged cache takes %u", t->sequences, p->cfg.max_sequences);
    if (!t->table || !t->pages) return invalid_argument(p->err, "table or pages are null");
    if (t->stride == 0) return zero_dimension(p->err, "stride");
    if (t->stride > (1ull << 28)) return size_overflow(p->err, "stride");
    return ITAK_OK;
}

// Every sequence's rows: with the launch, or in the handle's memory where they are more than that takes.
itak_status place_rows(itak_paged *p, const uint32_t *rows, uint32_t n, uint32_t *inline_rows, const uint32_t **rows_at) {
    *rows_at = nullptr;
    if (n <= kRowsInline) {
        std::copy(rows, rows + n, inline_rows);
        return ITAK_OK;
    }
    uint32_t *const there = p->rows_dev;
    for (uint32_t at = 0; at < n; at += kManyWords) send_words(there, at, rows + at, std::min(n - at, kManyWords), 0, nullptr, 0, p->stream);
    *rows_at = there;
    return ITAK_OK;
}

}  // namespace

extern "C" {

itak_status itak_paged_enable_trees(itak_paged *paged, uint64_t most_rows) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    if (most_rows == 0) return zero_dimension(paged->err, "most_rows");
    if (most_rows > kPagedMostRows) return size_overflow(paged->err, "most_rows");
    if (paged->tree_dev) return invalid_argument(paged->err, "trees are enabled already");
    if (capturing(paged->stream)) return invalid_argument(paged->err, "trees are enabled while the stream is being captured");
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    const uint64_t words = most_rows * (kTreeStride + 1);
    void *at = nullptr;
    HIP_TRY(paged, hipMalloc(&at, words * sizeof(uint32_t)), "allocate the records of trees");
    hipError_t he = hipMemset(at, 0, words * sizeof(uint32_t));
    if (he == hipSuccess) he = hipDeviceSynchronize();  // (whatever stream comes first finds it)
    if (he != hipSuccess) {
        (void)hipFree(at);
        return hip_error(paged->err, he, "clear the records of trees");
    }
    paged->tree_dev = static_cast<uint32_t *>(at);
    paged->tree_rows = most_rows;
    return ITAK_OK;
}

itak_status itak_paged_fit_tables_device(itak_paged *paged, const itak_page_tables *tables, const int32_t *lengths_dev, const uint32_t *rows,
                                         int32_t *status_dev) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_tables(paged, tables);
    if (st != ITAK_OK) return st;
    if (!tables->free_ids || !tables->free_count) return invalid_argument(paged->err, "free_ids or free_count are null");
    if (!lengths_dev) return invalid_argument(paged->err, "lengths are null");
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    FitTables a{};
    if (rows) st = place_rows(paged, rows, tables->sequences, a.inline_rows, &a.rows_at);
    if (st != ITAK_OK) return st;
    a.table = tables->table, a.stride = tables->stride, a.held = tables->pages;
    a.free_ids = tables->free_ids, a.free_count = tables->free_count;
    a.lengths = lengths_dev, a.status = status_dev;
    a.sequences = tables->sequences;
    a.page_shift = paged->g.page_shift;
    a.page_count = uint32_t(paged->cfg.page_count);
    a.plus_rows = rows != nullptr;
    launch_kernel(paged_fit_kernel, 1, kFitThreads, 0, paged->stream, a);
    HIP_TRY(paged, hipGetLastError(), "launch the fitting of page tables");
    return ITAK_OK;
}

itak_status itak_paged_set_batch_device(itak_paged *paged, const itak_page_tables *tables, const int32_t *positions_dev, const uint32_t *rows,
                                        uint64_t most_positions, const int32_t *parents_dev, int32_t *status_dev) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_tables(paged, tables);
    if (st != ITAK_OK) return st;
    if (!positions_dev || !rows) return invalid_argument(paged->err, "positions or rows are null");
    const uint32_t n = tables->sequences;
    uint64_t all = 0;
    uint32_t most = 0, tree_most = 0;
    for (uint32_t i = 0; i < n; ++i) {
        all += rows[i];
        most = std::max(most, rows[i]);
        if (parents_dev && rows[i] <= kTreeRows && rows[i] > 1) tree_most = std::max(tree_most, rows[i]);
    }
    if (most_positions >= (1ull << 31) || most_positions + most >= (1ull << 31)) return size_overflow(paged->err, "most_positions");
    if (all > kPagedMostRows) return size_overflow(paged->err, "rows");
    if (parents_dev && !paged->tree_dev)
        return unsupported(paged->err, "a batch of trees of a paged cache that takes none (itak_paged_enable_trees)");
    if (parents_dev && all > paged->tree_rows)
        return set_error(paged->err, ITAK_CAPACITY_EXCEEDED, "rows of trees", all, paged->tree_rows, 0, 0,
                         "a batch of trees of %llu rows, the paged cache takes %llu", ULL(all), ULL(paged->tree_rows));
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    try {
        // What the host knows of the batch: every sequence at the most positions it may have.
        PagedBatch &next = paged->next;
        next.head.assign(kPagedItem0, 0);
        next.ids.clear();
        next.items = n, next.rows = uint32_t(all), next.most_rows = most;
        next.trees = parents_dev != nullptr, next.tree_most = tree_most, next.on_device = true, next.sized[0] = next.sized[1] = 0;
        uint32_t row0 = 0;
        for (uint32_t i = 0; i < n; row0 += rows[i], ++i) {
            const uint32_t words[4] = {uint32_t(most_positions), rows[i], row0, 0};
            next.head.insert(next.head.end(), words, words + 4);
        }
        next.head[0] = n, next.head[1] = next.rows, next.head[2] = next.trees;
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
    if (!paged_replays_hold(paged, paged->next)) return size_overflow(paged->err, "a captured attention over the batch");
    DeviceBatch a{};
    st = place_rows(paged, rows, n, a.inline_rows, &a.rows_at);
    if (st != ITAK_OK) return st;
    a.batch = paged->batch_dev, a.tree = paged->tree_dev;
    a.parents = parents_dev, a.positions = positions_dev;
    a.table = tables->table, a.stride = tables->stride, a.held = tables->pages;
    a.status = status_dev;
    a.sequences = n, a.rows = uint32_t(all);
    a.page_shift = paged->g.page_shift;
    a.page_count = uint32_t(paged->cfg.page_count);
    a.most_positions = uint32_t(most_positions);
    a.ids_at = paged->g.ids_at, a.ids_room = paged->cfg.max_table_pages;
    // (The ids that the device has are the tables' from now on, and of a graph's replays whenever they run.)
    paged->ids_known = false;
    if (capturing(paged->stream)) paged->ids_never_known = true;
    launch_kernel(paged_device_batch_kernel, n, kThreads, 0, paged->stream, a);
    if (const hipError_t he = hipGetLastError(); he != hipSuccess) {
        paged->batch = PagedBatch{};
        return hip_error(paged->err, he, "launch the making of a batch");
    }
    std::swap(paged->batch, paged->next);
    return ITAK_OK;
}

itak_status itak_paged_batch_rows_device(itak_paged *paged, int64_t *positions_dev, int64_t *slots_dev) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    if (!positions_dev && !slots_dev) return invalid_argument(paged->err, "positions and slots are null");
    if (paged->batch.rows == 0) return ITAK_OK;
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    const BatchRows a{paged->batch_dev, paged->tree_dev, paged->g.page_shift, paged->batch.rows, positions_dev, slots_dev};
    launch_kernel(paged_batch_rows_kernel, paged->batch.items, kThreads, 0, paged->stream, a);
    HIP_TRY(paged, hipGetLastError(), "launch the rows of a batch");
    return ITAK_OK;
}

}  // extern "C"
