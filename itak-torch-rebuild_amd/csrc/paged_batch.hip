// A batch made on the device: the records of trees, items and page ids from lengths and page tables that lie there, and the tables
// themselves, which take their pages from a free list and give them back.
//
// All of it is a few words a sequence and a row; what it costs are launches and, inside one, the trips to memory that wait for one another.
// A workgroup serves a sequence and finds out for itself what stands before it (a sum over up to 1,024 lengths),
// so that a batch is one launch; the free list is one workgroup's, which every sequence's place in it has to pass through. Of 4 sequences the
// tables take 3.0 us, the batch with trees of 16 rows 4.0 and the rows 2.1; of 256 at up to 32,768, trees of 64 rows, 3.7, 5.2 and 3.1.
#include "mfma_common.h"
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

// The bits that any of a workgroup's threads has; all of them ask. `words`: a word a wavefront, another call's others.
__device__ __forceinline__ uint32_t any_bits(uint32_t mine, uint32_t *words) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine |= __shfl_xor(mine, o);
    if ((threadIdx.x & 63) == 0) words[threadIdx.x / 64] = mine;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) all |= words[w];
    return all;
}

// What parents are not: row 0's and so on those of a chain, and of a tree (a row before, or -1).
constexpr uint32_t kNoChain = 1, kNoTree = 2;
__device__ __forceinline__ uint32_t parent_is_not(int32_t parent, uint32_t r) {
    return (parent != int32_t(r) - 1 ? kNoChain : 0) | (parent < -1 || parent >= int32_t(r) ? kNoTree : 0);
}
// An item's records from its parents, the threads' rows' in `up` (LDS) where it is a tree; `not_`: what any of them is not, no kNoTree. What a row sees
// is doubled: its nearest 2^k rows upwards and as many of the row behind them are its nearest 2^(k+1). (The whole launch over 255 rows in one line and one
// beside took 28.2 us upwards row by row, and 6.2; over 32 5.6 and 2.4; over 256 rows of at most 20 levels 3.2 and 4.6, the one that loses.)
__device__ __forceinline__ void make_records(uint32_t *tree, uint32_t rows, uint32_t position, uint32_t not_, const int32_t *up) {
    __shared__ int32_t lds_at[kTreeRows];
    __shared__ u32x4 lds_sees[2][kTreeRows];
    const uint32_t tid = threadIdx.x;
    if (!not_) {
        for (uint32_t r = tid; r < rows; r += kThreads)
            *reinterpret_cast<uint2 *>(tree + uint64_t(r) * kTreeStride) = make_uint2(kTreeChain | r, r - 1);
        return;
    }
    constexpr uint32_t kWords = kTreeRows / 32;
    uint32_t sees[kWords];
    const int32_t parent = tid < rows ? up[tid] : -1;
    int32_t at = parent;
    if (rows <= 64) {
        // (One wavefront, in its registers.)
        if (tid >= 64) return;
        uint64_t mine = 1ull << tid;
        while (__builtin_amdgcn_ballot_w64(at >= 0) != 0) {
            const int32_t from = max(at, 0);
            const uint64_t theirs = __shfl(mine, from);
            const int32_t next = __shfl(at, from);
            if (at >= 0) mine |= theirs, at = next;
        }
#pragma unroll
        for (uint32_t w = 0; w < kWords; ++w) sees[w] = w < 2 ? uint32_t(mine >> (32 * w)) : 0;
    } else {
#pragma unroll
        for (uint32_t w = 0; w < kWords; ++w) sees[w] = tid / 32 == w ? 1u << tid % 32 : 0;
        // (Behind each of the two barriers everybody has read, or written.)
        while (__syncthreads_or(at >= 0)) {
            lds_at[tid] = at;
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x) lds_sees[x][tid] = u32x4{sees[4 * x], sees[4 * x + 1], sees[4 * x + 2], sees[4 * x + 3]};
            __syncthreads();
            if (at < 0) continue;
#pragma unroll
            for (uint32_t w = 0; w < kWords; ++w) sees[w] |= lds_sees[w / 4][at][w % 4];
            at = lds_at[at];
        }
    }
    if (tid >= rows) return;
    const uint32_t held = position % 32;
    uint32_t word[kTreeStride] = {}, seen = 0;
    word[kTreeParent] = uint32_t(parent);
#pragma unroll
    for (uint32_t w = 0; w < kTreeBlocks; ++w) {
        // (Row r is bit held + r.)
        const uint64_t pair = uint64_t(w < kWords ? sees[w] : 0) << 32 | (w ? sees[w - 1] : 0);
        word[kTreeSees + w] = uint32_t(pair >> (32 - held)) | (w ? 0 : (1u << held) - 1);
        seen += w < kWords ? __builtin_popcount(sees[w]) : 0;
    }
    word[kTreeDepth] = seen - 1;
#pragma unroll
    for (uint32_t w = 0; w < kTreeStride; w += 4)
        *reinterpret_cast<uint4 *>(tree + uint64_t(tid) * kTreeStride + w) = make_uint4(word[w], word[w + 1], word[w + 2], word[w + 3]);
}

// A batch of trees on its way to the device: its words as those of paged.hip travel, and the parents behind them. A workgroup makes an item's
// records, and the first stores the words besides.
template <uint32_t N>
struct TreeWords {
    uint32_t *batch, *tree;
    uint32_t n0;       // words of header and items
    uint32_t at1, n1;  // page ids, and where they go
    uint32_t pad;
    uint32_t w[N];     // and then the parents
};
template <uint32_t N>
__global__ __launch_bounds__(kThreads) void paged_tree_words_kernel(TreeWords<N> a) {
    __shared__ int32_t up[kTreeRows];
    __shared__ uint32_t words[kThreads / 64];
    const uint32_t tid = threadIdx.x;
    // (The arguments by their address: indexed as a value they would be copied first.)
    const uint32_t *const w = reinterpret_cast<const uint32_t *>(reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()) + offsetof(TreeWords<N>, w));
    const uint32_t *const item = w + kPagedItem0 + 4 * blockIdx.x;
    if (blockIdx.x == 0)
        for (uint32_t i = tid; i < a.n0 + a.n1; i += kThreads) a.batch[i < a.n0 ? i : a.at1 + (i - a.n0)] = w[i];
    const uint32_t position = item[0], rows = item[1], row0 = item[2];
    if (kPagedItem0 + 4 * blockIdx.x >= a.n0) return;  // (a batch without items)
    const int32_t *const parents = reinterpret_cast<const int32_t *>(w) + a.n0 + a.n1 + row0;
    uint32_t not_ = 0;
    for (uint32_t r = tid; r < rows; r += kThreads) {
        const int32_t parent = parents[r];
        if (r == tid && tid < kTreeRows) up[tid] = parent;
        not_ |= parent_is_not(parent, r);
    }
    not_ = any_bits(not_, words);
    make_records(a.tree + uint64_t(row0) * kTreeStride, rows, position, not_, up);
}

__global__ __launch_bounds__(kThreads) void paged_records_kernel(const uint32_t *batch, const int32_t *all_parents, uint32_t *tree) {
    __shared__ int32_t up[kTreeRows];
    __shared__ uint32_t words[kThreads / 64];
    const uint32_t tid = threadIdx.x;
    const uint4 item = *reinterpret_cast<const uint4 *>(batch + kPagedItem0 + 4 * blockIdx.x);
    const int32_t *const parents = all_parents + item.z;
    uint32_t not_ = 0;
    for (uint32_t r = tid; r < item.y; r += kThreads) {
        const int32_t parent = parents[r];
        if (r == tid && tid < kTreeRows) up[tid] = parent;
        not_ |= parent_is_not(parent, r);
    }
    not_ = any_bits(not_, words);
    make_records(tree + uint64_t(item.z) * kTreeStride, item.y, item.x, not_, up);
}

// Rows of every sequence, and the first of them among the batch's, travel with the launch, or lie at rows_at where they are more. (Few of them are a
// form of its own: 2 KiB of arguments cost the host a microsecond.)
constexpr uint32_t kRowsFew = 16, kRowsInline = 256;
struct DeviceBatchArgs {
    uint32_t *batch;
    uint32_t *tree;
    const int32_t *parents;    // null: no trees
    const int32_t *positions;
    const uint32_t *table;
    uint64_t stride;
    const int32_t *held;       // pages of every sequence
    int32_t *status;           // null: not asked for
    const uint32_t *rows_at;   // [sequences] rows, [sequences] first rows
    uint32_t sequences, rows;
    uint32_t page_shift;
    uint32_t page_count;
    uint32_t most_positions;
    uint32_t ids_at;
    uint64_t ids_room;
};
template <uint32_t N>
struct DeviceBatch : DeviceBatchArgs {
    uint32_t inline_rows[2 * N];
};

// Lengths, numbers of pages, the first 256 of its page ids and its parents are one trip to memory for a sequence's workgroup.
template <uint32_t N>
__global__ __launch_bounds__(kThreads) void paged_device_batch_kernel(DeviceBatch<N> a) {
    __shared__ uint64_t sums[kThreads / 64];
    __shared__ int32_t up[kTreeRows];
    __shared__ uint32_t words[kThreads / 64];
    const uint32_t i = blockIdx.x, tid = threadIdx.x;
    auto rows_of = [&](uint32_t s) { return a.rows_at ? a.rows_at[s] : a.inline_rows[s]; };
    const uint32_t rows = rows_of(i), row0 = a.rows_at ? a.rows_at[a.sequences + i] : a.inline_rows[N + i];
    const uint32_t first_id = tid < a.stride ? a.table[i * a.stride + tid] : 0;
    const int32_t first_parent = a.parents && tid < rows ? a.parents[row0 + tid] : -1;
    // What a sequence's positions are refused for, and the pages that they take otherwise.
    auto pages_of = [&](uint32_t s, uint32_t new_rows, uint32_t &pages) {
        const int32_t position = a.positions[s], held = a.held[s];
        pages = 0;
        if (!new_rows) return ITAK_TABLE_OK;
        if (position < 0 || uint32_t(position) > a.most_positions) return ITAK_TABLE_POSITION;
        const uint32_t need = (uint32_t(position) + new_rows + (1u << a.page_shift) - 1) >> a.page_shift;
        if (held < 0 || need > uint32_t(held) || uint32_t(held) > a.stride) return ITAK_TABLE_PAGES;
        pages = need;
        return ITAK_TABLE_OK;
    };
    uint32_t pages;
    int32_t status = pages_of(i, rows, pages);
    const uint32_t position = status == ITAK_TABLE_OK && rows ? uint32_t(a.positions[i]) : 0;
    uint64_t id0 = 0;
    for (uint32_t s = tid; s < i; s += kThreads) {
        uint32_t others;
        (void)pages_of(s, rows_of(s), others);
        id0 += others;
    }
    id0 = wave_sum(id0);
    if ((tid & 63) == 0) sums[tid / 64] = id0;
    uint32_t not_ = 0;
    constexpr uint32_t kNoPage = 4;
    if (status == ITAK_TABLE_OK) {
        for (uint32_t p = tid; p < pages; p += kThreads)
            if ((p == tid ? first_id : a.table[i * a.stride + p]) >= a.page_count) not_ |= kNoPage;
        if (a.parents)
            for (uint32_t r = tid; r < rows; r += kThreads) not_ |= parent_is_not(r == tid ? first_parent : a.parents[row0 + r], r);
    }
    up[tid] = first_parent;
    not_ = any_bits(not_, words);
    id0 = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) id0 += sums[w];
    if (status == ITAK_TABLE_OK) {
        if (id0 + pages > a.ids_room)
            status = ITAK_TABLE_ROOM;
        else if (not_ & kNoPage)
            status = ITAK_TABLE_ID;
        else if ((not_ & kNoTree) || ((not_ & kNoChain) && rows > kTreeRows))
            status = ITAK_TABLE_PARENTS;
    }
    const bool in = status == ITAK_TABLE_OK;
    if (in) {
        uint32_t *const ids = a.batch + a.ids_at + id0;
        for (uint32_t p = tid; p < pages; p += kThreads) ids[p] = p == tid ? first_id : a.table[i * a.stride + p];
        if (a.parents) make_records(a.tree + uint64_t(row0) * kTreeStride, rows, position, not_ & kNoChain, up);
    }
    if (tid == 0) {
        *reinterpret_cast<uint4 *>(a.batch + kPagedItem0 + 4 * i) =
            make_uint4(in ? position : 0, in ? rows : 0, row0, a.ids_at + uint32_t(in ? id0 : 0));
        if (a.status) a.status[i] = status;
        if (i == 0) *reinterpret_cast<uint4 *>(a.batch) = make_uint4(a.sequences, a.rows, a.parents ? 1 : 0, 0);
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
// (Workgroups that a graph captured may be fewer than the items of the batch that is there when it runs.)
__global__ __launch_bounds__(kThreads) void paged_batch_rows_kernel(BatchRows a) {
    const uint32_t n = a.batch[0];
    const bool trees = a.tree && a.batch[2];
    for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
        const uint4 item = *reinterpret_cast<const uint4 *>(a.batch + kPagedItem0 + 4 * i);
        const uint32_t end = min(a.rows, i + 1 < n ? a.batch[kPagedItem0 + 4 * (i + 1) + 2] : a.batch[1]);
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
}

// Page tables that grow and shrink to lengths. Pages given back come onto the free list's end in the order in which taking them from
// there finds them again; then sequences take theirs from the end, the first ones first.
struct FitTablesArgs {
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
};
template <uint32_t N>
struct FitTables : FitTablesArgs {
    uint32_t inline_rows[N];
};
// Inclusive sums over the workgroup; `sums` is a word a wavefront of LDS, which the caller lets go of behind a barrier.
template <uint32_t THREADS>
__device__ __forceinline__ uint64_t scan_all(uint64_t x, uint64_t *sums) {
    const uint32_t lane = __lane_id(), wave = threadIdx.x / 64;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up(x, d);
        x += lane >= uint32_t(d) ? y : 0;
    }
    if constexpr (THREADS > 64) {
        if (lane == 63) sums[wave] = x;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) x += sums[w];
    }
    return x;
}
// THREADS: as many as the sequences, or more: 64 are one wavefront, whose barriers cost nothing.
template <uint32_t THREADS, uint32_t N>
__global__ __launch_bounds__(THREADS) void paged_fit_kernel(FitTables<N> a) {
    __shared__ uint64_t sums[2][THREADS / 64];
    __shared__ uint64_t ends[THREADS];   // of every sequence's pages among those that move
    __shared__ uint32_t from[THREADS];   // its first of them
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
    const uint64_t back = need < held ? held - need : 0, back_end = scan_all<THREADS>(back, sums[0]);
    ends[i] = back_end, from[i] = need;
    __syncthreads();
    const uint64_t all_back = ends[THREADS - 1];
    const bool room = sound && count + all_back <= a.page_count;
    // The sequence that has number x of the pages that move, and which of its own that is.
    auto owner = [&](uint64_t x, uint64_t &own) {
        uint32_t s = 0;
#pragma unroll
        for (uint32_t step = THREADS / 2; step; step /= 2)
            if (ends[s + step - 1] <= x) s += step;
        own = x - (s ? ends[s - 1] : 0) + from[s];
        return s;
    };
    if (room)
        for (uint64_t x = i; x < all_back; x += THREADS) {
            uint64_t own;
            const uint32_t s = owner(x, own);
            a.free_ids[count + all_back - 1 - x] = a.table[s * a.stride + own];
        }
    __syncthreads();  // (what was given back is there to be taken)
    const uint64_t have_free = count + all_back;
    uint64_t take = room && need > held ? need - held : 0;
    const uint64_t take_end = scan_all<THREADS>(take, sums[1]);
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
    for (uint32_t w = 0; w < THREADS / 64; ++w) all_taken = sums[0][w] > all_taken ? sums[0][w] : all_taken;
    for (uint64_t x = i; x < all_taken; x += THREADS) {
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

template <uint32_t N>
void send_tree(uint32_t *batch, uint32_t *tree, const std::vector<uint32_t> &head, uint32_t ids_at, const uint32_t *ids, uint32_t id_count,
               const int32_t *parents, uint32_t rows, uint32_t items, hipStream_t stream) {
    TreeWords<N> a;
    a.batch = batch, a.tree = tree, a.n0 = uint32_t(head.size()), a.at1 = ids_at, a.n1 = id_count, a.pad = 0;
    std::copy(head.begin(), head.end(), a.w);
    std::copy(ids, ids + id_count, a.w + a.n0);
    std::copy(parents, parents + rows, reinterpret_cast<int32_t *>(a.w) + a.n0 + id_count);
    launch_kernel(paged_tree_words_kernel<N>, std::max(1u, items), kThreads, 0, stream, a);
}
bool send_tree_batch(uint32_t *batch, uint32_t *tree, const std::vector<uint32_t> &head, uint32_t ids_at, const uint32_t *ids, uint32_t id_count,
                     const int32_t *parents, uint32_t rows, uint32_t items, hipStream_t stream) {
    const uint64_t words = head.size() + id_count + rows;
    if (words > kManyWords) return false;
    (words <= kFewWords ? send_tree<kFewWords> : send_tree<kManyWords>)(batch, tree, head, ids_at, ids, id_count, parents, rows, items, stream);
    return true;
}

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

// Words of every sequence where they are more than travel with a launch, to the handle's memory, `at` words from its start.
void place_words(itak_paged *p, const uint32_t *words, uint32_t n, uint32_t at) {
    for (uint32_t i = 0; i < n; i += kManyWords)
        send_words(p->rows_dev, at + i, words + i, std::min(n - i, kManyWords), 0, nullptr, 0, p->stream);
}

template <uint32_t THREADS, uint32_t N>
void launch_fit(const FitTablesArgs &args, const uint32_t *rows, uint32_t n, hipStream_t stream) {
    FitTables<N> a;
    static_cast<FitTablesArgs &>(a) = args;
    if (rows) std::copy(rows, rows + n, a.inline_rows);
    launch_kernel(paged_fit_kernel<THREADS, N>, 1, THREADS, 0, stream, a);
}
template <uint32_t N>
void launch_device_batch(const DeviceBatchArgs &args, const uint32_t *rows, const uint32_t *first, uint32_t n, hipStream_t stream) {
    DeviceBatch<N> a;
    static_cast<DeviceBatchArgs &>(a) = args;
    if (rows) std::copy(rows, rows + n, a.inline_rows), std::copy(first, first + n, a.inline_rows + N);
    launch_kernel(paged_device_batch_kernel<N>, args.sequences, kThreads, 0, stream, a);
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
    try {
        if (const itak_status st = paged_reserve_trees(paged); st != ITAK_OK) return st;
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
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
    FitTablesArgs a{};
    const uint32_t n = tables->sequences;
    if (rows && n > kRowsInline) {
        place_words(paged, rows, n, 0);
        a.rows_at = paged->rows_dev;
    }
    a.table = tables->table, a.stride = tables->stride, a.held = tables->pages;
    a.free_ids = tables->free_ids, a.free_count = tables->free_count;
    a.lengths = lengths_dev, a.status = status_dev;
    a.sequences = tables->sequences;
    a.page_shift = paged->g.page_shift;
    a.page_count = uint32_t(paged->cfg.page_count);
    a.plus_rows = rows != nullptr;
    if (n <= 64 && (!rows || n <= kRowsFew))
        launch_fit<64, kRowsFew>(a, rows, n, paged->stream);
    else if (n <= 64)
        launch_fit<64, kRowsInline>(a, rows, n, paged->stream);
    else if (n <= kRowsInline)
        launch_fit<256, kRowsInline>(a, rows, n, paged->stream);
    else
        launch_fit<1024, kRowsFew>(a, nullptr, n, paged->stream);
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
    const bool captured = capturing(paged->stream);
    try {
        // What the host knows of the batch: every sequence at the most positions it may have.
        PagedBatch &next = paged->next;
        next.head.assign(kPagedItem0, 0);
        next.ids.clear();
        next.items = n, next.rows = uint32_t(all), next.most_rows = most;
        next.trees = parents_dev != nullptr, next.tree_most = tree_most, next.on_device = true, next.idle_kept = true;
        next.cuts[0] = next.cuts[1] = {};
        next.capture = captured ? capture_of(paged->stream) : 0;
        uint32_t row0 = 0;
        paged->first_rows.resize(n);
        for (uint32_t i = 0; i < n; row0 += rows[i], ++i) {
            const uint32_t words[4] = {uint32_t(most_positions), rows[i], row0, 0};
            next.head.insert(next.head.end(), words, words + 4);
            paged->first_rows[i] = row0;
        }
        next.head[0] = n, next.head[1] = next.rows, next.head[2] = next.trees;
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
    if (st = paged_replays_hold(paged, paged->next); st != ITAK_OK) return st;
    DeviceBatchArgs a{};
    if (n > kRowsInline) {
        place_words(paged, rows, n, 0);
        place_words(paged, paged->first_rows.data(), n, n);
        a.rows_at = paged->rows_dev;
    }
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
    if (captured) {
        paged->ids_never_known = true;
        auto &c = paged->captured_batch;
        c.position = std::max(c.position, uint32_t(most_positions)), c.rows = std::max(c.rows, most), c.tree_most = std::max(c.tree_most, tree_most);
    }
    const uint32_t *const first = paged->first_rows.data();
    if (n <= kRowsFew)
        launch_device_batch<kRowsFew>(a, rows, first, n, paged->stream);
    else if (n <= kRowsInline)
        launch_device_batch<kRowsInline>(a, rows, first, n, paged->stream);
    else
        launch_device_batch<kRowsFew>(a, nullptr, nullptr, n, paged->stream);
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
