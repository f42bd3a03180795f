// After a forward over drafted tokens: the walk down a tree along the tokens that the model chose, and the accepted rows to the front.
//
// The walk goes from row 0 to the lowest-numbered child whose token is the one chosen at its parent: a wavefront has all of a tree's rows
// in its registers, and a step is a few ballots. The rows it went through are in ascending order, row number j of them at or behind place j, so
// a thread that moves them in order, a few at once, reads each before anything is written over it. Words and launches: what bounds both is the
// chain of trips to memory (item, path, page ids, rows): a tree of 16 rows 2.0 us for the walk and 2.7 for the rows of 4 layers, 16 trees of 64 rows 3.8 and,
// 24 layers, 5.9, where a launch that stores some words takes 1.1 to 1.5.
#include "mfma_common.h"
#include "paged_handle.h"

#include <algorithm>

using namespace itak;

namespace itak {

namespace {

// The rows of the batch that are item i's: those it was given, whether the batch takes it or not.
__device__ __forceinline__ uint32_t rows_end(const uint32_t *batch, uint32_t n, uint32_t i, uint32_t rows) {
    return min(rows, i + 1 < n ? batch[kPagedItem0 + 4 * (i + 1) + 2] : batch[1]);
}

struct Accept {
    const uint32_t *batch;
    const uint32_t *tree;
    uint64_t tree_rows;
    const int32_t *tokens, *chosen;
    int32_t *path, *next;
    uint32_t rows;
};
__global__ __launch_bounds__(64) void paged_accept_kernel(Accept a) {
    constexpr uint32_t kOfLane = kTreeRows / 64;
    const uint32_t i = blockIdx.x, lane = threadIdx.x;
    const uint4 item = *reinterpret_cast<const uint4 *>(a.batch + kPagedItem0 + 4 * i);
    const uint32_t n = min(a.batch[0], gridDim.x), row0 = item.z;
    if (i >= n) return;
    const uint32_t end = rows_end(a.batch, n, i, a.rows);
    const uint32_t rows = row0 < end ? min(item.y, end - row0) : 0;
    // All of a tree's rows at once. (Those behind it are clamped to the batch's last.)
    int32_t parent[kOfLane], token[kOfLane], chosen[kOfLane];
#pragma unroll
    for (uint32_t k = 0; k < kOfLane; ++k) {
        parent[k] = -2, token[k] = chosen[k] = 0;
        if (64 * k >= rows) continue;
        const uint32_t at = min(row0 + 64 * k + lane, a.rows - 1);
        parent[k] = int32_t(a.tree[min(uint64_t(at), a.tree_rows - 1) * kTreeStride + kTreeParent]);
        token[k] = a.tokens[at], chosen[k] = a.chosen[at];
    }
    const bool chain = !a.batch[2] || (rows && a.tree[uint64_t(row0) * kTreeStride] & kTreeChain);
    uint32_t kept = 0;
    int32_t choice = 0;
    if (rows && chain) {
        // Up to the first row whose successor is not what was chosen there.
        uint32_t last = rows - 1;
        for (uint32_t at = 0; at + 1 < rows; at += 64) {
            const uint32_t r = at + lane;
            const bool stops = r + 1 < rows && a.tokens[row0 + r + 1] != a.chosen[row0 + r];
            const uint64_t mask = __builtin_amdgcn_ballot_w64(stops);
            if (mask) {
                last = at + __builtin_ctzll(mask);
                break;
            }
        }
        kept = last + 1;
        for (uint32_t r = lane; r < kept; r += 64) a.path[row0 + r] = int32_t(r);
        choice = a.chosen[row0 + last];
    } else if (rows) {
#pragma unroll
        for (uint32_t k = 0; k < kOfLane; ++k)
            if (64 * k + lane >= rows) parent[k] = -2;
        uint32_t at = 0;
        while (true) {  // (a child lies behind its parent: at most as many steps as rows)
            if (lane == 0) a.path[row0 + kept] = int32_t(at);
            ++kept;
#pragma unroll
            for (uint32_t k = 0; k < kOfLane; ++k)
                if (at / 64 == k) choice = __builtin_amdgcn_readlane(chosen[k], at & 63);
            uint32_t child = ~0u;
#pragma unroll
            for (uint32_t k = 0; k < kOfLane; ++k) {
                const uint64_t mask = __builtin_amdgcn_ballot_w64(parent[k] == int32_t(at) && token[k] == choice);
                if (mask && child == ~0u) child = 64 * k + __builtin_ctzll(mask);
            }
            if (child == ~0u) break;
            at = child;
        }
    }
    for (uint32_t r = row0 + kept + lane; r < end; r += 64) a.path[r] = -1;
    if (rows && lane == 0) a.next[i] = choice;
}

struct Keep {
    PagedGeom g;
    const uint32_t *batch;
    uint16_t *storage;
    uint64_t layer_stride;
    uint64_t pieces;          // of eight channels, of a row of all layers
    const int32_t *path;
    int32_t *lengths;         // null: not asked for
    uint32_t rows;
};
constexpr uint32_t kKeepThreads = 256;
__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(Keep a) {
    constexpr uint32_t kAtOnce = 8;
    __shared__ uint64_t lds_from[kKeepThreads], lds_to[kKeepThreads];
    __shared__ int32_t lds_path[kKeepThreads];
    __shared__ uint32_t lds_ids[kKeepThreads / 16 + 1];  // pages of as many rows
    __shared__ uint32_t lds_moves, lds_kept, lds_wrong;
    const uint32_t i = blockIdx.x, tid = threadIdx.x;
    const uint4 item = *reinterpret_cast<const uint4 *>(a.batch + kPagedItem0 + 4 * i);
    const uint32_t n = min(a.batch[0], gridDim.x), row0 = item.z;
    if (i >= n) return;
    const uint32_t end = rows_end(a.batch, n, i, a.rows);
    const uint32_t rows = row0 < end ? min(item.y, end - row0) : 0;
    if (!rows) return;
    // The path and the pages of the rows it may name are one trip, for the first 256 of them.
    const uint32_t first_page = item.x >> a.g.page_shift, last_page = (item.x + rows - 1) >> a.g.page_shift;
    lds_path[tid] = a.path[min(row0 + tid, a.rows - 1)];
    if (tid < kKeepThreads / 16 + 1) lds_ids[tid] = a.batch[item.w + min(first_page + tid, last_page)];
    auto path_of = [&](uint32_t j) { return j < kKeepThreads ? lds_path[j] : a.path[row0 + j]; };
    // How many are kept, and whether they ascend: looked through before anything moves.
    if (tid == 0) lds_kept = rows, lds_wrong = 0;
    __syncthreads();
    for (uint32_t j = tid; j < rows; j += kKeepThreads)
        if (path_of(j) < 0) {
            atomicMin(&lds_kept, j);
            break;
        }
    __syncthreads();
    const uint32_t kept = lds_kept;
    for (uint32_t j = tid; j < kept; j += kKeepThreads)
        if (path_of(j) >= int32_t(rows) || (j && path_of(j - 1) >= path_of(j))) lds_wrong = 1;
    __syncthreads();
    const bool wrong = lds_wrong != 0;
    if (blockIdx.y == 0 && tid == 0 && a.lengths) a.lengths[i] = wrong ? -1 : int32_t(item.x + kept);
    if (wrong) return;
    const uint32_t mask = (1u << a.g.page_shift) - 1;
    auto place = [&](uint32_t position) {
        const uint32_t page = position >> a.g.page_shift;
        const uint32_t id = position < item.x + kKeepThreads ? lds_ids[page - first_page] : a.batch[item.w + page];
        return id * a.g.page_stride + uint64_t(position & mask) * a.g.head_dim;
    };
    const uint32_t of_head = a.g.head_dim / 8;
    for (uint32_t j0 = 0; j0 < kept; j0 += kKeepThreads) {
        __syncthreads();
        if (tid == 0) lds_moves = 0;
        __syncthreads();
        const uint32_t j = j0 + tid;
        const uint32_t here = j < kept ? uint32_t(path_of(j)) : j;
        // (Rows that stay where they are come first: an ascending list that has left its places never comes back to them.)
        const bool moves = here != j;
        if (moves) {
            lds_from[tid] = place(item.x + here), lds_to[tid] = place(item.x + j);
            atomicAdd(&lds_moves, 1);
        }
        __syncthreads();
        const uint32_t moved = lds_moves, first = min(kKeepThreads, kept - j0) - moved;
        if (!moved) continue;
        for (uint64_t p = uint64_t(blockIdx.y) * kKeepThreads + tid; p < a.pieces; p += uint64_t(gridDim.y) * kKeepThreads) {
            uint64_t at = p / of_head;
            const uint32_t piece = uint32_t(p - at * of_head);
            const uint32_t heads = a.g.kv_heads, head = uint32_t(at % heads);
            at /= heads;
            uint16_t *const base = a.storage + (at / 2) * a.layer_stride + (at % 2) * a.g.side_stride + head * a.g.head_stride + piece * 8;
            for (uint32_t m = 0; m < moved; m += kAtOnce) {
                u32x4 x[kAtOnce];
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; ++u)
                    x[u] = *reinterpret_cast<const u32x4 *>(base + lds_from[first + min(m + u, moved - 1)]);
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; ++u)
                    if (m + u < moved) *reinterpret_cast<u32x4 *>(base + lds_to[first + m + u]) = x[u];
            }
        }
    }
}

}  // namespace

}  // namespace itak

namespace {

itak_status check_kept(itak_paged *p) {
    if (!p->tree_dev) return unsupported(p->err, "a paged cache that takes no trees (itak_paged_enable_trees)");
    // (Without the sequences that have no rows an item's number is not its sequence's.)
    if (p->batch.rows && !p->batch.idle_kept) return invalid_argument(p->err, "the batch was set before the paged cache took trees");
    return ITAK_OK;
}

}  // namespace

extern "C" {

itak_status itak_paged_accept_device(itak_paged *paged, const int32_t *tokens_dev, const int32_t *chosen_dev, int32_t *path_dev,
                                     int32_t *next_dev) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_kept(paged);
    if (st != ITAK_OK || paged->batch.rows == 0) return st;
    if (!tokens_dev || !chosen_dev || !path_dev || !next_dev) return invalid_argument(paged->err, "tokens, chosen, path or next are null");
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    const Accept a{paged->batch_dev, paged->tree_dev, paged->tree_rows, tokens_dev, chosen_dev, path_dev, next_dev, paged->batch.rows};
    launch_kernel(paged_accept_kernel, paged->batch.items, 64, 0, paged->stream, a);
    HIP_TRY(paged, hipGetLastError(), "launch the walk down a tree");
    return ITAK_OK;
}

itak_status itak_paged_keep_device(itak_paged *paged, const int32_t *path_dev, int32_t *lengths_dev) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_kept(paged);
    if (st != ITAK_OK || paged->batch.rows == 0) return st;
    if (!path_dev) return invalid_argument(paged->err, "the path is null");
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    Keep a{};
    a.g = paged->g;
    a.batch = paged->batch_dev;
    a.storage = reinterpret_cast<uint16_t *>(paged->storage);
    a.layer_stride = paged->layer_stride;
    a.pieces = uint64_t(paged->cfg.layer_count) * 2 * paged->g.kv_heads * (paged->g.head_dim / 8);
    a.path = path_dev, a.lengths = lengths_dev;
    a.rows = paged->batch.rows;
    const dim3 grid(paged->batch.items, uint32_t(std::min<uint64_t>((a.pieces + kKeepThreads - 1) / kKeepThreads, 1024)));
    launch_kernel(paged_keep_kernel, grid, kKeepThreads, 0, paged->stream, a);
    HIP_TRY(paged, hipGetLastError(), "launch the moving of kept rows");
    return ITAK_OK;
}

}  // extern "C"
