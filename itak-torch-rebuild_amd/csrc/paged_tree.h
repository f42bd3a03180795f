// Trees of drafted tokens in a batch of a paged cache: what rows they may be, and what the device holds of each.
//
// A tree is an item's new rows, each with the number of an earlier row that it continues, or -1 of one that continues the held
// positions. Row r lies in the pages at position held + r. Its depth is the number of rows above it; it is turned by, and a window is
// counted from, held + depth. It sees the held positions, the rows above it and itself.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define ITAK_BOTH __host__ __device__ __forceinline__
#else
#define ITAK_BOTH inline
#endif

namespace itak {

// Rows of an item that is a tree; one of more has to be a chain, every row continuing the one before.
constexpr uint32_t kTreeRows = 256;
// A row's record: its depth (of a row of a chain, which sees every row before it: kTreeChain beside it), its parent, then
// what it sees of the 32-key blocks from the one of the item's `position` on, a bit a key. (31 + 256 keys lie in up to nine blocks.)
// Twelve words: a record starts on 16 bytes.
constexpr uint32_t kTreeDepth = 0, kTreeParent = 1, kTreeSees = 2, kTreeBlocks = 9, kTreeStride = 12;
constexpr uint32_t kTreeChain = 1u << 31;

ITAK_BOTH uint32_t tree_depth(uint32_t word) { return word & ~kTreeChain; }
// Where a row's record begins. A batch without records may have more rows than there is room for: where one is read all the same, and
// what it says not looked at, it is the first.
ITAK_BOTH uint64_t tree_record_at(bool trees, uint64_t row) { return trees ? row * kTreeStride : 0; }

// Whether the parents of a whole item are those of a chain, and of a tree: every one a row before, or -1.
inline bool tree_is_chain(const int32_t *parents, uint64_t rows) {
    for (uint64_t r = 0; r < rows; ++r)
        if (parents[r] != int32_t(int64_t(r) - 1)) return false;
    return true;
}
inline uint64_t tree_first_wrong(const int32_t *parents, uint64_t rows) {
    for (uint64_t r = 0; r < rows; ++r)
        if (parents[r] < -1 || parents[r] >= int64_t(r)) return r;
    return rows;
}

#if defined(__HIPCC__)
// What a row sees of block kb of keys, a bit a key, of the record's words; `first`: the block of the item's position. All of a block before
// it, and of every block where the row is a chain's (a window, and the row's own place, bound that further).
__device__ __forceinline__ uint32_t tree_sees(const uint32_t *record, uint32_t depth_word, uint32_t kb, uint32_t first) {
    if (kb < first || (depth_word & kTreeChain)) return ~0u;
    return record[kTreeSees + (kb - first < kTreeBlocks ? kb - first : kTreeBlocks - 1)];
}
#endif

}  // namespace itak
