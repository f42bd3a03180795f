// A batch of a paged cache, on the host: what is checked of it, and the words it becomes on the device.
#pragma once

#include "../../include/itak_hip_kv.h"

#include <cstdio>
#include <string>
#include <vector>

namespace itak {

// The batch in device memory: four words (active items, their rows, whether rows have records as paged_tree.h says, 0), four words
// an active item (position, rows, first row among the batch's, the word at which its page ids begin), from ids_at on the page
// ids. Items without rows are left out, their page ids are not; of a handle that takes trees an item's number is its sequence's, and none is left out.
constexpr uint32_t kPagedItem0 = 4;  // the first item's first word
inline uint32_t paged_ids_at(uint32_t max_sequences) { return kPagedItem0 + 4 * max_sequences; }

// Launches have a workgroup of 256 threads a row, and a launch's threads are counted in 32 bits.
constexpr uint64_t kPagedMostRows = (1u << 24) - 1;

struct PagedLimits {
    uint64_t page_count;
    uint32_t page_rows;
    uint32_t max_sequences;
    uint64_t max_table_pages;
};

struct PagedRefusal {
    int32_t code = ITAK_OK;
    const char *what = "";
    uint64_t a = 0, b = 0;
    std::string text;
};

struct PagedBatch {
    std::vector<uint32_t> head;  // the header and the items
    std::vector<uint32_t> ids;
    uint32_t items = 0;          // active ones
    uint32_t rows = 0;           // of all of them
    uint32_t most_rows = 0;      // of one
    bool trees = false;          // its rows have records
    uint32_t tree_most = 0;      // rows of its largest tree
    // How attention's launch for trees is cut over it, without a window and with one; `key`: what that was found for.
    struct Cut {
        uint64_t key = 0;
        bool chunk = false;      // by the kernel of many rows
        uint32_t tile = 0, share = 0;
    } cuts[2];
    bool idle_kept = false;      // an item's number is its sequence's
    uint64_t capture = 0;        // the capture that it was set in
    bool on_device = false;      // lengths and tables are the device's: positions in `head` are the most they may be, and there are no ids
};

// Fills `batch`, or says why not. `marks` (page_count words, any content that `stamp` is greater than) belongs to the caller and
// is written; stamp grows by the call.
inline PagedRefusal make_paged_batch(const PagedLimits &lim, const itak_paged_item *items, uint32_t count, const uint32_t *pages,
                                     uint64_t page_ids, std::vector<uint32_t> &marks, uint32_t &stamp, PagedBatch &batch, bool keep_idle = false) {
    auto refuse = [](int32_t code, const char *what, uint64_t a, uint64_t b, std::string text) {
        PagedRefusal r;
        r.code = code, r.what = what, r.a = a, r.b = b, r.text = std::move(text);
        return r;
    };
    auto number = [](uint64_t x) { return std::to_string(x); };
    if (count > lim.max_sequences)
        return refuse(ITAK_CAPACITY_EXCEEDED, "sequences", count, lim.max_sequences,
                      "a batch of " + number(count) + " sequences, the paged cache takes " + number(lim.max_sequences));
    if (page_ids > lim.max_table_pages)
        return refuse(ITAK_CAPACITY_EXCEEDED, "page ids", page_ids, lim.max_table_pages,
                      "a batch of " + number(page_ids) + " page ids, the paged cache takes " + number(lim.max_table_pages));
    if ((count && !items) || (page_ids && !pages))
        return refuse(ITAK_INVALID_ARGUMENT, "items or pages are null", 0, 0, "invalid argument: items or pages are null");
    uint64_t named = 0, rows = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const itak_paged_item &it = items[i];
        if (it.position >= (1ull << 31) || it.position + it.rows >= (1ull << 31))
            return refuse(ITAK_SIZE_OVERFLOW, "positions", it.position, it.rows,
                          "item " + number(i) + ": positions reach 2^31");
        const uint64_t need = (it.position + it.rows + lim.page_rows - 1) / lim.page_rows;
        if (it.rows && it.pages < need)
            return refuse(ITAK_SHAPE_MISMATCH, "pages", need, it.pages,
                          "item " + number(i) + ": " + number(it.position + it.rows) + " positions need " + number(need) +
                              " pages, got " + number(it.pages));
        named += it.pages;
        rows += it.rows;
    }
    if (named != page_ids)
        return refuse(ITAK_SHAPE_MISMATCH, "page_ids", named, page_ids,
                      "page_ids: got " + number(page_ids) + ", the items name " + number(named));
    if (rows > kPagedMostRows) return refuse(ITAK_SIZE_OVERFLOW, "rows", rows, 0, "more than 2^24 - 1 rows in a batch");
    for (uint64_t i = 0; i < page_ids; ++i)
        if (pages[i] >= lim.page_count)
            return refuse(ITAK_INVALID_ARGUMENT, "page id", pages[i], lim.page_count,
                          "page " + number(pages[i]) + " out of range, the paged cache has " + number(lim.page_count));
    // Pages that take new rows are marked with this call's stamp; a second place that names one is refused.
    if (stamp == ~0u) marks.assign(marks.size(), 0), stamp = 0;
    ++stamp;
    auto shared = [&](uint32_t page) {
        return refuse(ITAK_INVALID_ARGUMENT, "page takes new rows and is named twice", page, 0,
                      "page " + number(page) + " takes new rows and is named in two places of the batch's tables");
    };
    uint64_t at = 0;
    for (uint32_t i = 0; i < count; at += items[i].pages, ++i) {
        if (!items[i].rows) continue;
        const uint64_t last = (items[i].position + items[i].rows - 1) / lim.page_rows;
        for (uint64_t p = items[i].position / lim.page_rows; p <= last; ++p) {
            uint32_t &mark = marks[pages[at + p]];
            if (mark == stamp) return shared(pages[at + p]);
            mark = stamp;
        }
    }
    at = 0;
    for (uint32_t i = 0; i < count; at += items[i].pages, ++i) {
        const uint64_t first = items[i].rows ? items[i].position / lim.page_rows : items[i].pages;
        const uint64_t last = items[i].rows ? (items[i].position + items[i].rows - 1) / lim.page_rows : 0;
        for (uint64_t p = 0; p < items[i].pages; ++p)
            if ((p < first || p > last) && marks[pages[at + p]] == stamp) return shared(pages[at + p]);
    }
    batch.items = batch.rows = batch.most_rows = 0;
    batch.head.assign(kPagedItem0, 0);
    batch.idle_kept = keep_idle;
    batch.ids.assign(pages, pages + page_ids);
    uint32_t id = paged_ids_at(lim.max_sequences);
    for (uint32_t i = 0; i < count; id += items[i].pages, ++i) {
        if (!items[i].rows && !keep_idle) continue;
        const uint32_t words[4] = {uint32_t(items[i].position), items[i].rows, batch.rows, id};
        batch.head.insert(batch.head.end(), words, words + 4);
        ++batch.items;
        batch.rows += items[i].rows;
        if (items[i].rows > batch.most_rows) batch.most_rows = items[i].rows;
    }
    batch.head[0] = batch.items;
    batch.head[1] = batch.rows;
    return PagedRefusal{};
}

}  // namespace itak
