// The handle of a paged cache, for the files that hold its entry points.
#pragma once

#include "paged.h"

#include "errors.h"

struct itak_paged {
    itak_paged_config cfg{};
    itak::PagedGeom g{};
    itak::PagedLimits limits{};
    uint64_t layer_stride = 0;  // elements
    uint64_t bytes = 0;
    unsigned char *storage = nullptr;
    bool owns = false;
    hipStream_t stream = nullptr;
    uint32_t *batch_dev = nullptr;
    uint64_t zeros_at = 0;           // words of the batch's memory up to sixteen bytes of zeros
    itak::PagedBatch batch;                // as it is set
    itak::PagedBatch next;                 // as it is being made
    std::vector<uint32_t> ids_there; // page ids as the device has them, all of its table
    std::vector<uint32_t> marks;
    uint32_t stamp = 0;
    // Buffers grow by being replaced, and what was replaced stays until the handle is gone: a captured graph may still name it.
    std::vector<void *> buffers;
    float *ws = nullptr;             // split partials
    uint64_t ws_bytes = 0;
    void *turned = nullptr;          // a step's rotated queries
    uint64_t turned_bytes = 0;
    // The most units that an attention call under capture has launched, of calls without a window and with one, whose largest and
    // smallest it is.
    struct Captured {
        uint64_t units;
        uint32_t window, least_window;
    } captured[2] = {};
    // What batches that graphs set may hold at most: positions, new rows of an item, rows of a tree.
    struct {
        uint32_t position, rows, tree_most;
    } captured_batch = {};
    // Of a handle that takes trees: a record for each of up to tree_rows rows (paged_tree.h), then those rows' parents on their way there.
    uint32_t *tree_dev = nullptr;
    uint64_t tree_rows = 0;
    uint32_t *rows_dev = nullptr;    // every sequence's rows, and its first, on their way to a batch that the device makes
    std::vector<uint32_t> first_rows;
    bool ids_known = true;           // what the device has of page ids is what ids_there says
    bool ids_never_known = false;    // a captured graph may set the batch
    mutable itak::ErrorState err;
};


namespace itak {

#define HIP_TRY(paged, call, doing)                                       \
    do {                                                                  \
        const hipError_t _e = (call);                                     \
        if (_e != hipSuccess) return hip_error((paged)->err, _e, doing);  \
    } while (0)

inline bool capturing(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(stream, &status) != hipSuccess || status != hipStreamCaptureStatusNone;
}

// Which capture a stream is in: 0 of none.
inline unsigned long long capture_of(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    return hipStreamGetCaptureInfo(stream, &status, &id) == hipSuccess && status == hipStreamCaptureStatusActive ? id : 0;
}

// paged.hip: words to dst + at0 and the n1 behind them to dst + at1, and what a batch of these words is refused for where attention was captured.
constexpr uint32_t kFewWords = 112, kManyWords = 960;
void send_words(uint32_t *dst, uint32_t at0, const uint32_t *w0, uint32_t n0, uint32_t at1, const uint32_t *w1, uint32_t n1,
                hipStream_t stream);
itak_status paged_replays_hold(const itak_paged *p, const PagedBatch &batch);
// The memory that attention over trees may need, captured or not.
itak_status paged_reserve_trees(itak_paged *p);
// paged_batch.hip: a batch of trees, of few enough words for one launch, and the records of one whose items and parents the device has.
bool send_tree_batch(uint32_t *batch, uint32_t *tree, const std::vector<uint32_t> &head, uint32_t ids_at, const uint32_t *ids, uint32_t id_count,
                     const int32_t *parents, uint32_t rows, uint32_t items, hipStream_t stream);
hipError_t launch_paged_records(const uint32_t *batch, uint32_t items, const int32_t *parents, uint32_t *tree, hipStream_t stream);

}  // namespace itak
