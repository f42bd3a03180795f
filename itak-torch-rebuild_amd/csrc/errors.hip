// The error state's texts and the diagnostic channel (errors.h).
#include "errors.h"

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

namespace itak {

ErrorState &thread_error() {
    static thread_local ErrorState state;
    return state;
}

// ------------------------------------------------------------------------------ debug channel
// attention::diag (crates/attention/src/diag.rs:13-33,71-79): off by default; the switch or
// ITAK_HIP_KV_DEBUG in the environment (any value but "0" or empty, looked up at every event as
// the reference looks its variable up) turns one stderr line per event on.
static std::atomic<bool> g_debug_enabled{false};

void set_diag_enabled(bool on) { g_debug_enabled.store(on, std::memory_order_relaxed); }

bool diag_enabled() {
    if (g_debug_enabled.load(std::memory_order_relaxed)) return true;
    const char *v = getenv("ITAK_HIP_KV_DEBUG");
    return v && v[0] != '\0' && !(v[0] == '0' && v[1] == '\0');
}

void diag_emit(const char *fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    fprintf(stderr, "[itak_hip_kv::diag] %s\n", buf);
}

// ------------------------------------------------------------------------------ errors

itak_status set_error(ErrorState &e, int32_t code, const char *what, uint64_t a, uint64_t b,
                      uint64_t c, uint64_t d, const char *fmt, ...) {
    e.info = itak_error_info{};
    e.info.code = code;
    if (what) snprintf(e.info.what, sizeof(e.info.what), "%s", what);
    e.info.a = a;
    e.info.b = b;
    e.info.c = c;
    e.info.d = d;
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    e.message = buf;
    ITAK_DIAG("refused code=%d: %s", int(code), buf);  // every refusal says why
    return code;
}

// The Display texts of AttentionError (crates/attention/src/error.rs:129-214).
itak_status zero_dimension(ErrorState &e, const char *what) {
    return set_error(e, ITAK_ZERO_DIMENSION, what, 0, 0, 0, 0, "%s must be positive, got 0", what);
}
itak_status invalid_window(ErrorState &e, uint64_t window) {
    return set_error(e, ITAK_INVALID_WINDOW, nullptr, window, 0, 0, 0,
                     "sliding window must be positive, got %llu", ULL(window));
}
itak_status size_overflow(ErrorState &e, const char *what) {
    return set_error(e, ITAK_SIZE_OVERFLOW, what, 0, 0, 0, 0, "%s: element count overflows usize",
                     what);
}
itak_status shape_mismatch(ErrorState &e, const char *what, uint64_t expected, uint64_t actual) {
    return set_error(e, ITAK_SHAPE_MISMATCH, what, expected, actual, 0, 0,
                     "%s: got %llu, expected %llu", what, ULL(actual), ULL(expected));
}
itak_status invalid_layer(ErrorState &e, uint64_t layer, uint64_t layer_count) {
    return set_error(e, ITAK_INVALID_LAYER, nullptr, layer, layer_count, 0, 0,
                     "layer %llu out of range, cache has %llu layers", ULL(layer),
                     ULL(layer_count));
}
itak_status out_of_order(ErrorState &e, uint64_t layer, uint64_t expected, uint64_t actual) {
    return set_error(e, ITAK_OUT_OF_ORDER_POSITION, nullptr, layer, expected, actual, 0,
                     "layer %llu appends must be in order: expected position %llu, got %llu",
                     ULL(layer), ULL(expected), ULL(actual));
}
itak_status non_divisible(ErrorState &e, uint64_t q_heads, uint64_t kv_heads) {
    return set_error(e, ITAK_NON_DIVISIBLE_HEADS, nullptr, q_heads, kv_heads, 0, 0,
                     "%llu query heads do not divide evenly across %llu KV heads", ULL(q_heads),
                     ULL(kv_heads));
}
itak_status no_visible_keys(ErrorState &e, uint64_t position) {
    return set_error(e, ITAK_NO_VISIBLE_KEYS, nullptr, position, 0, 0, 0,
                     "query at position %llu has no visible keys", ULL(position));
}
itak_status checkpoint_busy(ErrorState &e) {
    return set_error(e, ITAK_CHECKPOINT_BUSY, nullptr, 0, 0, 0, 0,
                     "a checkpoint is already outstanding on this cache; release it before "
                     "taking another");
}
itak_status stale_checkpoint(ErrorState &e, uint64_t serial) {
    return set_error(e, ITAK_STALE_CHECKPOINT, nullptr, serial, 0, 0, 0,
                     "checkpoint %llu is not this cache's live checkpoint (already released or "
                     "foreign)",
                     ULL(serial));
}
itak_status range_exceeded(ErrorState &e, uint64_t layer, uint64_t position, uint64_t limit) {
    return set_error(e, ITAK_CHECKPOINT_RANGE_EXCEEDED, nullptr, layer, position, limit, 0,
                     "layer %llu append at position %llu is outside the live checkpoint's saved "
                     "range (first unsaved position %llu); refusing so a later rewind cannot meet "
                     "a slot it cannot restore",
                     ULL(layer), ULL(position), ULL(limit));
}
itak_status not_fresh(ErrorState &e, uint64_t layer, uint64_t appended) {
    return set_error(e, ITAK_BULK_RESTORE_NOT_FRESH, nullptr, layer, appended, 0, 0,
                     "layer %llu already holds %llu appended positions; bulk restore installs "
                     "into a fresh layer only",
                     ULL(layer), ULL(appended));
}
itak_status rewind_range(ErrorState &e, uint64_t layer, uint64_t base, uint64_t appended,
                         uint64_t target) {
    return set_error(e, ITAK_REWIND_OUT_OF_RANGE, nullptr, layer, base, appended, target,
                     "rewind target %llu is outside layer %llu's checkpoint range [%llu, %llu]",
                     ULL(target), ULL(layer), ULL(base), ULL(appended));
}
itak_status hip_error(ErrorState &e, hipError_t code, const char *doing) {
    (void)hipGetLastError();  // (told here: not to be found by the next call, or by the program's own)
    return set_error(e, ITAK_HIP_ERROR, doing, uint64_t(code), 0, 0, 0, "%s: HIP error %d (%s)",
                     doing, int(code), hipGetErrorString(code));
}
itak_status invalid_argument(ErrorState &e, const char *what) {
    return set_error(e, ITAK_INVALID_ARGUMENT, what, 0, 0, 0, 0, "invalid argument: %s", what);
}
itak_status capacity_exceeded(ErrorState &e, uint64_t layer, uint64_t need, uint64_t capacity) {
    return set_error(e, ITAK_CAPACITY_EXCEEDED, nullptr, layer, need, capacity, 0,
                     "layer %llu would hold %llu positions but the pool's slots hold %llu",
                     ULL(layer), ULL(need), ULL(capacity));
}
itak_status unsupported(ErrorState &e, const char *what) {
    return set_error(e, ITAK_UNSUPPORTED, what, 0, 0, 0, 0, "unsupported: %s", what);
}

}  // namespace itak
