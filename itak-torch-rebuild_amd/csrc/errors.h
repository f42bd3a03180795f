// The library's error state and its diagnostic channel, shared by the files that hold entry points.
#pragma once

#include "../../include/itak_hip_kv.h"

#include <hip/hip_runtime.h>

#include <string>

namespace itak {

struct ErrorState {
    std::string message;
    itak_error_info info{};
};

// Of the last failed call on this thread that has no handle to keep it (itak_last_error(NULL)).
ErrorState &thread_error();

void set_diag_enabled(bool on);
bool diag_enabled();
__attribute__((format(printf, 1, 2))) void diag_emit(const char *fmt, ...);

#define ITAK_DIAG(...)                          \
    do {                                        \
        if (diag_enabled()) diag_emit(__VA_ARGS__); \
    } while (0)

#define ULL(x) static_cast<unsigned long long>(x)

__attribute__((format(printf, 8, 9))) itak_status set_error(ErrorState &e, int32_t code, const char *what, uint64_t a,
                                                            uint64_t b, uint64_t c, uint64_t d, const char *fmt, ...);
itak_status zero_dimension(ErrorState &e, const char *what);
itak_status invalid_window(ErrorState &e, uint64_t window);
itak_status size_overflow(ErrorState &e, const char *what);
itak_status shape_mismatch(ErrorState &e, const char *what, uint64_t expected, uint64_t actual);
itak_status invalid_layer(ErrorState &e, uint64_t layer, uint64_t layer_count);
itak_status out_of_order(ErrorState &e, uint64_t layer, uint64_t expected, uint64_t actual);
itak_status non_divisible(ErrorState &e, uint64_t q_heads, uint64_t kv_heads);
itak_status no_visible_keys(ErrorState &e, uint64_t position);
itak_status checkpoint_busy(ErrorState &e);
itak_status stale_checkpoint(ErrorState &e, uint64_t serial);
itak_status range_exceeded(ErrorState &e, uint64_t layer, uint64_t position, uint64_t limit);
itak_status not_fresh(ErrorState &e, uint64_t layer, uint64_t appended);
itak_status rewind_range(ErrorState &e, uint64_t layer, uint64_t base, uint64_t appended, uint64_t target);
itak_status hip_error(ErrorState &e, hipError_t code, const char *doing);
itak_status invalid_argument(ErrorState &e, const char *what);
itak_status capacity_exceeded(ErrorState &e, uint64_t layer, uint64_t need, uint64_t capacity);
itak_status unsupported(ErrorState &e, const char *what);

}  // namespace itak
