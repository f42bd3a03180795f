// Dynamic LDS that a launch has only where its kernel has been granted it.
#pragma once

#include <atomic>
#include <cstdint>

namespace itak {

// Calls `grant` (0: granted) the first time a device's launch of `Kernel` asks, and again until it has succeeded. The kernel is a part
// of the function's name and not an argument of its type: kernels of one signature share a type, and would share the mark.
template <auto Kernel, typename Grant>
auto granted_once(int device, Grant grant) -> decltype(grant()) {
    static std::atomic<uint64_t> done{0};
    const uint64_t mark = device >= 0 && device < 64 ? uint64_t(1) << device : 0;  // (of others every time)
    if (done.load(std::memory_order_relaxed) & mark) return decltype(grant())(0);
    const auto status = grant();
    if (status == decltype(grant())(0)) done.fetch_or(mark, std::memory_order_relaxed);
    return status;
}

}  // namespace itak
