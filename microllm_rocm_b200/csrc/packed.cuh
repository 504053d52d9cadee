// A launcher called with its arguments in one block of memory, each at its natural alignment, in the order of its parameters.  A call
// through ctypes spends 0.1 us on every argument (24 of them: 2.8 us, a block of them 0.6); kernels/ops.py packs the block.
#pragma once

#include <tuple>

#include "common.cuh"

namespace mlb {

template <typename T> inline T take_argument(const char*& at) {
    at = (const char*)(((uintptr_t)at + alignof(T) - 1) / alignof(T) * alignof(T));
    const T v = *reinterpret_cast<const T*>(at);
    at += sizeof(T);
    return v;
}

template <typename... Args> inline int call_packed(int (*launcher)(Args...), const void* block) {
    const char* at = (const char*)block;
    const std::tuple<Args...> arguments{take_argument<Args>(at)...};       // (braces: from the left)
    return std::apply(launcher, arguments);
}

}  // namespace mlb

#define MLB_PACKED(launcher) \
    MLB_EXPORT int launcher##_packed(const void* block) { return mlb::call_packed(launcher, block); }
