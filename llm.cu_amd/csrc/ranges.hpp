// Whether two pieces of memory have bytes in common (host checks of arguments).
#pragma once
#include <cstddef>
#include <cstdint>

static inline bool ranges_meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + b_bytes && y < x + a_bytes;
}
