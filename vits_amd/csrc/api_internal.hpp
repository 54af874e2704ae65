#pragma once
#include <stdint.h>
// Records a thread-local error message and returns `code` (shared by every entry point).
int vk_fail(int code, const char* msg);

// Strides of a view in elements: kernels add them up in unsigned and 64-bit numbers, so none may be negative, nor so large
// (2 TiB of bf16 and more) that a sum wraps.
inline bool vk_strides_ok(int64_t bstride, int64_t cstride)
{
    constexpr int64_t most = (int64_t)1 << 40;
    return bstride >= 0 && bstride <= most && cstride >= 0 && cstride <= most;
}

// Views that a pass writes: rows must not overlap.  The strides are fine as above.
inline bool vk_rows_apart(int64_t bstride, int64_t cstride, int64_t channels, int64_t length, int64_t batch)
{
    if (channels > 1 && cstride < length) return false;
    if (batch <= 1) return true;
    int64_t item;
    return !__builtin_mul_overflow(channels - 1, channels > 1 ? cstride : 0, &item) && bstride - length >= item;
}
