#pragma once
// 16 bytes of a time-contiguous row, near the end of the row too.
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef unsigned chunk_t __attribute__((ext_vector_type(4)));

// The elements of c moved `s` places towards the front, zeros behind them.
template <int E>
__device__ __forceinline__ chunk_t chunk_shift(chunk_t c, int s)
{
    if constexpr (E == 8) {
        c = (s & 4) ? chunk_t{c[2], c[3], 0u, 0u} : c;
        c = (s & 2) ? chunk_t{c[1], c[2], c[3], 0u} : c;
        c = (s & 1) ? chunk_t{__builtin_amdgcn_alignbit(c[1], c[0], 16), __builtin_amdgcn_alignbit(c[2], c[1], 16),
                              __builtin_amdgcn_alignbit(c[3], c[2], 16), c[3] >> 16} : c;
    } else {
        c = (s & 2) ? chunk_t{c[2], c[3], 0u, 0u} : c;
        c = (s & 1) ? chunk_t{c[1], c[2], c[3], 0u} : c;
    }
    return s >= E ? chunk_t{0u, 0u, 0u, 0u} : c;
}

// Elements t .. t + 15 / sizeof(T) of `row`; those at or behind `limit` are zero and nothing behind it is read.  A chunk
// that reaches over the limit is read where it ends there and moved, without a branch, so that the loads of a tile at
// the end of a row are in flight together like any others.  Rows of odd length start anywhere: the load is declared
// unaligned (the memory system takes it as one access).
template <typename T>
__device__ __forceinline__ chunk_t load_chunk(const T* row, int t, int limit)
{
    constexpr int E = 16 / (int)sizeof(T);
    chunk_t r = {0u, 0u, 0u, 0u};
    if (limit >= E) {                                       // the same for the whole workgroup
        const int at = t + E <= limit ? t : limit - E;
        __builtin_memcpy(&r, row + at, 16);
        return chunk_shift<E>(r, t - at < E ? t - at : E);
    }
    // rows shorter than a chunk: a loop, so that this rare case costs few instructions
    unsigned long long v[2] = {0, 0};
#pragma unroll 1
    for (int e = 0; e < limit - t; ++e) {
        const T x = row[t + e];
        unsigned bits = 0;
        __builtin_memcpy(&bits, &x, sizeof(T));
        const int pos = e * 8 * (int)sizeof(T);
        v[0] |= pos < 64 ? (unsigned long long)bits << pos : 0;
        v[1] |= pos >= 64 ? (unsigned long long)bits << (pos - 64) : 0;
    }
    return chunk_t{(unsigned)v[0], (unsigned)(v[0] >> 32), (unsigned)v[1], (unsigned)(v[1] >> 32)};
}
