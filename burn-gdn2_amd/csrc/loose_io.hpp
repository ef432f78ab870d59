// Runs of N consecutive values at any element's address, whole or cut off.
#pragma once

#include "vec_io.hpp"

namespace gdn2 {

// (One wide load or store: global memory needs no alignment here beyond the
// element's, and an aligned address costs the same as by an aligned type.)
template <typename T, int N> __device__ __forceinline__ Raw<T, N> loose(const T *p) {
    Raw<T, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
// stream: by a hint that the caches need not keep it (the same for every lane), which is
// worth 2 to 4 % where a result is as large as they are, and costs as much where not.
constexpr double kStreamBytes = 1 << 27;
template <typename T, int N> __device__ __forceinline__ void loose_store(T *p, const float *x, bool stream = false) {
    typedef T Loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    Loose v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    if (stream) __builtin_nontemporal_store(v, reinterpret_cast<Loose *>(p));
    else *reinterpret_cast<Loose *>(p) = v;
}

// The first `left` of N values, zeros behind them (left <= 0: none is read).  WHOLE: left
// is N or more, or none (a tenth of the code, and of the branches).
template <typename T, int N, bool WHOLE = false> __device__ __forceinline__ Raw<T, N> loose_part(const T *p, int64_t left) {
    if (WHOLE) {
        Raw<T, N> v = {};
        if (left > 0) v = loose<T, N>(p);
        return v;
    }
    if (left >= N) return loose<T, N>(p);
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : (T)0.f;
    return v;
}
template <typename T, int N, bool WHOLE = false> __device__ __forceinline__ void load_part(const T *p, int64_t left, float *x) {
    const Raw<T, N> v = loose_part<T, N, WHOLE>(p, left);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)v[j];
}
template <typename T, int N, bool WHOLE = false> __device__ __forceinline__ void store_part(T *p, int64_t left, const float *x, bool stream = false) {
    if (WHOLE) {
        if (left > 0) loose_store<T, N>(p, x, stream);
    } else if (left >= N) {
        loose_store<T, N>(p, x, stream);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < left) p[j] = (T)x[j];
    }
}

// Values c .. c + N - 1 of a row of C, zeros behind its last: without a branch, as the
// row's last N, turned by as many as they start before c (only rows of less than N go
// value by value).
template <typename T, int N, bool WHOLE> __device__ __forceinline__ Raw<T, N> row_raw(const T *row, int c, int C) {
    if (WHOLE || C < N) return loose_part<T, N, WHOLE>(row + c, C - c);
    constexpr int WORDS = N * sizeof(T) / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(WORDS)));
    const int from = min(c, C - N), bytes = min(c - from, N) * (int)sizeof(T);
    const Raw<T, N> raw = loose<T, N>(row + from);
    Words w = __builtin_bit_cast(Words, raw);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = __builtin_amdgcn_alignbit(i + 1 < WORDS ? w[i + 1] : 0u, w[i], (bytes & 2) * 8);
    }
#pragma unroll
    for (int by = 1; by <= WORDS; by *= 2)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = bytes & (4 * by) ? (i + by < WORDS ? w[i + by] : 0u) : w[i];
    return __builtin_bit_cast(Raw<T, N>, w);
}
template <typename T, int N, bool WHOLE> __device__ __forceinline__ void row_part(const T *row, int c, int C, float *x) {
    const Raw<T, N> v = row_raw<T, N, WHOLE>(row, c, C);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)v[j];
}

}  // namespace gdn2
