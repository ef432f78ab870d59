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
template <typename T, int N> __device__ __forceinline__ void loose_store(T *p, const float *x) {
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    __builtin_memcpy(p, &v, sizeof(v));
}

// The first `left` of N values, zeros behind them (left <= 0: none is read).
template <typename T, int N> __device__ __forceinline__ Raw<T, N> loose_part(const T *p, int64_t left) {
    if (left >= N) return loose<T, N>(p);
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : (T)0.f;
    return v;
}
template <typename T, int N> __device__ __forceinline__ void load_part(const T *p, int64_t left, float *x) {
    const Raw<T, N> v = loose_part<T, N>(p, left);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)v[j];
}
template <typename T, int N> __device__ __forceinline__ void store_part(T *p, int64_t left, const float *x) {
    if (left >= N) {
        loose_store<T, N>(p, x);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < left) p[j] = (T)x[j];
    }
}

}  // namespace gdn2
