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

}  // namespace gdn2
