// Runs of N consecutive values, f32 or bf16 in memory and f32 in registers.
#pragma once

#include "common.hpp"

namespace gdn2 {

typedef __bf16 bf16;

template <typename T, int N> struct Vec {
    typedef T type __attribute__((ext_vector_type(N)));
};
// as they lie in memory; nothing waits for the load
template <typename T, int N> using Raw = typename Vec<T, N>::type;
template <typename T, int N> __device__ __forceinline__ Raw<T, N> raw_n(const T *p) {
    return *reinterpret_cast<const Raw<T, N> *>(p);
}
template <typename T, int N> __device__ __forceinline__ void load_n(const T *p, float *x) {
    const Raw<T, N> v = raw_n<T, N>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)v[j];
}
// each value rounded once, to nearest even
template <typename T, int N> __device__ __forceinline__ void store_n(T *p, const float *x) {
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    *reinterpret_cast<Raw<T, N> *>(p) = v;
}

}  // namespace gdn2
