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

// ... for results that are larger than the caches and not read again here: a hint
// that leaves the caches to what is (up to a tenth of a kernel's time)
template <typename T, int N> __device__ __forceinline__ void stream_n(T *p, const float *x) {
    Raw<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    __builtin_nontemporal_store(v, reinterpret_cast<Raw<T, N> *>(p));
}

// Sums of n values over the 2^log_l neighbouring lanes of each group of lanes, to
// all of them (log_l the same in the wave).  Up to 16 lanes by the adder's own lane
// moves: the other lane of a pair, the other pair, and, the sums being the same in
// a quad by then, the mirrored half and the mirrored row.
template <int N> __device__ __forceinline__ void lanes_sum(float (&v)[N], int log_l) {
#define GDN2_STEP(least, other)                              \
    if (log_l >= least) {                                    \
        _Pragma("unroll") for (int i = 0; i < N; ++i) {      \
            const int x = __builtin_bit_cast(int, v[i]);     \
            v[i] += __builtin_bit_cast(float, (other));      \
        }                                                    \
    }
    GDN2_STEP(1, __builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, true))  // quad_perm [1, 0, 3, 2]
    GDN2_STEP(2, __builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, true))  // quad_perm [2, 3, 0, 1]
    GDN2_STEP(3, __builtin_amdgcn_mov_dpp(x, 0x141, 0xF, 0xF, true)) // row_half_mirror
    GDN2_STEP(4, __builtin_amdgcn_mov_dpp(x, 0x140, 0xF, 0xF, true)) // row_mirror
    GDN2_STEP(5, __builtin_amdgcn_ds_swizzle(x, 0x401F))             // lane ^ 16
    GDN2_STEP(6, __shfl_xor(x, 32, kWave))
#undef GDN2_STEP
}
__device__ __forceinline__ float lanes_sum(float x, int log_l) {
    float v[1] = {x};
    lanes_sum<1>(v, log_l);
    return v[0];
}

}  // namespace gdn2
