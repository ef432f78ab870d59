// The random words of dropout: Philox-4x32 with 7 rounds (J. K. Salmon, M. A. Moraes,
// R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), the
// counter a 64-bit number, the key the seed.  A round is two products of 32 x 32 bits
// into 64, which issue at a quarter of the rate of a sum: 7 rounds for 4 elements take
// about as long as the memory does for their 4 bytes of bfloat16 in and out (32768 x
// 2048: 45 us, 43 the bytes at a copy's rate), and so overlap with it; 10, the paper's
// safety margin, would bound the pass.
#pragma once

#include <cmath>

#include "common.hpp"
#include "gdn2_block.h"

namespace gdn2 {

// A call's dropout as kernels take it.
struct Drop {
    uint64_t seed, offset;
    const uint64_t *rng;
    uint32_t least; // words >> 8 from here on are kept
    float scale;    // of what is kept
};

inline bool drop_ok(const gdn2_dropout &d) { return d.p >= 0. && d.p <= 1.; } // (NaN: no)
// p = 1 (or so near it that every word is below): scale never used.
inline Drop drop_of(const gdn2_dropout &d) {
    Drop r{};
    r.seed = d.seed;
    r.offset = d.offset;
    r.rng = d.rng;
    r.least = (uint32_t)std::floor(d.p * 16777216. + 0.5);
    r.scale = d.p < 1. ? (float)(1. / (1. - d.p)) : 0.f;
    return r;
}

// With the caller's two words taken in (the same for every lane).
__device__ __forceinline__ void drop_begin(Drop &d) {
    if (d.rng) {
        d.seed = d.rng[0];
        d.offset += d.rng[1];
    }
}

// The four words at a counter.
__device__ __forceinline__ void philox7(uint64_t seed, uint64_t counter, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

// x of N channels (a multiple of 4) from counter `at` on: times `factor`, or 0.
template <int N> __device__ __forceinline__ void drop_n(const Drop &d, uint64_t at, float factor, float *x) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t w[4];
        philox7(d.seed, d.offset + at + q, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * q + j] = (w[j] >> 8) >= d.least ? x[4 * q + j] * factor : 0.f;
    }
}

}  // namespace gdn2
