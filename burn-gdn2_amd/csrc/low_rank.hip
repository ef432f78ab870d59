// gdn2_low_rank_add_*: low-rank adapters of many requests beside a shared projection,
// and their adjoint.  For a row x of a request with adapter l:
//   h = x a_l^T (a [L, R, D]),  out = y + s_l h b_l (b [L, R, O])
//   dh = s_l dy b_l^T,  dx = dh a_l,  da_l = sum dh^T x,  db_l = s_l sum h^T dy
//
// Kernels:
//   adapt   up to 64 ranks: h and out (or dh and dx) of 16 or 32 rows.  The waves of a
//           workgroup share the wide dimension of h, then the columns of out; h stays in
//           LDS.  Each wide tensor is read or written once.
//   shrink, expand  the same in two launches, for more ranks
//   outer   da, db: ranks by 16 VC columns a wave, a block of one request's rows
//   sums    those of an adapter's blocks, in order, in f64
// A tile of rows lies in one request.  Packed requests (cu_seqlens) may take
// floor(first row / tile) + n tiles before request n's: the slots of neighbours never
// overlap, so a workgroup finds its rows from the offsets alone.
//
// Types.  f32: 16x16x4 products of f32.  bfloat16: 16x16x32 products, whose f32 sums are
// exact products of the operands; h and dh are not rounded but enter as three bfloat16
// terms (each the upper half of what is left, 24 bits together: nothing is lost).
//
// Operands.  A lane holds KV neighbouring k of a row of a (one load) and of x, whose rows
// come 256 bytes at a time through LDS of the wave's own.  Where the sum runs over the rows
// instead (b in out; x and dy in da and db), it loads 16 bytes of VC columns from each of
// KV rows and turns them in registers (32 byte permutations for 64 values); a lane's
// column tiles are then its VC neighbouring columns, so that results leave in 16 bytes,
// 16 lanes side by side.
//
// Bound.  2048 features.  8 x 4096 f32 rows, 16 ranks: 158 us, 5.1 TB/s: x alone is read
// at 4.2 (a sum over as much reaches 4.0), y and out pass at 4.9, and the phases of the
// workgroups overlap little.  32767 packed bfloat16 rows, 64 ranks: 128 us, a tile's chain
// of loads and its adapter's 0.5 MB from L2.  64 f32 rows, an adapter of 16 ranks each:
// 13 us, a chain of latencies (offsets or adapter, x and a, the waves' sums, b and y).
// Gradients at 4 x 2048 bfloat16 rows, 16 ranks: 20 us dh and dx, 14 the products, 4
// the sums.  Slower: tiles in the order of the XCDs (211 us for 169).  The same: chunks
// that start elsewhere in each workgroup, x's operands straight from memory.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2_block.h"
#include "loose_io.hpp"

namespace gdn2 {
namespace {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// A place `bytes` behind one that is the same for every lane: 32 bits a lane.  (What the
// lane holds is made opaque, or the compiler forms the 64-bit sums ahead of the loops and
// keeps two registers for each.)
template <typename T> __device__ __forceinline__ const T *behind(const T *p, uint32_t &bytes) {
    asm("" : "+v"(bytes));
    return reinterpret_cast<const T *>(reinterpret_cast<const char *>(p) + bytes);
}
template <typename T> __device__ __forceinline__ T *behind(T *p, uint32_t &bytes) {
    asm("" : "+v"(bytes));
    return reinterpret_cast<T *>(reinterpret_cast<char *>(p) + bytes);
}

template <typename T> struct Mm;
template <> struct Mm<float> {
    static constexpr int KV = 4, VC = 4; // k and columns a lane
    typedef Raw<float, 4> Op;
    typedef Op Wide; // of f32 values
    static __device__ __forceinline__ floatx4 mma(const Op &a, const Op &b, floatx4 c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = mfma16(a[s], b[s], c);
        return c;
    }
    static __device__ __forceinline__ Wide wide(const float *x) { return Op{x[0], x[1], x[2], x[3]}; }
    static __device__ __forceinline__ floatx4 mmw(const Wide &a, const Op &b, floatx4 c) { return mma(a, b, c); }
    static __device__ __forceinline__ void turn(const Raw<float, 4> (&rows)[4], Op (&cols)[4]) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) cols[t][i] = rows[i][t];
    }
};
template <> struct Mm<bf16> {
    static constexpr int KV = 8, VC = 8;
    typedef Raw<bf16, 8> Op;
    struct Wide {
        Op t[3];
    };
    static __device__ __forceinline__ floatx4 mma(const Op &a, const Op &b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Wide wide(const float *x) {
        Wide w;
        float left[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) left[i] = x[i];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uintx4 d;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u0 = __builtin_bit_cast(uint32_t, left[2 * i]), u1 = __builtin_bit_cast(uint32_t, left[2 * i + 1]);
                d[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
                // (an infinity or a NaN is all in the first term)
                left[2 * i] = fabsf(left[2 * i]) < __builtin_inff() ? left[2 * i] - __builtin_bit_cast(float, u0 & 0xFFFF0000u) : 0.f;
                left[2 * i + 1] = fabsf(left[2 * i + 1]) < __builtin_inff() ? left[2 * i + 1] - __builtin_bit_cast(float, u1 & 0xFFFF0000u) : 0.f;
            }
            w.t[k] = __builtin_bit_cast(Op, d);
        }
        return w;
    }
    static __device__ __forceinline__ floatx4 mmw(const Wide &a, const Op &b, floatx4 c) {
        c = mma(a.t[2], b, c);
        c = mma(a.t[1], b, c);
        return mma(a.t[0], b, c);
    }
    static __device__ __forceinline__ void turn(const Raw<bf16, 8> (&rows)[8], Op (&cols)[8]) {
        uintx4 r[8], c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = __builtin_bit_cast(uintx4, rows[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[2 * q][i] = __builtin_amdgcn_perm(r[2 * i + 1][q], r[2 * i][q], 0x05040100);
                c[2 * q + 1][i] = __builtin_amdgcn_perm(r[2 * i + 1][q], r[2 * i][q], 0x07060302);
            }
#pragma unroll
        for (int t = 0; t < 8; ++t) cols[t] = __builtin_bit_cast(Op, c[t]);
    }
};

// -- which rows --------------------------------------------------------------------

struct Requests {
    const int32_t *adapters, *cu;
    int64_t T, M; // rows of a batch entry, of all
    int N, L;     // requests, adapters
    int per;      // without cu: tiles a request
};
struct Tile { // (the same for every lane)
    int b, t0, row; // batch entry, first token, its place among all rows
    int rows;       // <= 0: none
    int adapter;    // -1: none
};

// Row 0, the offsets, the end of the rows: requests 1 .. N between rows of none.
__device__ __forceinline__ int bound_at(const Requests &r, int n) {
    if (n == 0) return 0;
    if (n == r.N + 2) return (int)r.M;
    return min(max(r.cu[n - 1], 0), (int)r.M);
}

// Of the wave's tile w (the same for every lane) of up to `size` rows.
__device__ __forceinline__ Tile tile_at(const Requests &r, int w, int size) {
    Tile t{};
    t.adapter = -1;
    int n;
    if (!r.cu) {
        n = w / r.per;
        t.b = n;
        t.t0 = (w - n * r.per) * size; // (the last request's last tile: < 2^30 + 64)
        t.row = n * (int)r.T + t.t0;
        t.rows = min(size, (int)r.T - t.t0);
    } else {
        // the last n with bound / size + n <= w: 64 at a time
        int lo = 0, len = r.N + 2;
        while (len > 1) {
            const int step = (len + kWave - 1) / kWave, i = lo + (int)(threadIdx.x & 63) * step;
            const bool before = i < lo + len && bound_at(r, i) / size + i <= w;
            const int c = max(1, (int)__popcll(__ballot(before)));
            const int end = lo + len;
            lo += (c - 1) * step;
            len = step == 1 ? 1 : min(step, end - lo);
        }
        n = __builtin_amdgcn_readfirstlane(lo);
        const int first = __builtin_amdgcn_readfirstlane(bound_at(r, n));
        const int64_t t0 = first + (int64_t)(w - (first / size + n)) * size;
        const int64_t rows = min((int64_t)size, __builtin_amdgcn_readfirstlane(bound_at(r, n + 1)) - t0);
        if (t0 < 0 || rows <= 0) return t; // (offsets that decrease; a slot without a tile)
        t.t0 = t.row = (int)t0;
        t.rows = (int)rows;
        if (n == 0 || n == r.N + 1) return t;
        --n;
    }
    const int id = __builtin_amdgcn_readfirstlane(r.adapters[n]);
    if (id >= 0 && id < r.L) t.adapter = id;
    return t;
}

// -- shrink ----------------------------------------------------------------------------

struct ShrinkParams {
    Requests req;
    const void *x, *w; // [.., K]; [L, R, K]
    const float *scale;
    float *h; // [M][P], zeros behind rank R
    int64_t xb, xt, wl, wr;
    int64_t K;
    int R, P;
};

constexpr int kStagePitch = 17; // (16 bytes: a row's 16 and one)

// acc of wave 0: the tile's rows by 16 NR ranks from r0 on.  lds: W MT 16 kStagePitch or
// MT NR 64 W / 2 of 16 bytes.  A wave takes 256 bytes of each of its rows at a time, 16 lanes a row, and turns them
// into operands through LDS of its own; the next ones' loads are in flight meanwhile.
// (Operands loaded as they are used, 64 bytes of each of 16 rows a load, kept the same
// tiles at 3.3 TB/s.)
template <typename T, int MT, int NR, int W>
__device__ __forceinline__ void shrink_rows(floatx4 *lds, const void *px, int64_t xb, int64_t xt, const void *pw, int64_t wl, int64_t wr,
                                            int64_t K, int R, int r0, const Tile &at, floatx4 (&acc)[MT][NR]) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, STEP = 4 * KV, U = 4, CHUNK = U * STEP, kStageW = MT * 16 * kStagePitch;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    // (rows behind the tile's last, ranks behind the last: the last one's again, not stored)
    const T *x = static_cast<const T *>(px) + (int64_t)at.b * xb + (int64_t)at.t0 * xt;
    const T *w = static_cast<const T *>(pw) + (int64_t)at.adapter * wl + (int64_t)r0 * wr;
    uint32_t xo[MT * 4], wo[NR];
#pragma unroll
    for (int j = 0; j < MT * 4; ++j) xo[j] = (uint32_t)(min(4 * j + g, at.rows - 1) * (uint32_t)xt + KV * i) * sizeof(T);
#pragma unroll
    for (int n = 0; n < NR; ++n) wo[n] = (uint32_t)(min(16 * n + i, R - 1 - r0) * (uint32_t)wr + KV * g) * sizeof(T);
    floatx4 *stage = lds + wave * kStageW;
    typename X::Op ahead[MT * 4], b[U][NR];
    auto load_x = [&](int64_t k) {
#pragma unroll
        for (int j = 0; j < MT * 4; ++j) ahead[j] = loose<T, KV>(behind(x + k, xo[j]));
    };
    auto load_w = [&](int64_t k, int s) {
#pragma unroll
        for (int n = 0; n < NR; ++n) b[s][n] = loose<T, KV>(behind(w + k + s * STEP, wo[n]));
    };
    int64_t k = (int64_t)wave * CHUNK;
    if (k + CHUNK <= K) {
        load_x(k);
#pragma unroll
        for (int s = 0; s < U; ++s) load_w(k, s);
    }
    for (; k + CHUNK <= K; k += W * CHUNK) {
#pragma unroll
        for (int j = 0; j < MT * 4; ++j) stage[(4 * j + g) * kStagePitch + i] = __builtin_bit_cast(floatx4, ahead[j]);
        const bool more = k + (W + 1) * CHUNK <= K;
        const int64_t next = more ? k + W * CHUNK : k; // (the last chunk's again, not used)
        load_x(next);
        __builtin_amdgcn_wave_barrier(); // (one wave's LDS operations are done in order)
#pragma unroll
        for (int s = 0; s < U; ++s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const typename X::Op a = __builtin_bit_cast(typename X::Op, stage[(16 * m + i) * kStagePitch + 4 * s + g]);
#pragma unroll
                for (int n = 0; n < NR; ++n) acc[m][n] = X::mma(a, b[s][n], acc[m][n]);
            }
            load_w(next, s);
        }
        __builtin_amdgcn_wave_barrier();
    }
    // less than a chunk: a step each of the waves whose turn it is
    const int64_t whole = K / CHUNK;
    for (int64_t t = whole * CHUNK + ((wave + W - (int)(whole % W)) % W) * STEP; t < K; t += W * STEP) {
        const int64_t left = K - t - KV * g;
#pragma unroll
        for (int n = 0; n < NR; ++n) b[0][n] = loose_part<T, KV>(behind(w + t, wo[n]), left);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const typename X::Op a = loose_part<T, KV>(x + min(16 * m + i, at.rows - 1) * xt + t + KV * g, left);
#pragma unroll
            for (int n = 0; n < NR; ++n) acc[m][n] = X::mma(a, b[0][n], acc[m][n]);
        }
    }
    // the waves' sums: the upper half's onto the lower, and so on
    auto red = [&](int w, int n) -> floatx4 & { return lds[(w * MT * NR + n) * kWave + lane]; };
#pragma unroll
    for (int half = W / 2; half >= 1; half /= 2) {
        __syncthreads(); // what was here has been read
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NR; ++n) red(wave - half, m * NR + n) = acc[m][n];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NR; ++n) acc[m][n] += red(wave, m * NR + n);
    }
}

template <typename T, int MT, int NR, int W> __global__ __launch_bounds__(64 * W, 2) void shrink_kernel(ShrinkParams p) {
    constexpr int kStage = W * MT * 16 * kStagePitch, kSums = MT * NR * kWave * (W / 2);
    __shared__ floatx4 lds[kStage > kSums ? kStage : kSums];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, r0 = blockIdx.y * NR * 16;
    const Tile at = tile_at(p.req, blockIdx.x, MT * 16);
    if (at.rows <= 0) return;
    floatx4 acc[MT][NR];
    if (at.adapter >= 0) {
        shrink_rows<T, MT, NR, W>(lds, p.x, p.xb, p.xt, p.w, p.wl, p.wr, p.K, p.R, r0, at, acc);
    } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NR; ++n) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (threadIdx.x >= 64) return;
    const float s = p.scale && at.adapter >= 0 ? p.scale[at.adapter] : 1.f;
    float *h = p.h + (int64_t)at.row * p.P;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * m + 4 * g + q, r = r0 + 16 * n + i;
                if (row < at.rows && r < p.P) h[(int64_t)row * p.P + r] = r < p.R ? s * acc[m][n][q] : 0.f;
            }
}

// -- expand ----------------------------------------------------------------------------

constexpr int kExpandRows = 32;

struct ExpandParams {
    Requests req;
    const float *h; // [M][P], zeros behind rank R
    const void *w;  // [L, R, C]
    const void *y;  // or NULL
    void *out;
    const float *scale;
    float *hidden; // [M][R] h's copy for the caller, or NULL
    int64_t wl, wr, yb, yt, ob, ot;
    int64_t C;
    int R, P, groups; // workgroups over the columns
    int copies; // rows without an adapter are written too (out is not y's memory)
};

// Rows without an adapter: y as it is, NaN and all, or zeros.
template <typename T, typename P> __device__ __forceinline__ void copy_columns(const P &p, const Tile &at, int64_t c0) {
    constexpr int VC = Mm<T>::VC;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int64_t c = c0 + VC * i, left = p.C - c;
    const T *y = p.y ? static_cast<const T *>(p.y) + (int64_t)at.b * p.yb + (int64_t)at.t0 * p.yt + c : nullptr;
    T *out = static_cast<T *>(p.out) + (int64_t)at.b * p.ob + (int64_t)at.t0 * p.ot + c;
    for (int row = g; row < at.rows; row += 4) {
        float v[VC];
#pragma unroll
        for (int t = 0; t < VC; ++t) v[t] = 0.f;
        if (y) load_part<T, VC>(y + row * p.yt, left, v);
        store_part<T, VC>(out + row * p.ot, left, v);
    }
}
template <typename T> __device__ __forceinline__ void expand_copy(const ExpandParams &p, const Tile &at, int64_t c0, bool keep) {
    if (keep)
        for (int64_t k = threadIdx.x & 63; k < (int64_t)at.rows * p.R; k += kWave) p.hidden[(int64_t)at.row * p.R + k] = 0.f;
    if (p.copies) copy_columns<T>(p, at, c0);
}

// WHOLE: VC columns or more are left.  A lane whose columns would end behind the last
// takes the last VC ones: what another lane of the wave takes too, with the same result.
template <typename T, int MT, bool WHOLE>
__device__ __forceinline__ void expand_tile(const ExpandParams &p, const Tile &at, int64_t c0, bool keep) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, VC = X::VC, STEP = 4 * KV;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int64_t c = WHOLE ? min(c0 + VC * i, p.C - VC) : c0 + VC * i, left = p.C - c;
    auto cols_at = [&](const T *q) { return WHOLE ? loose<T, VC>(q) : loose_part<T, VC>(q, left); };
    const T *w = static_cast<const T *>(p.w) + (int64_t)at.adapter * p.wl + c;
    Raw<T, VC> rows[KV];
    float h[MT][KV];
    auto load = [&](int r0) { // (behind the last rank: zeros)
        const int r = r0 + KV * g;
#pragma unroll
        for (int k = 0; k < KV; ++k) rows[k] = cols_at(w + (int64_t)min(r + k, p.R - 1) * p.wr);
#pragma unroll
        for (int m = 0; m < MT; ++m)
            load_n<float, KV>(p.h + (int64_t)(at.row + min(16 * m + i, at.rows - 1)) * p.P + min(r, p.P - KV), h[m]);
        if (r0 + STEP > p.R) {
#pragma unroll
            for (int k = 0; k < KV; ++k)
                if (r + k >= p.R)
#pragma unroll
                    for (int t = 0; t < VC; ++t) rows[k][t] = (T)0.f;
            if (r >= p.P)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int k = 0; k < KV; ++k) h[m][k] = 0.f;
        }
    };
    load(0);
    Raw<T, VC> old[MT][4];
    if (p.y) {
        const T *y = static_cast<const T *>(p.y) + (int64_t)at.b * p.yb + (int64_t)at.t0 * p.yt + c;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < 4; ++q) old[m][q] = cols_at(y + min(16 * m + 4 * g + q, at.rows - 1) * p.yt);
    }
    floatx4 acc[MT][VC];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < VC; ++t) acc[m][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < p.R; r0 += STEP) {
        typename X::Op cols[VC];
        X::turn(rows, cols);
        typename X::Wide hw[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            hw[m] = X::wide(h[m]);
            const int r = r0 + KV * g;
            if (keep && 16 * m + i < at.rows) store_part<float, KV>(p.hidden + (int64_t)(at.row + 16 * m + i) * p.R + r, p.R - r, h[m]);
        }
        if (r0 + STEP < p.R) load(r0 + STEP);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < VC; ++t) acc[m][t] = X::mmw(hw[m], cols[t], acc[m][t]);
    }
    const float s = p.scale ? p.scale[at.adapter] : 1.f;
    T *out = static_cast<T *>(p.out) + (int64_t)at.b * p.ob + (int64_t)at.t0 * p.ot + c;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = 16 * m + 4 * g + q;
            if (row >= at.rows) continue;
            float v[VC];
#pragma unroll
            for (int t = 0; t < VC; ++t) v[t] = __builtin_fmaf(s, acc[m][t][q], p.y ? (float)old[m][q][t] : 0.f);
            if constexpr (WHOLE) loose_store<T, VC>(out + row * p.ot, v);
            else store_part<T, VC>(out + row * p.ot, left, v);
        }
}

template <typename T> __global__ __launch_bounds__(256, 2) void expand_kernel(ExpandParams p) {
    constexpr int VC = Mm<T>::VC;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x / p.groups, group = blockIdx.x - tile * p.groups;
    const int64_t c0 = (int64_t)(group * 4 + wave) * 16 * VC;
    if (c0 >= p.C && !(p.hidden && c0 == 0)) return;
    const Tile at = tile_at(p.req, tile, kExpandRows);
    if (at.rows <= 0) return;
    const bool keep = p.hidden && c0 == 0;
    if (at.adapter < 0 || p.R == 0) expand_copy<T>(p, at, c0, keep);
    else if (p.C - c0 >= VC) expand_tile<T, kExpandRows / 16, true>(p, at, c0, keep);
    else expand_tile<T, kExpandRows / 16, false>(p, at, c0, keep);
}

// -- adapt: both at once, up to 64 ranks -----------------------------------------------

struct AdaptParams {
    Requests req;
    const void *x, *w1; // [.., K]; [L, R, K]
    const void *w2, *y; // [L, R, C]; y or NULL
    void *out;          // or NULL
    const float *scale;
    float *hidden; // [M][pitch] h for the caller, or NULL
    int64_t xb, xt, w1l, w1r, w2l, w2r, yb, yt, ob, ot, pitch;
    int64_t K, C;
    int R;
    int copies;        // rows without an adapter are written too (out is not y's memory)
    int scale_hidden;  // hidden times the scale (dh)
    int stream;        // out is too large for the caches
};

// h of a tile in LDS, as the second product's operands.
template <typename T, int MT, int NR> struct Kept;
template <int MT, int NR> struct Kept<float, MT, NR> {
    static constexpr int KR = NR, PITCH = 16 * NR + 4;
    static constexpr int BYTES = MT * 16 * PITCH * 4;
    static __device__ __forceinline__ void put(void *lds, int row, int r, float v) { static_cast<float *>(lds)[row * PITCH + r] = v; }
    static __device__ __forceinline__ float value(const void *lds, int row, int r) { return static_cast<const float *>(lds)[row * PITCH + r]; }
    static __device__ __forceinline__ Mm<float>::Wide get(const void *lds, int row, int r) {
        return *reinterpret_cast<const Mm<float>::Op *>(static_cast<const float *>(lds) + row * PITCH + r);
    }
};
template <int MT, int NR> struct Kept<bf16, MT, NR> { // three planes of terms
    static constexpr int KR = (NR + 1) / 2, PITCH = 32 * KR + 8, PLANE = MT * 16 * PITCH;
    static constexpr int BYTES = 3 * PLANE * 2;
    static __device__ __forceinline__ void put(void *lds, int row, int r, float v) {
        uint16_t *to = static_cast<uint16_t *>(lds) + row * PITCH + r;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t u = __builtin_bit_cast(uint32_t, v);
            to[k * PLANE] = (uint16_t)(u >> 16);
            v = fabsf(v) < __builtin_inff() ? v - __builtin_bit_cast(float, u & 0xFFFF0000u) : 0.f;
        }
    }
    static __device__ __forceinline__ float value(const void *lds, int row, int r) {
        const uint16_t *from = static_cast<const uint16_t *>(lds) + row * PITCH + r;
        float v = 0.f;
#pragma unroll
        for (int k = 2; k >= 0; --k) v += __builtin_bit_cast(float, (uint32_t)from[k * PLANE] << 16);
        return v;
    }
    static __device__ __forceinline__ Mm<bf16>::Wide get(const void *lds, int row, int r) {
        Mm<bf16>::Wide w;
#pragma unroll
        for (int k = 0; k < 3; ++k)
            w.t[k] = *reinterpret_cast<const Mm<bf16>::Op *>(static_cast<const uint16_t *>(lds) + k * PLANE + row * PITCH + r);
        return w;
    }
};

// A wave's columns of a tile's rows: 16 VC of every W times as many, the next ones' y
// (and b, where the registers do) in flight.
// (Fewer than VC columns behind the last whole tile are adapt_rest's.)
template <typename T, int MT, int NR, int W> struct Columns {
    typedef Mm<T> X;
    typedef Kept<T, MT, NR> H;
    static constexpr int KV = X::KV, VC = X::VC, STEP = 4 * KV, KR = H::KR, NEXT = W * 16 * VC;
    static constexpr bool AHEAD = sizeof(T) == 4 && NR <= 2;
    const AdaptParams &p;
    const Tile &at;
    const int i, g;
    const T *w, *y;
    T *out;
    Raw<T, VC> rows[KR][KV], old[MT][4];

    __device__ __forceinline__ Columns(const AdaptParams &p, const Tile &at)
        : p(p), at(at), i(threadIdx.x & 15), g((threadIdx.x & 63) >> 4),
          w(static_cast<const T *>(p.w2) + (int64_t)at.adapter * p.w2l),
          y(p.y ? static_cast<const T *>(p.y) + (int64_t)at.b * p.yb + (int64_t)at.t0 * p.yt : nullptr),
          out(static_cast<T *>(p.out) + (int64_t)at.b * p.ob + (int64_t)at.t0 * p.ot) {}

    // a lane's columns from c0 on: where they would end behind the last, the last VC
    __device__ __forceinline__ int place(int64_t c0) const { return min(VC * i, (int)min(p.C - VC - c0, (int64_t)(16 * VC))); }
    __device__ __forceinline__ bool more(int64_t c0) const { return p.out && c0 + VC <= p.C; }
    __device__ __forceinline__ void load_w(int64_t c0) {
        const int c = place(c0);
#pragma unroll
        for (int s = 0; s < KR; ++s)
#pragma unroll
            for (int k = 0; k < KV; ++k) {
                uint32_t o = (uint32_t)(min(s * STEP + KV * g + k, p.R - 1) * (uint32_t)p.w2r + c) * sizeof(T);
                rows[s][k] = loose<T, VC>(behind(w + c0, o));
            }
    }
    __device__ __forceinline__ void load_y(int64_t c0, int m) {
        const int c = place(c0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t o = (uint32_t)(min(16 * m + 4 * g + q, at.rows - 1) * (uint32_t)p.yt + c) * sizeof(T);
            old[m][q] = loose<T, VC>(behind(y + c0, o));
        }
    }
    __device__ __forceinline__ void load(int64_t c0) {
        if (!more(c0)) return;
        load_w(c0);
        if (y)
#pragma unroll
            for (int m = 0; m < MT; ++m) load_y(c0, m);
    }
    // (after load(c0))
    __device__ __forceinline__ void run(const void *kept, int64_t c0) {
        for (; more(c0); c0 += NEXT) {
            typename X::Op cols[KR][VC];
#pragma unroll
            for (int s = 0; s < KR; ++s) {
                if ((s + 1) * STEP > p.R) // behind the last rank: zeros
#pragma unroll
                    for (int k = 0; k < KV; ++k)
                        if (s * STEP + KV * g + k >= p.R)
#pragma unroll
                            for (int t = 0; t < VC; ++t) rows[s][k][t] = (T)0.f;
                X::turn(rows[s], cols[s]);
            }
            const bool next = more(c0 + NEXT);
            if (AHEAD && next) load_w(c0 + NEXT);
            const int c = place(c0);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (16 * m >= at.rows) break;
                typename X::Wide hw[KR];
#pragma unroll
                for (int s = 0; s < KR; ++s) hw[s] = H::get(kept, 16 * m + i, s * STEP + KV * g);
                floatx4 acc[VC];
#pragma unroll
                for (int t = 0; t < VC; ++t) {
                    acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KR; ++s) acc[t] = X::mmw(hw[s], cols[s][t], acc[t]);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = 16 * m + 4 * g + q;
                    if (row >= at.rows) continue;
                    float v[VC];
#pragma unroll
                    for (int t = 0; t < VC; ++t) v[t] = acc[t][q] + (y ? (float)old[m][q][t] : 0.f);
                    uint32_t o = (uint32_t)(row * (uint32_t)p.ot + c) * sizeof(T);
                    loose_store<T, VC>(behind(out + c0, o), v, p.stream);
                }
                if (y && next) load_y(c0 + NEXT, m);
            }
            if (!AHEAD && next) {
                __builtin_amdgcn_sched_barrier(0); // (not ahead of the products: for the registers)
                load_w(c0 + NEXT);
            }
        }
    }
};

// The few columns from c0 on, one value a lane at a time.
template <typename T, int MT, int NR> __device__ __forceinline__ void adapt_rest(const AdaptParams &p, const Tile &at, const void *kept, int64_t c0) {
    typedef Kept<T, MT, NR> H;
    const int n = (int)(p.C - c0);
    const T *w = static_cast<const T *>(p.w2) + (int64_t)at.adapter * p.w2l + c0;
    const T *y = p.y ? static_cast<const T *>(p.y) + (int64_t)at.b * p.yb + (int64_t)at.t0 * p.yt + c0 : nullptr;
    T *out = static_cast<T *>(p.out) + (int64_t)at.b * p.ob + (int64_t)at.t0 * p.ot + c0;
    for (int e = threadIdx.x & 63; e < at.rows * n; e += kWave) {
        const int row = e / n, c = e - row * n;
        float sum = 0.f;
#pragma unroll 8
        for (int r = 0; r < p.R; ++r) sum = __builtin_fmaf(H::value(kept, row, r), (float)w[r * p.w2r + c], sum);
        out[row * p.ot + c] = (T)(sum + (y ? (float)y[row * p.yt + c] : 0.f));
    }
}

template <typename T, int MT, int NR, int W, int WPE> __global__ __launch_bounds__(64 * W, WPE) void adapt_kernel(AdaptParams p) {
    typedef Mm<T> X;
    typedef Kept<T, MT, NR> H;
    constexpr int VC = X::VC, kStage = W * MT * 16 * kStagePitch * 16, kSums = MT * NR * kWave * (W / 2) * 16;
    constexpr int kLds = (kStage > kSums ? kStage : kSums) > H::BYTES ? (kStage > kSums ? kStage : kSums) : H::BYTES;
    __shared__ __attribute__((aligned(16))) char lds[kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const Tile at = tile_at(p.req, blockIdx.x, MT * 16);
    if (at.rows <= 0) return;
    if (at.adapter < 0) {
        if (p.hidden)
            for (int k = threadIdx.x; k < at.rows * p.R; k += 64 * W) p.hidden[(int64_t)(at.row + k / p.R) * p.pitch + k % p.R] = 0.f;
        if (p.out && p.copies)
            for (int64_t c0 = (int64_t)wave * 16 * VC; c0 < p.C; c0 += W * 16 * VC) copy_columns<T>(p, at, c0);
        return;
    }
    floatx4 acc[MT][NR];
    shrink_rows<T, MT, NR, W>(reinterpret_cast<floatx4 *>(lds), p.x, p.xb, p.xt, p.w1, p.w1l, p.w1r, p.K, p.R, 0, at, acc);
    __syncthreads(); // the last sums have been read
    if (wave == 0) {
        const float s = p.scale ? p.scale[at.adapter] : 1.f;
        // (bfloat16: a step of 32 ranks, of which 16 may be beyond the tiles: zeros)
        constexpr int NZ = H::KR * 4 * X::KV / 16;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NZ; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = 16 * m + 4 * g + q, r = 16 * n + i;
                    const float v = n < NR && r < p.R ? acc[m][n < NR ? n : 0][q] : 0.f;
                    H::put(lds, row, r, s * v);
                    if (p.hidden && row < at.rows && r < p.R) p.hidden[(int64_t)(at.row + row) * p.pitch + r] = p.scale_hidden ? s * v : v;
                }
    }
    if (!p.out) return;
    Columns<T, MT, NR, W> columns(p, at);
    columns.load((int64_t)wave * 16 * VC);
    __syncthreads();
    columns.run(lds, (int64_t)wave * 16 * VC);
    // the last tile of columns, where it has less than a lane's: one wave's
    const int64_t last = p.C / (16 * VC);
    if (p.C - last * 16 * VC > 0 && p.C - last * 16 * VC < VC && wave == last % W)
        adapt_rest<T, MT, NR>(p, at, lds, last * 16 * VC);
}

// -- outer -----------------------------------------------------------------------------

struct OuterParams {
    Requests req;
    const void *z[2];  // x with dh for da, dy with h for db
    const float *h[2]; // [M][pitch]
    int64_t pitch[2];
    float *part[2];    // [blocks][R][C]
    int64_t zb[2], zt[2], C[2];
    int tiles[2]; // column tiles
    int *adapter; // of each block
    int R, rows;  // rows a block
};

// Waves: WS shares of the ranks, 16 NR each, by 4 / WS shares of the rows.
template <typename T, int NR, int WS, bool WHOLE>
__device__ __forceinline__ void outer_tile(const OuterParams &p, const Tile &at, int block, int which, int64_t c0, int rs,
                                           floatx4 (*red)[WS][NR * Mm<T>::VC][kWave]) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, VC = X::VC, STEP = 4 * KV, NS = 4 / WS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, ws = wave % WS, ms = wave / WS;
    const int r0 = (rs * WS + ws) * NR * 16;
    const int64_t C = p.C[which], c = WHOLE ? min(c0 + VC * i, C - VC) : c0 + VC * i, left = C - c;
    const T *z = static_cast<const T *>(p.z[which]) + (int64_t)at.b * p.zb[which] + (int64_t)at.t0 * p.zt[which] + c;
    const int64_t zt = p.zt[which], pitch = p.pitch[which];
    const float *h[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) h[n] = p.h[which] + (int64_t)at.row * pitch + min(r0 + 16 * n + i, p.R - 1);
    floatx4 acc[NR][VC];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int t = 0; t < VC; ++t) acc[n][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    Raw<T, VC> rows[KV];
    float hv[NR][KV];
    auto load = [&](int m0) { // (ranks behind the last: the last one's again, not stored)
        const int m = m0 + KV * g;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int row = min(m + k, at.rows - 1);
            rows[k] = WHOLE ? loose<T, VC>(z + row * zt) : loose_part<T, VC>(z + row * zt, left);
#pragma unroll
            for (int n = 0; n < NR; ++n) hv[n][k] = h[n][row * pitch];
        }
        if (m0 + STEP > at.rows) // behind the last row: zeros
#pragma unroll
            for (int k = 0; k < KV; ++k)
                if (m + k >= at.rows) {
#pragma unroll
                    for (int t = 0; t < VC; ++t) rows[k][t] = (T)0.f;
#pragma unroll
                    for (int n = 0; n < NR; ++n) hv[n][k] = 0.f;
                }
    };
    if (ms * STEP < at.rows) load(ms * STEP);
    for (int m0 = ms * STEP; m0 < at.rows; m0 += NS * STEP) {
        typename X::Op cols[VC];
        X::turn(rows, cols);
        typename X::Wide hw[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) hw[n] = X::wide(hv[n]);
        if (m0 + NS * STEP < at.rows) load(m0 + NS * STEP);
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int t = 0; t < VC; ++t) acc[n][t] = X::mmw(hw[n], cols[t], acc[n][t]);
    }
#pragma unroll
    for (int half = NS / 2; half >= 1; half /= 2) {
        if (ms >= half && ms < 2 * half)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int t = 0; t < VC; ++t) red[ms - half][ws][n * VC + t][lane] = acc[n][t];
        __syncthreads();
        if (ms < half)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int t = 0; t < VC; ++t) acc[n][t] += red[ms][ws][n * VC + t][lane];
        if (half > 1) __syncthreads();
    }
    if (ms) return;
    float *part = p.part[which] + (int64_t)block * p.R * C + c;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = r0 + 16 * n + 4 * g + q;
            if (r >= p.R) continue;
            float v[VC];
#pragma unroll
            for (int t = 0; t < VC; ++t) v[t] = acc[n][t][q];
            if constexpr (WHOLE) loose_store<float, VC>(part + r * C, v);
            else store_part<float, VC>(part + r * C, left, v);
        }
}

template <typename T, int NR, int WS> __global__ __launch_bounds__(256, 2) void outer_kernel(OuterParams p) {
    constexpr int VC = Mm<T>::VC;
    __shared__ floatx4 red[2 / WS][WS][NR * VC][kWave];
    const int tiles = p.tiles[0] + p.tiles[1], block = blockIdx.x / tiles, ct = blockIdx.x - block * tiles;
    const int which = ct >= p.tiles[0];
    const Tile at = tile_at(p.req, block, p.rows);
    const bool any = at.rows > 0 && at.adapter >= 0;
    if (ct == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.adapter[block] = any ? at.adapter : -1;
    if (!any) return;
    const int64_t c0 = (int64_t)(ct - which * p.tiles[0]) * 16 * VC;
    if (p.C[which] - c0 >= VC) outer_tile<T, NR, WS, true>(p, at, block, which, c0, blockIdx.y, red);
    else outer_tile<T, NR, WS, false>(p, at, block, which, c0, blockIdx.y, red);
}

struct SumsParams {
    const float *part[2];
    float *out[2];
    int64_t n[2]; // R C
    int tiles[2]; // workgroups an adapter
    const int *adapter;
    const float *scale; // of db
    int blocks;
};

// 256 values a workgroup: each of its waves adds every fourth of the adapter's blocks,
// eight of them in flight.
__global__ __launch_bounds__(256) void adapter_sums_kernel(SumsParams p) {
    __shared__ double red[3][kWave][4];
    const int tiles = p.tiles[0] + p.tiles[1], l = blockIdx.x / tiles, ct = blockIdx.x - l * tiles;
    const int which = ct >= p.tiles[0], lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n = p.n[which], e = ((int64_t)(ct - which * p.tiles[0]) * kWave + lane) * 4, left = n - e;
    const float *part = p.part[which] + e;
    double sum[4] = {0., 0., 0., 0.};
    bool any = false; // (the same in every wave)
    for (int b0 = 0; b0 < p.blocks; b0 += kWave) {
        const int b = b0 + lane;
        uint64_t mine = __ballot(b < p.blocks && p.adapter[b < p.blocks ? b : 0] == l);
        any |= mine != 0;
        while (mine) {
            int at[8], count = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) at[k] = 0;
            // (the same for every lane)
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const int first = mine ? __builtin_ctzll(mine) : 0;
                if (mine && (k & 3) == wave) at[k / 4] = b0 + first, count = k / 4 + 1;
                mine &= mine - 1; // (0 stays 0)
            }
            float v[8][4];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < count) load_part<float, 4>(part + at[k] * n, left, v[k]);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < count)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[j] += v[k][j];
        }
    }
    if (wave)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[wave - 1][lane][j] = sum[j];
    __syncthreads();
    if (wave || left <= 0) return;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double t = (sum[j] + red[0][lane][j]) + (red[1][lane][j] + red[2][lane][j]);
        v[j] = (float)(which && p.scale && any ? p.scale[l] * t : t); // (no rows: 0)
    }
    store_part<float, 4>(p.out[which] + l * n + e, left, v);
}

// -- the calls -------------------------------------------------------------------------

constexpr int kMostRank = 512;

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t up(int64_t n, int64_t d) { return (n + d - 1) / d; }

struct Shape {
    int64_t M, N; // rows, requests
    bool packed;
    int64_t T;
    int64_t tiles(int size) const { return packed ? M / size + N + 2 : N * up(T, size); }
};
Shape shape_of(const gdn2_low_rank_args &a) {
    Shape s{};
    s.M = a.batch * a.seq_len;
    s.packed = a.cu_seqlens != nullptr;
    s.N = s.packed ? a.num_seqs : a.batch;
    s.T = a.seq_len;
    return s;
}
Requests requests_of(const gdn2_low_rank_args &a, const Shape &s, int size) {
    Requests r{};
    r.adapters = a.adapters; r.cu = a.cu_seqlens;
    r.T = a.seq_len; r.M = s.M;
    r.N = (int)s.N; r.L = (int)a.num_adapters;
    r.per = (int)std::max<int64_t>(1, up(a.seq_len, size));
    return r;
}

// Rows a block of the outer products: 256 blocks by columns, while each has 128 rows or
// more and at most 4096 (4 x 2048 x 2048 bf16, 16 ranks: the whole backward 37.8 us; 512
// of them 39.5, 1024 40.5: more to add up).
int block_rows(const Shape &s, int64_t columns, int tile_columns) {
    const int64_t per = up(columns, tile_columns);
    int rows = 4096;
    while (rows > 128 && s.tiles(rows) * per < 256) rows /= 2;
    return rows;
}

bool sizes_ok(const gdn2_low_rank_args &a) {
    const double M = (double)a.batch * (double)a.seq_len;
    return M < 1073741824. && a.batch < (1 << 30) && a.seq_len < (1 << 30) && a.num_seqs < (1 << 24) && a.rank <= kMostRank &&
           a.in_features < (1 << 24) && a.out_features < (1 << 24) && a.num_adapters < (1 << 24);
}


int64_t pitch_of(int64_t R) { return up(R, 16) * 16; }
// Bytes of h.
size_t hidden_bytes(const Shape &s, int64_t R) { return align256(sizeof(float) * (size_t)s.M * (size_t)pitch_of(R)); }

constexpr int kFusedRank = 64; // ranks that adapt's tiles hold

// Rows a tile of adapt: 32 where a request has more than 16 and the adapter's ranks cost
// more to read again than tiles that fill the card: from 1024 such tiles on for 17 to 32
// ranks (2048 features, f32: 182 us against 198 at 32768 rows, 99 against 95 at 16384),
// from 256 on for more (64 ranks, bfloat16: 128 against 168 at 32767, 36 against 43 at
// 8192, 27 against 24 at 4096).  Of up to 16 ranks 16 rows (f32: 159 us against 180 at
// 32768, 26 against 33 at 4096) but in bfloat16, of half as many bytes a row, where tiles of
// 32 come at most one to a compute unit (the registers of its form allow one there) and tiles
// of 16 come more than one: 128 to 256 tiles of 32 (the gradients at 160, 192 and 256: 31.8,
// 33.5 and 39.0 us, of 16 rows 34.2, 35.9 and 40.7; the forward 23.0, 22.9 and 29.1 against
// 23.2, 23.9 and 27.2; at 64 and 128 both the same; from 257 on, where a second round
// follows, 51.9 against 46.7 and 40.8 against 34.9).
int adapt_rows(const Shape &s, int64_t R, size_t element) {
    if (s.N <= 0 || up(s.M, s.N) <= 16) return 16;
    const int64_t tiles = s.tiles(32);
    if (R <= 16) return element == 2 && tiles >= 128 && tiles <= 256 ? 32 : 16;
    return tiles >= (R <= 32 ? 1024 : 256) ? 32 : 16;
}

template <typename T> gdn2_status launch_adapt(AdaptParams p, const gdn2_low_rank_args &a, const Shape &sh, hipStream_t s) {
    const int size = adapt_rows(sh, p.R, sizeof(T));
    const int64_t tiles = sh.tiles(size);
    p.req = requests_of(a, sh, size);
    p.stream = (double)sh.M * (double)p.C * sizeof(T) >= kStreamBytes;
#define GDN2_RUN(MT, NR, W, WPE) hipLaunchKernelGGL((adapt_kernel<T, MT, NR, W, WPE>), dim3((unsigned)tiles), dim3(64 * W), 0, s, p)
    // Eight waves a tile where tiles are few: their share of a chain of loads is shorter;
    // four of them from 512 tiles of 16 rows on (16 ranks, 16384 bfloat16 rows: 46 us
    // against 50; 64 ranks 81 and 92; 8192 f32 rows, 16 ranks: 47 and 46).
    if (size == 32) {
        if (p.R <= 16) {
            if constexpr (sizeof(T) == 2) GDN2_RUN(2, 1, 8, 2); // (f32: never of so few ranks)
        } else if (p.R <= 32) GDN2_RUN(2, 2, 4, 3);
        else GDN2_RUN(2, 4, 4, 2);
    } else if (tiles >= 512) {
        if (p.R <= 16) GDN2_RUN(1, 1, 4, 4);
        else if (p.R <= 32) GDN2_RUN(1, 2, 4, 4);
        else GDN2_RUN(1, 4, 4, 2);
    } else {
        if (p.R <= 16) GDN2_RUN(1, 1, 8, 4);
        else if (p.R <= 32) GDN2_RUN(1, 2, 8, 4);
        else GDN2_RUN(1, 4, 8, 2);
    }
#undef GDN2_RUN
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

// More ranks: 64 of them a workgroup in shrink, and 64 rows where there are 512 tiles of
// them (128 ranks, 8 x 4096 bfloat16 rows: 170 us of the whole call against 297; 8 x 1024
// f32 rows 103 against 145; 64 requests of one or 16 of 33 rows: the same).
int shrink_rows_of(const Shape &s) { return s.N > 0 && up(s.M, s.N) > 32 && s.tiles(64) >= 128 ? 64 : 16; }
template <typename T> gdn2_status launch_shrink(ShrinkParams p, const gdn2_low_rank_args &a, const Shape &sh, hipStream_t s) {
    const int size = shrink_rows_of(sh);
    p.req = requests_of(a, sh, size);
    const dim3 grid((unsigned)sh.tiles(size), (unsigned)up(p.R, 64));
    if (size == 64) hipLaunchKernelGGL((shrink_kernel<T, 4, 4, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((shrink_kernel<T, 1, 4, 8>), grid, dim3(512), 0, s, p);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

template <typename T> int64_t groups_of(int64_t C) { return std::max<int64_t>(1, up(C, 4 * 16 * Mm<T>::VC)); }

template <typename T> gdn2_status launch_expand(ExpandParams p, const gdn2_low_rank_args &a, const Shape &sh, hipStream_t s) {
    p.req = requests_of(a, sh, kExpandRows);
    p.groups = (int)groups_of<T>(p.C);
    hipLaunchKernelGGL((expand_kernel<T>), dim3((unsigned)(sh.tiles(kExpandRows) * p.groups)), dim3(256), 0, s, p);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

template <typename T> bool grids_ok(const Shape &sh, int64_t C, int64_t R) {
    if (R > 0 && R <= kFusedRank) return sh.tiles(adapt_rows(sh, R, sizeof(T))) < (1 << 22);
    return sh.tiles(shrink_rows_of(sh)) < (1 << 23) && sh.tiles(kExpandRows) * groups_of<T>(C) < (1 << 24);
}

gdn2_status check(const gdn2_low_rank_args *a, const std::string &who) {
    if (!a) return fail(GDN2_EINVAL, who + "null args");
    if (a->batch < 0 || a->seq_len < 0 || a->in_features < 0 || a->out_features < 0 || a->rank < 0 || a->num_adapters < 0)
        return fail(GDN2_EINVAL, who + "negative dimension");
    if (a->cu_seqlens && (a->batch != 1 || a->num_seqs < 0))
        return fail(GDN2_EINVAL, who + "packed requests need a batch of 1");
    for (const int64_t stride : {a->stride_x_b, a->stride_x_t, a->stride_y_b, a->stride_y_t, a->stride_out_b, a->stride_out_t,
                                 a->stride_a_l, a->stride_a_r, a->stride_b_l, a->stride_b_r})
        if (stride < 0) return fail(GDN2_EINVAL, who + "negative stride");
    for (const int64_t stride : {a->stride_x_t, a->stride_y_t, a->stride_out_t, a->stride_a_r, a->stride_b_r})
        if (stride >= (1 << 24)) return fail(GDN2_NOT_APPLICABLE, who + "rows too far apart");
    if (!sizes_ok(*a)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    return GDN2_OK;
}
bool workspace_ok(const void *p, size_t have, size_t need) {
    return !need || (p && have >= need && reinterpret_cast<uintptr_t>(p) % 256 == 0);
}

template <typename T> gdn2_status forward(const gdn2_low_rank_args *a, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    gdn2_status st = check(a, who);
    if (st != GDN2_OK) return st;
    const Shape sh = shape_of(*a);
    if (sh.M == 0) return GDN2_OK;
    if (a->out_features == 0 && !a->hidden) return GDN2_OK;
    const int64_t D = a->in_features, O = a->out_features, R = a->rank;
    if ((D > 0 && R > 0 && a->num_adapters > 0 && (!a->x || !a->a)) || (O > 0 && (!a->y || !a->out || (R > 0 && a->num_adapters > 0 && !a->b))) ||
        (sh.N > 0 && !a->adapters))
        return fail(GDN2_EINVAL, who + "null pointer");
    if (O > 0 && a->out == a->y && ((a->batch > 1 && a->stride_out_b != a->stride_y_b) || (a->seq_len > 1 && a->stride_out_t != a->stride_y_t)))
        return fail(GDN2_EINVAL, who + "in place, the strides must be equal");
    if (!grids_ok<T>(sh, O, R)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    if (R > 0 && R <= kFusedRank) {
        AdaptParams p{};
        p.x = a->x; p.w1 = a->a; p.w2 = a->b; p.y = a->y; p.out = O > 0 ? a->out : nullptr; p.scale = a->scale; p.hidden = a->hidden;
        p.xb = a->stride_x_b; p.xt = a->stride_x_t; p.w1l = a->stride_a_l; p.w1r = a->stride_a_r;
        p.w2l = a->stride_b_l; p.w2r = a->stride_b_r; p.yb = a->stride_y_b; p.yt = a->stride_y_t;
        p.ob = a->stride_out_b; p.ot = a->stride_out_t; p.pitch = R;
        p.K = D; p.C = O; p.R = (int)R;
        p.copies = a->out != a->y;
        return launch_adapt<T>(p, *a, sh, s);
    }
    if (!workspace_ok(a->workspace, a->workspace_bytes, R > 0 ? hidden_bytes(sh, R) : 0))
        return fail(GDN2_EINVAL, who + "workspace missing, too small or not 256-byte aligned");
    float *h = static_cast<float *>(a->workspace);
    const int P = (int)pitch_of(R);
    if (R > 0) {
        ShrinkParams p{};
        p.x = a->x; p.w = a->a; p.h = h;
        p.xb = a->stride_x_b; p.xt = a->stride_x_t; p.wl = a->stride_a_l; p.wr = a->stride_a_r;
        p.K = D; p.R = (int)R; p.P = P;
        if ((st = launch_shrink<T>(p, *a, sh, s)) != GDN2_OK) return st;
    }
    ExpandParams p{};
    p.h = h; p.w = a->b; p.y = a->y; p.out = a->out; p.scale = a->scale; p.hidden = R > 0 ? a->hidden : nullptr;
    p.wl = a->stride_b_l; p.wr = a->stride_b_r; p.yb = a->stride_y_b; p.yt = a->stride_y_t;
    p.ob = a->stride_out_b; p.ot = a->stride_out_t;
    p.C = O; p.R = (int)R; p.P = P;
    p.copies = a->out != a->y;
    return launch_expand<T>(p, *a, sh, s);
}

struct BwdPlan {
    int rows;
    int64_t blocks;
    size_t h, ids, part[2], bytes;
};
template <typename T> BwdPlan bwd_plan(const gdn2_low_rank_bwd_args &b) {
    const gdn2_low_rank_args &a = b.fwd;
    const Shape sh = shape_of(a);
    BwdPlan p{};
    const int64_t C[2] = {b.da ? a.in_features : 0, b.db ? a.out_features : 0};
    p.rows = block_rows(sh, C[0] + C[1], 16 * Mm<T>::VC);
    p.blocks = sh.tiles(p.rows);
    p.h = hidden_bytes(sh, a.rank);
    p.ids = align256(sizeof(int) * (size_t)p.blocks);
    for (int i = 0; i < 2; ++i) p.part[i] = align256(sizeof(float) * (size_t)p.blocks * (size_t)a.rank * (size_t)C[i]);
    p.bytes = p.h + p.ids + p.part[0] + p.part[1];
    return p;
}

template <typename T> gdn2_status backward(const gdn2_low_rank_bwd_args *b, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    const gdn2_low_rank_args *a = b ? &b->fwd : nullptr;
    gdn2_status st = check(a, who);
    if (st != GDN2_OK) return st;
    if (b->stride_d_out_b < 0 || b->stride_d_out_t < 0 || b->stride_dx_b < 0 || b->stride_dx_t < 0)
        return fail(GDN2_EINVAL, who + "negative stride");
    if (b->stride_d_out_t >= (1 << 24) || b->stride_dx_t >= (1 << 24)) return fail(GDN2_NOT_APPLICABLE, who + "rows too far apart");
    const Shape sh = shape_of(*a);
    const int64_t D = a->in_features, O = a->out_features, R = a->rank, L = a->num_adapters;
    const BwdPlan p = bwd_plan<T>(*b);
    if (!grids_ok<T>(sh, D, R) || p.blocks * (up(D, 16 * Mm<T>::VC) + up(O, 16 * Mm<T>::VC)) >= (1 << 24))
        return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    SumsParams t{};
    t.n[0] = b->da ? R * D : 0;
    t.n[1] = b->db ? R * O : 0;
    for (int i = 0; i < 2; ++i) t.tiles[i] = (int)up(t.n[i], 256);
    t.out[0] = b->da; t.out[1] = b->db; t.scale = a->scale;
    if (L * (t.tiles[0] + t.tiles[1]) >= (1 << 24)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    if (sh.M > 0) {
        const bool some = R > 0 && L > 0;
        if ((sh.N > 0 && !a->adapters) || (O > 0 && some && (!b->d_out || !a->b)) || (D > 0 && some && b->dx && !a->a) ||
            (D > 0 && some && b->da && !a->x) || (O > 0 && some && b->db && !a->hidden))
            return fail(GDN2_EINVAL, who + "null pointer");
        if (R > 0 && !workspace_ok(b->workspace, b->workspace_bytes, p.bytes))
            return fail(GDN2_EINVAL, who + "workspace missing, too small or not 256-byte aligned");
        char *ws = static_cast<char *>(b->workspace);
        float *dh = reinterpret_cast<float *>(ws);
        ws += p.h;
        int *ids = reinterpret_cast<int *>(ws);
        ws += p.ids;
        const int P = (int)pitch_of(R);
        if (R > 0 && R <= kFusedRank) {
            AdaptParams k{};
            k.x = b->d_out; k.w1 = a->b; k.w2 = a->a; k.y = b->accumulate_dx ? b->dx : nullptr; k.out = D > 0 ? b->dx : nullptr;
            k.scale = a->scale; k.hidden = b->da ? dh : nullptr; k.scale_hidden = 1;
            k.xb = b->stride_d_out_b; k.xt = b->stride_d_out_t; k.w1l = a->stride_b_l; k.w1r = a->stride_b_r;
            k.w2l = a->stride_a_l; k.w2r = a->stride_a_r; k.yb = k.ob = b->stride_dx_b; k.yt = k.ot = b->stride_dx_t; k.pitch = P;
            k.K = O; k.C = D; k.R = (int)R;
            k.copies = !b->accumulate_dx;
            if ((k.out || k.hidden) && (st = launch_adapt<T>(k, *a, sh, s)) != GDN2_OK) return st;
        }
        if (R > kFusedRank && (b->dx || b->da)) {
            ShrinkParams k{};
            k.x = b->d_out; k.w = a->b; k.scale = a->scale; k.h = dh;
            k.xb = b->stride_d_out_b; k.xt = b->stride_d_out_t; k.wl = a->stride_b_l; k.wr = a->stride_b_r;
            k.K = O; k.R = (int)R; k.P = P;
            if ((st = launch_shrink<T>(k, *a, sh, s)) != GDN2_OK) return st;
        }
        if ((R > kFusedRank || R == 0) && b->dx && D > 0) {
            ExpandParams k{};
            k.h = dh; k.w = a->a; k.y = b->accumulate_dx ? b->dx : nullptr; k.out = b->dx;
            k.wl = a->stride_a_l; k.wr = a->stride_a_r;
            k.yb = k.ob = b->stride_dx_b; k.yt = k.ot = b->stride_dx_t;
            k.C = D; k.R = (int)R; k.P = P;
            k.copies = !b->accumulate_dx;
            if ((st = launch_expand<T>(k, *a, sh, s)) != GDN2_OK) return st;
        }
        if (R > 0 && (b->da || b->db)) {
            OuterParams k{};
            k.req = requests_of(*a, sh, p.rows);
            k.z[0] = a->x; k.z[1] = b->d_out;
            k.h[0] = dh; k.h[1] = a->hidden; k.pitch[0] = P; k.pitch[1] = R;
            k.part[0] = reinterpret_cast<float *>(ws); k.part[1] = reinterpret_cast<float *>(ws + p.part[0]);
            k.zb[0] = a->stride_x_b; k.zt[0] = a->stride_x_t; k.zb[1] = b->stride_d_out_b; k.zt[1] = b->stride_d_out_t;
            k.C[0] = b->da ? D : 0; k.C[1] = b->db ? O : 0;
            for (int i = 0; i < 2; ++i) k.tiles[i] = (int)up(k.C[i], 16 * Mm<T>::VC);
            k.adapter = ids; k.R = (int)R; k.rows = p.rows;
            // (more than 32 ranks: two waves' shares, for the registers)
            const dim3 grid((unsigned)(p.blocks * (k.tiles[0] + k.tiles[1])), (unsigned)up(R, 64));
            if (grid.x > 0) {
                if (R <= 16) hipLaunchKernelGGL((outer_kernel<T, 1, 1>), grid, dim3(256), 0, s, k);
                else if (R <= 32) hipLaunchKernelGGL((outer_kernel<T, 2, 1>), grid, dim3(256), 0, s, k);
                else hipLaunchKernelGGL((outer_kernel<T, 2, 2>), grid, dim3(256), 0, s, k);
            }
            t.part[0] = k.part[0]; t.part[1] = k.part[1];
            t.adapter = ids; t.blocks = (int)p.blocks;
        }
    }
    if (L * (t.tiles[0] + t.tiles[1]) > 0)
        hipLaunchKernelGGL(adapter_sums_kernel, dim3((unsigned)(L * (t.tiles[0] + t.tiles[1]))), dim3(256), 0, s, t);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

bool countable(const gdn2_low_rank_args &a) {
    return a.batch > 0 && a.seq_len > 0 && a.in_features >= 0 && a.out_features >= 0 && a.rank > 0 && a.num_adapters >= 0 &&
           a.num_seqs >= 0 && sizes_ok(a);
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_low_rank_add_workspace_bytes(const gdn2_low_rank_args *a) {
    return a && gdn2::countable(*a) && a->rank > gdn2::kFusedRank ? gdn2::hidden_bytes(gdn2::shape_of(*a), a->rank) : 0;
}
// (the larger of the two types')
extern "C" size_t gdn2_low_rank_add_bwd_workspace_bytes(const gdn2_low_rank_bwd_args *b) {
    if (!b || !gdn2::countable(b->fwd)) return 0;
    return std::max(gdn2::bwd_plan<float>(*b).bytes, gdn2::bwd_plan<gdn2::bf16>(*b).bytes);
}

#define GDN2_ENTRY(suffix, T)                                                                                      \
    extern "C" gdn2_status gdn2_low_rank_add_##suffix(const gdn2_low_rank_args *args, gdn2_stream_t stream) {      \
        try { /* no exception leaves a C entry */                                                                  \
            return gdn2::forward<T>(args, (hipStream_t)stream, "gdn2_low_rank_add_" #suffix);                      \
        } catch (const std::exception &) {                                                                         \
            return GDN2_EHIP;                                                                                      \
        }                                                                                                          \
    }                                                                                                              \
    extern "C" gdn2_status gdn2_low_rank_add_bwd_##suffix(const gdn2_low_rank_bwd_args *args, gdn2_stream_t stream) { \
        try {                                                                                                      \
            return gdn2::backward<T>(args, (hipStream_t)stream, "gdn2_low_rank_add_bwd_" #suffix);                 \
        } catch (const std::exception &) {                                                                         \
            return GDN2_EHIP;                                                                                      \
        }                                                                                                          \
    }
GDN2_ENTRY(f32, float)
GDN2_ENTRY(bf16, gdn2::bf16)
