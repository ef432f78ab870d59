// gdn2_low_rank_add_*: low-rank adapters of many requests beside a shared projection,
// and their adjoint.  For a row x of a request with adapter l:
//   h = x a_l^T (a [L, R, D]),  out = y + s_l h b_l (b [L, R, O])
//   dh = s_l dy b_l^T,  dx = dh a_l,  da_l = sum dh^T x,  db_l = s_l sum h^T dy
//
// Four kernels, each of which streams one wide tensor past matrix instructions:
//   shrink  h or dh: rows of 16 MT by all ranks, the wide dimension split over the waves
//           of a workgroup and over KS workgroups
//   expand  out or dx: rows of 16 MT by 16 VC columns a wave, y read and out written once
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
// Operands.  A lane holds KV neighbouring k of a row of a (or of x in shrink): one load.
// Where the sum runs over the rows instead, it loads 16 bytes of VC columns from each of
// KV rows and turns them in registers (32 byte permutations for 64 values), so nothing
// goes through LDS; a lane's column tiles are then its VC neighbouring columns, so that
// results leave in 16 bytes, 16 lanes side by side.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2_block.h"
#include "loose_io.hpp"

namespace gdn2 {
namespace {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

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
struct Tile {
    int64_t b, t0, row; // batch entry, first token, its place among all rows
    int rows;           // <= 0: none
    int adapter;        // -1: none
};

// Row 0, the offsets, the end of the rows: requests 1 .. N between rows of none.
__device__ __forceinline__ int64_t bound_at(const Requests &r, int n) {
    if (n == 0) return 0;
    if (n == r.N + 2) return r.M;
    return min(max((int64_t)r.cu[n - 1], (int64_t)0), r.M);
}

// Of the wave's tile w (the same for every lane) of up to `size` rows.
__device__ __forceinline__ Tile tile_at(const Requests &r, int w, int size) {
    Tile t{};
    t.adapter = -1;
    int n;
    if (!r.cu) {
        n = w / r.per;
        t.b = n;
        t.t0 = (int64_t)(w - n * r.per) * size;
        t.row = n * r.T + t.t0;
        t.rows = (int)min((int64_t)size, r.T - t.t0);
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
        const int64_t first = bound_at(r, n);
        t.t0 = first + (w - (first / size + n)) * (int64_t)size;
        t.row = t.t0;
        t.rows = (int)max((int64_t)0, min((int64_t)size, bound_at(r, n + 1) - t.t0));
        if (t.t0 < 0) t.rows = 0; // (offsets that decrease)
        if (n == 0 || n == r.N + 1) return t;
        --n;
    }
    const int id = r.adapters[n];
    if (id >= 0 && id < r.L) t.adapter = id;
    return t;
}

// -- shrink ----------------------------------------------------------------------------

struct ShrinkParams {
    Requests req;
    const void *x, *w; // [.., K]; [L, R, K]
    const float *scale;
    float *h; // [KS][M][R]
    int64_t xb, xt, wl, wr;
    int64_t K;
    int R, KS;
};

template <typename T, int MT, int NR> __global__ __launch_bounds__(256) void shrink_kernel(ShrinkParams p) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, STEP = 4 * KV, CHUNK = 4 * STEP;
    __shared__ floatx4 red[2][MT * NR][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x / p.KS, ks = blockIdx.x - tile * p.KS, r0 = blockIdx.y * NR * 16;
    const Tile at = tile_at(p.req, tile, MT * 16);
    if (at.rows <= 0) return;
    floatx4 acc[MT][NR];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (at.adapter >= 0) {
        // (rows behind the tile's last, ranks behind the last: the last one's again, not stored)
        const T *x[MT], *w[NR];
#pragma unroll
        for (int m = 0; m < MT; ++m)
            x[m] = static_cast<const T *>(p.x) + at.b * p.xb + (at.t0 + min(16 * m + i, at.rows - 1)) * p.xt + KV * g;
#pragma unroll
        for (int n = 0; n < NR; ++n)
            w[n] = static_cast<const T *>(p.w) + at.adapter * p.wl + min(r0 + 16 * n + i, p.R - 1) * p.wr + KV * g;
        for (int64_t k0 = (int64_t)(ks * 4 + wave) * CHUNK; k0 < p.K; k0 += (int64_t)p.KS * 4 * CHUNK) {
            if (k0 + CHUNK <= p.K) {
                typename X::Op a[4][MT], b[4][NR];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) a[s][m] = loose<T, KV>(x[m] + k0 + s * STEP);
#pragma unroll
                    for (int n = 0; n < NR; ++n) b[s][n] = loose<T, KV>(w[n] + k0 + s * STEP);
                }
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int n = 0; n < NR; ++n) acc[m][n] = X::mma(a[s][m], b[s][n], acc[m][n]);
            } else {
                for (int64_t k = k0; k < p.K; k += STEP) {
                    const int64_t left = p.K - k - KV * g;
                    typename X::Op a[MT], b[NR];
#pragma unroll
                    for (int m = 0; m < MT; ++m) a[m] = loose_part<T, KV>(x[m] + k, left);
#pragma unroll
                    for (int n = 0; n < NR; ++n) b[n] = loose_part<T, KV>(w[n] + k, left);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int n = 0; n < NR; ++n) acc[m][n] = X::mma(a[m], b[n], acc[m][n]);
                }
            }
        }
    }
    // the four waves' sums: 0 + 2 and 1 + 3, then those two
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NR; ++n) red[wave - half][m * NR + n][lane] = acc[m][n];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NR; ++n) acc[m][n] += red[wave][m * NR + n][lane];
        __syncthreads();
    }
    if (wave) return;
    const float s = p.scale && at.adapter >= 0 ? p.scale[at.adapter] : 1.f;
    float *h = p.h + ((int64_t)ks * p.req.M + at.row) * p.R;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * m + 4 * g + q, r = r0 + 16 * n + i;
                if (row < at.rows && r < p.R) h[(int64_t)row * p.R + r] = s * acc[m][n][q];
            }
}

// -- expand ----------------------------------------------------------------------------

struct ExpandParams {
    Requests req;
    const float *h; // [KS][M][R]
    const void *w;  // [L, R, C]
    const void *y;  // or NULL
    void *out;      // or NULL
    const float *scale;
    float *hidden; // the sum over KS, or NULL
    int64_t wl, wr, yb, yt, ob, ot;
    int64_t C;
    int R, KS, groups; // workgroups over the columns
    int copies; // rows without an adapter are written too (out is not y's memory)
};

template <typename T, int MT> __global__ __launch_bounds__(256) void expand_kernel(ExpandParams p) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, VC = X::VC, STEP = 4 * KV;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x / p.groups, group = blockIdx.x - tile * p.groups;
    const int64_t c0 = (int64_t)(group * 4 + wave) * 16 * VC;
    if (c0 >= p.C) return;
    const Tile at = tile_at(p.req, tile, MT * 16);
    if (at.rows <= 0) return;
    const int64_t c = c0 + VC * i, left = p.C - c;
    const bool keep = p.hidden && group == 0 && wave == 0, write = p.out && (at.adapter >= 0 || p.copies);
    if (!keep && !write) return;
    const T *y = p.y ? static_cast<const T *>(p.y) + at.b * p.yb + at.t0 * p.yt + c : nullptr;
    Raw<T, VC> old[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int t = 0; t < VC; ++t) old[m][q][t] = (T)0.f;
            const int row = 16 * m + 4 * g + q;
            if (y && row < at.rows) old[m][q] = loose_part<T, VC>(y + row * p.yt, left);
        }
    floatx4 acc[MT][VC];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < VC; ++t) acc[m][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    float s = 1.f;
    if (at.adapter >= 0) {
        if (p.scale) s = p.scale[at.adapter];
        const T *w = static_cast<const T *>(p.w) + at.adapter * p.wl + c;
        for (int r0 = 0; r0 < p.R; r0 += STEP) {
            const int r = r0 + KV * g;
            Raw<T, VC> rows[KV];
#pragma unroll
            for (int k = 0; k < KV; ++k) rows[k] = loose_part<T, VC>(w + (int64_t)min(r + k, p.R - 1) * p.wr, r + k < p.R ? left : 0);
            typename X::Op cols[VC];
            X::turn(rows, cols);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int64_t place = (at.row + min(16 * m + i, at.rows - 1)) * p.R + r;
                float h[KV];
                load_part<float, KV>(p.h + place, p.R - r, h);
                for (int k = 1; k < p.KS; ++k) {
                    float more[KV];
                    load_part<float, KV>(p.h + k * p.req.M * p.R + place, p.R - r, more);
#pragma unroll
                    for (int j = 0; j < KV; ++j) h[j] += more[j];
                }
                if (keep && 16 * m + i < at.rows) store_part<float, KV>(p.hidden + place, p.R - r, h);
                const typename X::Wide hw = X::wide(h);
#pragma unroll
                for (int t = 0; t < VC; ++t) acc[m][t] = X::mmw(hw, cols[t], acc[m][t]);
            }
        }
    } else if (keep) {
        for (int64_t k = lane; k < (int64_t)at.rows * p.R; k += kWave) p.hidden[at.row * p.R + k] = 0.f;
    }
    if (!write) return;
    T *out = static_cast<T *>(p.out) + at.b * p.ob + at.t0 * p.ot + c;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = 16 * m + 4 * g + q;
            if (row >= at.rows) continue;
            float v[VC];
#pragma unroll
            for (int t = 0; t < VC; ++t) // (rows without an adapter: as they are, NaN and all)
                v[t] = at.adapter >= 0 ? __builtin_fmaf(s, acc[m][t][q], (float)old[m][q][t]) : (float)old[m][q][t];
            store_part<T, VC>(out + row * p.ot, left, v);
        }
}

// -- outer -----------------------------------------------------------------------------

struct OuterParams {
    Requests req;
    const void *z[2];  // x with dh for da, dy with h for db
    const float *h[2]; // [M][R]
    float *part[2];    // [blocks][R][C]
    int64_t zb[2], zt[2], C[2];
    int tiles[2]; // column tiles
    int *adapter; // of each block
    int R, rows;  // rows a block
};

template <typename T, int NR> __global__ __launch_bounds__(256) void outer_kernel(OuterParams p) {
    typedef Mm<T> X;
    constexpr int KV = X::KV, VC = X::VC, STEP = 4 * KV;
    __shared__ floatx4 red[2][NR * VC][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int tiles = p.tiles[0] + p.tiles[1], block = blockIdx.x / tiles, ct = blockIdx.x - block * tiles;
    const int which = ct >= p.tiles[0], r0 = blockIdx.y * NR * 16;
    const Tile at = tile_at(p.req, block, p.rows);
    const bool any = at.rows > 0 && at.adapter >= 0;
    if (ct == 0 && r0 == 0 && threadIdx.x == 0) p.adapter[block] = any ? at.adapter : -1;
    if (!any) return;
    const int64_t C = p.C[which], c = (int64_t)(ct - which * p.tiles[0]) * 16 * VC + VC * i, left = C - c;
    const T *z = static_cast<const T *>(p.z[which]) + at.b * p.zb[which] + at.t0 * p.zt[which] + c;
    const int64_t zt = p.zt[which];
    const float *h = p.h[which] + at.row * p.R;
    floatx4 acc[NR][VC];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int t = 0; t < VC; ++t) acc[n][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    Raw<T, VC> rows[KV];
    float hv[NR][KV];
    auto load = [&](int m0) { // rows behind the last, ranks behind the last: zeros
        const int m = m0 + KV * g;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int row = min(m + k, at.rows - 1);
            rows[k] = loose_part<T, VC>(z + row * zt, m + k < at.rows ? left : 0);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int r = r0 + 16 * n + i;
                const float v = h[(int64_t)row * p.R + min(r, p.R - 1)];
                hv[n][k] = m + k < at.rows ? v : 0.f;
            }
        }
    };
    if (wave * STEP < at.rows) load(wave * STEP);
    for (int m0 = wave * STEP; m0 < at.rows; m0 += 4 * STEP) {
        typename X::Op cols[VC];
        X::turn(rows, cols);
        typename X::Wide hw[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) hw[n] = X::wide(hv[n]);
        if (m0 + 4 * STEP < at.rows) load(m0 + 4 * STEP);
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int t = 0; t < VC; ++t) acc[n][t] = X::mmw(hw[n], cols[t], acc[n][t]);
    }
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int t = 0; t < VC; ++t) red[wave - half][n * VC + t][lane] = acc[n][t];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int t = 0; t < VC; ++t) acc[n][t] += red[wave][n * VC + t][lane];
        __syncthreads();
    }
    if (wave) return;
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
            store_part<float, VC>(part + r * C, left, v);
        }
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

__global__ __launch_bounds__(256) void adapter_sums_kernel(SumsParams p) {
    const int tiles = p.tiles[0] + p.tiles[1], l = blockIdx.x / tiles, ct = blockIdx.x - l * tiles;
    const int which = ct >= p.tiles[0];
    const int64_t n = p.n[which], e = ((int64_t)(ct - which * p.tiles[0]) * 256 + threadIdx.x) * 4;
    const int64_t left = n - e;
    double sum[4] = {0., 0., 0., 0.};
    bool some = false;
    for (int b0 = 0; b0 < p.blocks; b0 += kWave) {
        const int b = b0 + (int)(threadIdx.x & 63);
        uint64_t mine = __ballot(b < p.blocks && p.adapter[b < p.blocks ? b : 0] == l);
        while (mine) {
            const int at = b0 + __builtin_ctzll(mine);
            mine &= mine - 1;
            some = true;
            float v[4];
            load_part<float, 4>(p.part[which] + at * n + e, left, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += v[j];
        }
    }
    if (left <= 0) return;
    const double s = which && some && p.scale ? p.scale[l] : 1.;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)(s * sum[j]);
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

// Row tiles of 16 mt: the larger, the fewer times an adapter is read from the caches;
// but no more than a request has, and while 128 tiles remain.
int mt_of(const Shape &s) {
    const int64_t mean = s.N > 0 ? up(s.M, s.N) : 1;
    if (mean > 32 && s.tiles(64) >= 128) return 4;
    return 1;
}
// Workgroups that share the wide dimension: while fewer than 512, and each wave has a
// chunk of 128 (f32: 64).
int ks_of(int64_t tiles, int64_t K, int element) {
    const int64_t most = std::max<int64_t>(1, K / (4 * (element == 2 ? 128 : 64)));
    int ks = 1;
    while (ks < 8 && 2 * ks <= most && tiles * ks < 512) ks *= 2;
    return ks;
}
int nr_of(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : 4; }

// Rows a block of the outer products: 1024 blocks by columns, while each has 128 rows or
// more and at most 4096.
int block_rows(const Shape &s, int64_t columns, int tile_columns) {
    const int64_t per = up(columns, tile_columns);
    int rows = 4096;
    while (rows > 128 && s.tiles(rows) * per < 1024) rows /= 2;
    return rows;
}

bool sizes_ok(const gdn2_low_rank_args &a) {
    const double M = (double)a.batch * (double)a.seq_len;
    return M < 1073741824. && a.batch < (1 << 30) && a.seq_len < (1 << 30) && a.num_seqs < (1 << 24) && a.rank <= kMostRank &&
           a.in_features < (1 << 24) && a.out_features < (1 << 24) && a.num_adapters < (1 << 24);
}

// Bytes of a forward's workspace: h of each share of the wide dimension.
size_t hidden_bytes(const Shape &s, int64_t R, int ks) { return align256(sizeof(float) * (size_t)ks * (size_t)s.M * (size_t)R); }

struct Plan {
    int mt, ks;
    int64_t tiles, groups;
};
template <typename T> Plan plan_of(const Shape &s, int64_t K, int64_t C) {
    Plan q{};
    q.mt = mt_of(s);
    q.tiles = s.tiles(16 * q.mt);
    q.ks = C > 0 ? ks_of(q.tiles, K, sizeof(T)) : 1; // (expand joins the shares)
    q.groups = up(C, 4 * 16 * Mm<T>::VC);
    return q;
}

template <typename T> gdn2_status launch_shrink(const ShrinkParams &p, const Plan &q, hipStream_t s) {
    const int nr = nr_of(p.R);
    const dim3 grid((unsigned)(q.tiles * q.ks), (unsigned)up(p.R, 16 * nr));
#define GDN2_RUN(MT, NR) hipLaunchKernelGGL((shrink_kernel<T, MT, NR>), grid, dim3(256), 0, s, p)
    if (q.mt == 4) {
        if (nr == 1) GDN2_RUN(4, 1);
        else if (nr == 2) GDN2_RUN(4, 2);
        else GDN2_RUN(4, 4);
    } else {
        if (nr == 1) GDN2_RUN(1, 1);
        else if (nr == 2) GDN2_RUN(1, 2);
        else GDN2_RUN(1, 4);
    }
#undef GDN2_RUN
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

template <typename T> gdn2_status launch_expand(const ExpandParams &p, const Plan &q, hipStream_t s) {
    const dim3 grid((unsigned)(q.tiles * q.groups));
    if (q.mt == 4) hipLaunchKernelGGL((expand_kernel<T, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((expand_kernel<T, 1>), grid, dim3(256), 0, s, p);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

gdn2_status check(const gdn2_low_rank_args *a, const std::string &who) {
    if (!a) return fail(GDN2_EINVAL, who + "null args");
    if (a->batch < 0 || a->seq_len < 0 || a->in_features < 0 || a->out_features < 0 || a->rank < 0 || a->num_adapters < 0)
        return fail(GDN2_EINVAL, who + "negative dimension");
    if (a->cu_seqlens && (a->batch != 1 || a->num_seqs < 0))
        return fail(GDN2_EINVAL, who + "packed requests need a batch of 1");
    if (!sizes_ok(*a)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    return GDN2_OK;
}
bool workspace_ok(const void *p, size_t have, size_t need) {
    return !need || (p && have >= need && reinterpret_cast<uintptr_t>(p) % 256 == 0);
}
bool grid_ok(const Plan &q) { return q.tiles * std::max<int64_t>(q.groups, q.ks) < (1 << 24); }

template <typename T> gdn2_status forward(const gdn2_low_rank_args *a, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    gdn2_status st = check(a, who);
    if (st != GDN2_OK) return st;
    const Shape sh = shape_of(*a);
    if (sh.M == 0) return GDN2_OK;
    const int64_t D = a->in_features, O = a->out_features, R = a->rank;
    if ((D > 0 && R > 0 && a->num_adapters > 0 && (!a->x || !a->a)) || (O > 0 && (!a->y || !a->out || (R > 0 && a->num_adapters > 0 && !a->b))) ||
        (sh.N > 0 && !a->adapters))
        return fail(GDN2_EINVAL, who + "null pointer");
    if (O > 0 && a->out == a->y && ((a->batch > 1 && a->stride_out_b != a->stride_y_b) || (a->seq_len > 1 && a->stride_out_t != a->stride_y_t)))
        return fail(GDN2_EINVAL, who + "in place, the strides must be equal");
    if (O == 0 && !a->hidden) return GDN2_OK;
    const Plan q = plan_of<T>(sh, D, O);
    if (!grid_ok(q)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    const bool direct = q.ks == 1 && a->hidden; // h needs no joining
    const size_t need = R > 0 && !direct ? hidden_bytes(sh, R, q.ks) : 0;
    if (!workspace_ok(a->workspace, a->workspace_bytes, need))
        return fail(GDN2_EINVAL, who + "workspace missing, too small or not 256-byte aligned");
    float *h = direct ? a->hidden : static_cast<float *>(a->workspace);
    const Requests req = requests_of(*a, sh, 16 * q.mt);
    if (R > 0) {
        ShrinkParams p{};
        p.req = req;
        p.x = a->x; p.w = a->a; p.h = h;
        p.xb = a->stride_x_b; p.xt = a->stride_x_t; p.wl = a->stride_a_l; p.wr = a->stride_a_r;
        p.K = D; p.R = (int)R; p.KS = q.ks;
        if ((st = launch_shrink<T>(p, q, s)) != GDN2_OK) return st;
    }
    if (O == 0) return GDN2_OK;
    ExpandParams p{};
    p.req = req;
    p.h = h; p.w = a->b; p.y = a->y; p.out = a->out; p.scale = a->scale; p.hidden = direct || R == 0 ? nullptr : a->hidden;
    p.wl = a->stride_b_l; p.wr = a->stride_b_r; p.yb = a->stride_y_b; p.yt = a->stride_y_t;
    p.ob = a->stride_out_b; p.ot = a->stride_out_t;
    p.C = O; p.R = (int)R; p.KS = q.ks; p.groups = (int)q.groups;
    p.copies = a->out != a->y;
    return launch_expand<T>(p, q, s);
}

struct BwdPlan {
    Plan q;
    int rows;
    int64_t blocks;
    size_t h, one, ids, part[2], bytes;
};
template <typename T> BwdPlan bwd_plan(const gdn2_low_rank_bwd_args &b) {
    const gdn2_low_rank_args &a = b.fwd;
    const Shape sh = shape_of(a);
    BwdPlan p{};
    p.q = plan_of<T>(sh, a.out_features, a.in_features);
    const int64_t C[2] = {b.da ? a.in_features : 0, b.db ? a.out_features : 0};
    p.rows = block_rows(sh, C[0] + C[1], 16 * Mm<T>::VC);
    p.blocks = sh.tiles(p.rows);
    p.h = hidden_bytes(sh, a.rank, p.q.ks);
    p.one = p.q.ks > 1 ? hidden_bytes(sh, a.rank, 1) : 0;
    p.ids = align256(sizeof(int) * (size_t)p.blocks);
    for (int i = 0; i < 2; ++i) p.part[i] = align256(sizeof(float) * (size_t)p.blocks * (size_t)a.rank * (size_t)C[i]);
    p.bytes = p.h + p.one + p.ids + p.part[0] + p.part[1];
    return p;
}

template <typename T> gdn2_status backward(const gdn2_low_rank_bwd_args *b, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    const gdn2_low_rank_args *a = b ? &b->fwd : nullptr;
    gdn2_status st = check(a, who);
    if (st != GDN2_OK) return st;
    const Shape sh = shape_of(*a);
    const int64_t D = a->in_features, O = a->out_features, R = a->rank, L = a->num_adapters;
    const BwdPlan p = bwd_plan<T>(*b);
    if (!grid_ok(p.q) || p.blocks * (up(D, 16 * Mm<T>::VC) + up(O, 16 * Mm<T>::VC)) >= (1 << 24))
        return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    SumsParams t{};
    t.n[0] = b->da ? R * D : 0;
    t.n[1] = b->db ? R * O : 0;
    for (int i = 0; i < 2; ++i) t.tiles[i] = (int)up(t.n[i], 1024);
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
        float *h = reinterpret_cast<float *>(ws);
        float *dh = p.one ? reinterpret_cast<float *>(ws + p.h) : h;
        ws += p.h + p.one;
        int *ids = reinterpret_cast<int *>(ws);
        ws += p.ids;
        const bool want_dh = b->dx || b->da;
        const Requests req = requests_of(*a, sh, 16 * p.q.mt);
        if (R > 0 && want_dh) {
            ShrinkParams k{};
            k.req = req;
            k.x = b->d_out; k.w = a->b; k.scale = a->scale; k.h = h;
            k.xb = b->stride_d_out_b; k.xt = b->stride_d_out_t; k.wl = a->stride_b_l; k.wr = a->stride_b_r;
            k.K = O; k.R = (int)R; k.KS = p.q.ks;
            if ((st = launch_shrink<T>(k, p.q, s)) != GDN2_OK) return st;
        }
        if (want_dh && (b->dx || p.one) && D > 0) {
            ExpandParams k{};
            k.req = req;
            k.h = h; k.w = a->a; k.y = b->accumulate_dx ? b->dx : nullptr; k.out = b->dx;
            k.hidden = p.one && R > 0 ? dh : nullptr;
            k.wl = a->stride_a_l; k.wr = a->stride_a_r;
            k.yb = k.ob = b->stride_dx_b; k.yt = k.ot = b->stride_dx_t;
            k.C = D; k.R = (int)R; k.KS = p.q.ks; k.groups = (int)p.q.groups;
            k.copies = !b->accumulate_dx;
            if ((st = launch_expand<T>(k, p.q, s)) != GDN2_OK) return st;
        }
        if (R > 0 && (b->da || b->db)) {
            OuterParams k{};
            k.req = requests_of(*a, sh, p.rows);
            k.z[0] = a->x; k.z[1] = b->d_out;
            k.h[0] = dh; k.h[1] = a->hidden;
            k.part[0] = reinterpret_cast<float *>(ws); k.part[1] = reinterpret_cast<float *>(ws + p.part[0]);
            k.zb[0] = a->stride_x_b; k.zt[0] = a->stride_x_t; k.zb[1] = b->stride_d_out_b; k.zt[1] = b->stride_d_out_t;
            k.C[0] = b->da ? D : 0; k.C[1] = b->db ? O : 0;
            for (int i = 0; i < 2; ++i) k.tiles[i] = (int)up(k.C[i], 16 * Mm<T>::VC);
            k.adapter = ids; k.R = (int)R; k.rows = p.rows;
            const int nr = nr_of(R);
            const dim3 grid((unsigned)(p.blocks * (k.tiles[0] + k.tiles[1])), (unsigned)up(R, 16 * nr));
            if (grid.x > 0) {
                if (nr == 1) hipLaunchKernelGGL((outer_kernel<T, 1>), grid, dim3(256), 0, s, k);
                else if (nr == 2) hipLaunchKernelGGL((outer_kernel<T, 2>), grid, dim3(256), 0, s, k);
                else hipLaunchKernelGGL((outer_kernel<T, 4>), grid, dim3(256), 0, s, k);
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

// (the larger of the two types')
extern "C" size_t gdn2_low_rank_add_workspace_bytes(const gdn2_low_rank_args *a) {
    if (!a || !gdn2::countable(*a)) return 0;
    const gdn2::Shape s = gdn2::shape_of(*a);
    if (a->out_features == 0 && !a->hidden) return 0;
    const int ks = std::max(gdn2::plan_of<float>(s, a->in_features, a->out_features).ks,
                            gdn2::plan_of<gdn2::bf16>(s, a->in_features, a->out_features).ks);
    return ks == 1 && a->hidden ? 0 : gdn2::hidden_bytes(s, a->rank, ks);
}
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
