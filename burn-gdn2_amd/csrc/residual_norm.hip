// gdn2_residual_norm_*: the residual path between two blocks, and its adjoint.
//   p = y sy post, r = alpha x + sigma drop(act(gate) p), n = r sr pre
//   sy, sr = 1 / sqrt(mean of squares + eps)
// Backward, for the r and statistics that the forward wrote (rn = r sr, yn = y sy):
//   e = dn pre,  dpre = sum dn rn,  d = dr + sr (e - rn mean(e rn)),  dx = alpha d
//   b = sigma drop(d),  dgate = b p act'(gate),  q = b act(gate)
//   dpost = sum q yn,  f = q post,  dy = sy (f - yn mean(f yn))
//
// A row stays in the registers of its lanes, 8 channels a lane (16 above 4096 channels):
// up to 512 channels the 2^log_l lanes of a part of a wave, up to 2048 the four
// waves of a workgroup, up to 8192 eight.  So each operand is read once and each
// result written once, and the two means of a row are sums over its lanes.
//
// Bound: HBM.  Forward: 32768 x 2048 bfloat16 with a gate 124 us, 5.4 TB/s (129 at 4096
// channels, where 16 a lane took 138; 126 at 8192); 8192 x 2048 with an f32 stream and
// dropout 41 to 43 us, 4.8.  Backward: 8192 x 2048 bfloat16 with gate and dropout 53 us
// and 5 for the weights' sums, 4.7 TB/s together; its instructions (generator, gate, two
// norms) take about 35 us of a SIMD, which overlap with the bytes only in part.  Of 4096 channels
// 64 us (16 a lane: 106), of 8192 93.  Rows that are no multiple of 8 bfloat16 (4 f32) go
// by a form with a branch a run, since each row ends in the middle of one: 32768 x 321
// bfloat16 80 us, of 320 57.  (Without branches, a row's last whole run turned to its place:
// 87; its values all loaded first: 88.)
//
// The backward's workgroups walk the rows of one gate row (all rows, or a sample's
// where the gate is a sample's) with their sums for the weights in registers: at most
// kMostRows rows a lane in f32.  Lanes of the same channels are added in f64, by all of the
// workgroup's threads (200000 x 8 f32: 27 us; by the lanes of one row 193), and those of all
// workgroups (rounded to f32 between) by a second kernel, in f64 too.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2_block.h"
#include "loose_io.hpp"
#include "philox.hpp"

namespace gdn2 {
namespace {

constexpr int kMostC = 8192, kMostRows = 128;

struct Rows { // of a tensor [N, S, C]
    int64_t n, s;
};

struct ResParams {
    const void *x, *y, *gate, *dr, *dn;
    const float *post, *pre;
    void *out, *normed; // forward
    void *dx, *dy, *dgate;
    float *stats;
    Rows sx, sy, sgate, sout, snormed;
    Rows sdr, sdn, sdx, sdy, sdgate; // backward
    int64_t M;
    int S, C, act, log_l;
    uint32_t quads; // counters a row
    float inv_c, eps, alpha, sigma; // sigma: with 1 / (1 - p)
    int has_drop;
    int stream; // forward: results too large for the caches
    Drop drop;
    // backward: rows of a gate row, workgroups that share them; what they leave, [workgroup][C] each
    int64_t seg_rows;
    int blocks_a_seg;
    float *part_pre, *part_post, *part_gate;
};

// (v_rcp_f32 is within one unit in the last place)
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z)); }

// 1 / sqrt(v), v >= 0 (v_rsq_f32 takes a subnormal v, which eps = 0 allows, as 0)
__device__ __forceinline__ float rstd_f(float v) {
    const bool tiny = v < 0x1p-126f;
    const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p48f : v);
    return tiny ? r * 0x1p24f : r;
}

// a = act(z), d = act'(z)
__device__ __forceinline__ void gate_of(int act, float z, float &a, float &d) {
    if (act == GDN2_GATE_NONE) {
        a = z;
        d = 1.f;
        return;
    }
    const float s = sigmoid_f(z);
    if (act == GDN2_GATE_SILU) {
        a = z * s;
        d = s * __builtin_fmaf(z, 1.f - s, 1.f);
    } else {
        a = s;
        d = s * (1.f - s);
    }
}

template <int N, bool WHOLE> __device__ __forceinline__ void weights_n(const float *w, int c, int C, float *x) {
    load_part<float, N, WHOLE>(w + c, C - c, x);
}

// Sums over the lanes of a row, to all of them.  WPR waves a row; `turn` alternates
// between two places in LDS, so that one barrier a sum is enough.
template <int WPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int log_l, float (*red)[WPR][N], int &turn) {
    lanes_sum<N>(v, WPR == 1 ? log_l : 6);
    if constexpr (WPR > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[turn][wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = red[turn][0][i];
#pragma unroll
            for (int w = 1; w < WPR; ++w) v[i] += red[turn][w][i];
        }
        turn ^= 1;
    }
}

// The place of a thread: row `local` of those its workgroup holds at once, channels
// from c[k] on.
template <int VEC, int NV, int WPR> struct Place {
    int local, c[NV], rows; // rows a workgroup holds
    __device__ Place(int log_l) {
        int first, l;
        if constexpr (WPR == 1) {
            l = 1 << log_l;
            local = threadIdx.x >> log_l;
            first = threadIdx.x & (l - 1);
            rows = 256 >> log_l;
        } else {
            l = kWave * WPR;
            local = 0;
            first = threadIdx.x;
            rows = 1;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) c[k] = (k * l + first) * VEC;
    }
};

__device__ __forceinline__ int64_t row_at(const Rows &r, int64_t m, int S) {
    const uint32_t n = (uint32_t)m / (uint32_t)S;
    return n * r.n + (int64_t)((uint32_t)m - n * (uint32_t)S) * r.s;
}

// TS, TB: the stream's and the branch's types.  WHOLE: C is a multiple of VEC.
template <typename TS, typename TB, int VEC, int NV, int WPR, bool WHOLE>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void residual_norm_kernel(ResParams p) {
    __shared__ float red[2][WPR][1];
    int turn = 0;
    const Place<VEC, NV, WPR> at(p.log_l);
    if (p.has_drop) drop_begin(p.drop);
    // (one turn but for more rows than a launch takes; the same for every thread: barriers)
    for (int64_t m0 = (int64_t)blockIdx.x * at.rows; m0 < p.M; m0 += (int64_t)gridDim.x * at.rows) {
        const bool ok = m0 + at.local < p.M;
        const int64_t m = ok ? m0 + at.local : p.M - 1;
        Raw<TS, VEC> rx[NV];
        Raw<TB, VEC> ry[NV], rg[NV];
        {
            const TS *x = static_cast<const TS *>(p.x) + row_at(p.sx, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) rx[k] = loose_part<TS, VEC, WHOLE>(x + at.c[k], p.C - at.c[k]);
        }
        if (p.y) {
            const TB *y = static_cast<const TB *>(p.y) + row_at(p.sy, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) ry[k] = loose_part<TB, VEC, WHOLE>(y + at.c[k], p.C - at.c[k]);
            if (p.gate) {
                const TB *g = static_cast<const TB *>(p.gate) + row_at(p.sgate, m, p.S);
#pragma unroll
                for (int k = 0; k < NV; ++k) rg[k] = loose_part<TB, VEC, WHOLE>(g + at.c[k], p.C - at.c[k]);
            }
        }
        float r[NV][VEC], sy = 0.f, sr = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) r[k][j] = p.alpha * (float)rx[k][j];
        if (p.y) {
            if (p.post) {
                float sum[1] = {0.f};
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum[0] = __builtin_fmaf((float)ry[k][j], (float)ry[k][j], sum[0]);
                row_sum<WPR, 1>(sum, p.log_l, red, turn);
                sy = rstd_f(__builtin_fmaf(sum[0], p.inv_c, p.eps));
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float b[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) b[j] = (float)ry[k][j];
                if (p.post) {
                    float w[VEC];
                    weights_n<VEC, WHOLE>(p.post, at.c[k], p.C, w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) b[j] = b[j] * sy * w[j];
                }
                if (p.gate) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float a, d;
                        gate_of(p.act, (float)rg[k][j], a, d);
                        b[j] *= a;
                    }
                }
                if (p.has_drop) {
                    drop_n<VEC>(p.drop, (uint64_t)m * p.quads + at.c[k] / 4, p.sigma, b);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) r[k][j] += b[j];
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) r[k][j] = __builtin_fmaf(p.sigma, b[j], r[k][j]);
                }
            }
        }
        if (p.out && ok) {
            TS *out = static_cast<TS *>(p.out) + row_at(p.sout, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) store_part<TS, VEC, WHOLE>(out + at.c[k], p.C - at.c[k], r[k], p.stream);
        }
        if (p.pre) {
            float sum[1] = {0.f};
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[0] = __builtin_fmaf(r[k][j], r[k][j], sum[0]);
            row_sum<WPR, 1>(sum, p.log_l, red, turn);
            sr = rstd_f(__builtin_fmaf(sum[0], p.inv_c, p.eps));
            TB *normed = static_cast<TB *>(p.normed) + row_at(p.snormed, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float w[VEC];
                weights_n<VEC, WHOLE>(p.pre, at.c[k], p.C, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) r[k][j] = r[k][j] * sr * w[j];
                if (ok) store_part<TB, VEC, WHOLE>(normed + at.c[k], p.C - at.c[k], r[k], p.stream);
            }
        }
        if (p.stats && ok && at.c[0] == 0) {
            p.stats[2 * m] = sy;
            p.stats[2 * m + 1] = sr;
        }
    }
}

// Sums of a workgroup's rows: lanes of the same channels, in a fixed order and f64, to part.
template <int VEC, int NV, int WPR, bool WHOLE> __device__ __forceinline__ void leave_sums(const Place<VEC, NV, WPR> &at, int C, int log_l,
                                                                               float (&v)[NV][VEC], float *part) {
    part += (int64_t)blockIdx.x * C;
    if constexpr (WPR == 1) {
        __shared__ float red[4][NV][kWave][VEC + 1];
        __shared__ double sums[256];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) red[wave][k][lane][j] = v[k][j];
        __syncthreads();
        // a column's 256 / l lanes in as many shares as there are threads for the l N columns
        constexpr int N = NV * VEC;
        const int l = 1 << log_l, columns = l * N, shares = columns < 256 ? 256 / columns : 1;
        for (int o0 = 0; o0 < columns; o0 += 256) {
            const int share = shares > 1 ? threadIdx.x / columns : 0, o = o0 + (int)threadIdx.x - share * columns;
            const int i = o / N, k = o % N / VEC, j = o % VEC, c = (k * l + i) * VEC + j;
            double s = 0.; // (up to 256 lanes of kMostRows rows each)
            for (int q = share; q < 256 >> log_l; q += shares)
                s += red[q >> (6 - log_l)][k][i + ((q & ((kWave >> log_l) - 1)) << log_l)][j];
            if (shares > 1) {
                sums[threadIdx.x] = s;
                __syncthreads();
                if (share) continue;
                for (int h = 1; h < shares; ++h) s += sums[h * columns + o];
            }
            if (c < C) part[c] = (float)s;
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) store_part<float, VEC, WHOLE>(part + at.c[k], C - at.c[k], v[k]);
    }
}

template <typename TS, typename TB, int VEC, int NV, int WPR, bool WHOLE, bool GSUM>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void residual_norm_bwd_kernel(ResParams p) {
    __shared__ float red[2][WPR][1];
    int turn = 0;
    const Place<VEC, NV, WPR> at(p.log_l);
    const int seg = blockIdx.x / p.blocks_a_seg, j0 = blockIdx.x - seg * p.blocks_a_seg;
    const int64_t base = seg * p.seg_rows;
    if (p.has_drop) drop_begin(p.drop);
    float dpre[NV][VEC], dpost[NV][VEC], dgate[GSUM ? NV : 1][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            dpre[k][j] = dpost[k][j] = 0.f;
            if constexpr (GSUM) dgate[k][j] = 0.f;
        }
    float wpre[NV][VEC], wpost[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) wpre[k][j] = wpost[k][j] = 0.f;
        if (p.pre) weights_n<VEC, WHOLE>(p.pre, at.c[k], p.C, wpre[k]);
        if (p.post) weights_n<VEC, WHOLE>(p.post, at.c[k], p.C, wpost[k]);
    }
    // A row's operands, the next one's in flight while this one's are used (8192 x 2048
    // bfloat16, gated, with dropout: 57 us, without 66).
    struct Row {
        Raw<TS, VEC> o[NV], d[NV];
        Raw<TB, VEC> n[NV], y[NV], g[NV];
        float sy, sr;
        int64_t m;
        bool ok;
    };
    auto load = [&](Row &r, int64_t i0) {
        r.ok = i0 + at.local < p.seg_rows;
        r.m = base + (r.ok ? i0 + at.local : p.seg_rows - 1);
        const int64_t out_at = row_at(p.sout, r.m, p.S), dr_at = row_at(p.sdr, r.m, p.S);
        if (p.dr)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                r.d[k] = loose_part<TS, VEC, WHOLE>(static_cast<const TS *>(p.dr) + dr_at + at.c[k], p.C - at.c[k]);
        if (p.pre) {
            const TB *dn = static_cast<const TB *>(p.dn) + row_at(p.sdn, r.m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                r.o[k] = loose_part<TS, VEC, WHOLE>(static_cast<const TS *>(p.out) + out_at + at.c[k], p.C - at.c[k]);
                r.n[k] = loose_part<TB, VEC, WHOLE>(dn + at.c[k], p.C - at.c[k]);
            }
        }
        if (p.post || p.gate) {
            const TB *y = static_cast<const TB *>(p.y) + row_at(p.sy, r.m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) r.y[k] = loose_part<TB, VEC, WHOLE>(y + at.c[k], p.C - at.c[k]);
        }
        if (p.gate) {
            const TB *g = static_cast<const TB *>(p.gate) + row_at(p.sgate, r.m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) r.g[k] = loose_part<TB, VEC, WHOLE>(g + at.c[k], p.C - at.c[k]);
        }
        r.sy = p.post ? p.stats[2 * r.m] : 0.f;
        r.sr = p.pre ? p.stats[2 * r.m + 1] : 0.f;
    };
    const int64_t step = (int64_t)p.blocks_a_seg * at.rows;
    // (16 channels a lane would not have the registers; ragged rows: 16760 x 1001 f32 119 us
    // without it, 180 with it)
    constexpr bool AHEAD = WHOLE && NV * VEC == 8;
    Row next;
    if constexpr (AHEAD) load(next, (int64_t)j0 * at.rows); // (every workgroup has a row)
    // (the trip count is the same for every thread: barriers)
    for (int64_t i0 = (int64_t)j0 * at.rows; i0 < p.seg_rows; i0 += step) {
        Row row;
        if constexpr (AHEAD) {
            row = next;
            if (i0 + step < p.seg_rows) load(next, i0 + step);
        } else {
            load(row, i0);
        }
        const bool ok = row.ok;
        const int64_t m = row.m;
        const float sy = row.sy, sr = row.sr;
        const auto &ro = row.o, &rd = row.d;
        const auto &rn = row.n, &ry = row.y, &rg = row.g;

        float d[NV][VEC];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[k][j] = p.dr ? (float)rd[k][j] : 0.f;
        if (p.pre) {
            float sum[1] = {0.f}, e[NV][VEC];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float dn = (float)rn[k][j], x = (float)ro[k][j] * sr;
                    e[k][j] = dn * wpre[k][j];
                    if (ok) dpre[k][j] = __builtin_fmaf(dn, x, dpre[k][j]);
                    sum[0] = __builtin_fmaf(e[k][j], x, sum[0]);
                }
            }
            row_sum<WPR, 1>(sum, p.log_l, red, turn);
            const float mean = sum[0] * p.inv_c;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    d[k][j] = __builtin_fmaf(sr, e[k][j] - (float)ro[k][j] * sr * mean, d[k][j]);
        }
        if (p.dx && ok) {
            TS *dx = static_cast<TS *>(p.dx) + row_at(p.sdx, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float v[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = p.alpha * d[k][j];
                store_part<TS, VEC, WHOLE>(dx + at.c[k], p.C - at.c[k], v);
            }
        }
        if (!p.dy) continue;
        TB *dgate_to = static_cast<TB *>(p.dgate) + row_at(p.sdgate, m, p.S);
        float sum[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) { // d becomes b, then q, then f
            if (p.has_drop) {
                drop_n<VEC>(p.drop, (uint64_t)m * p.quads + at.c[k] / 4, p.sigma, d[k]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[k][j] *= p.sigma;
            }
            if (p.gate) {
                float g[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float y = (float)ry[k][j], pj = p.post ? y * sy * wpost[k][j] : y;
                    float a, da;
                    gate_of(p.act, (float)rg[k][j], a, da);
                    g[j] = d[k][j] * pj * da;
                    d[k][j] *= a;
                    if constexpr (GSUM) {
                        if (ok) dgate[k][j] += g[j];
                    }
                }
                if constexpr (!GSUM) {
                    if (ok) store_part<TB, VEC, WHOLE>(dgate_to + at.c[k], p.C - at.c[k], g);
                }
            }
            if (p.post) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float yn = (float)ry[k][j] * sy;
                    if (ok) dpost[k][j] = __builtin_fmaf(d[k][j], yn, dpost[k][j]);
                    d[k][j] *= wpost[k][j];
                    sum[0] = __builtin_fmaf(d[k][j], yn, sum[0]);
                }
            }
        }
        if (p.post) {
            row_sum<WPR, 1>(sum, p.log_l, red, turn);
            const float mean = sum[0] * p.inv_c;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[k][j] = sy * (d[k][j] - (float)ry[k][j] * sy * mean);
        }
        if (ok) {
            TB *dy = static_cast<TB *>(p.dy) + row_at(p.sdy, m, p.S);
#pragma unroll
            for (int k = 0; k < NV; ++k) store_part<TB, VEC, WHOLE>(dy + at.c[k], p.C - at.c[k], d[k]);
        }
    }
    if (p.pre) leave_sums<VEC, NV, WPR, WHOLE>(at, p.C, p.log_l, dpre, p.part_pre);
    if (p.post) leave_sums<VEC, NV, WPR, WHOLE>(at, p.C, p.log_l, dpost, p.part_post);
    if constexpr (GSUM) leave_sums<VEC, NV, WPR, WHOLE>(at, p.C, p.log_l, dgate, p.part_gate);
}

struct SumParams {
    const float *pre, *post, *gate; // [blocks][C]
    float *dpre, *dpost;
    void *dgate;
    int64_t sgate; // gate rows apart by
    int C, tiles, segs;
    int64_t blocks, blocks_a_seg;
};

// The sums over workgroups: 32 columns of one result a workgroup, four a thread, in f64.
template <typename TB> __global__ __launch_bounds__(256) void residual_sums_kernel(SumParams p) {
    __shared__ double red[32][32 + 1];
    const int what = blockIdx.x / p.tiles, col = (threadIdx.x & 7) * 4, r = threadIdx.x >> 3;
    const int c0 = (blockIdx.x - what * p.tiles) * 32, c = c0 + col, left = p.C - c;
    const float *part = what == 0 ? p.pre : what == 1 ? p.post : p.gate;
    if (!part) return;
    const int64_t b0 = what < 2 ? 0 : (what - 2) * p.blocks_a_seg, b1 = what < 2 ? p.blocks : b0 + p.blocks_a_seg;
    double sum[4] = {0., 0., 0., 0.};
    auto add = [&](const float *v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[j];
    };
    int64_t b = b0 + r;
    for (; b + 7 * 32 < b1; b += 8 * 32) { // eight in flight
        float v[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) load_part<float, 4>(part + (b + 32 * k) * p.C + c, left, v[k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) add(v[k]);
    }
    for (; b < b1; b += 32) {
        float v[4];
        load_part<float, 4>(part + b * p.C + c, left, v);
        add(v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[r][col + j] = sum[j];
    __syncthreads();
    const int t = threadIdx.x;
    if (t >= 32 || c0 + t >= p.C) return;
    double all = 0.;
#pragma unroll
    for (int k = 0; k < 32; ++k) all += red[k][t];
    if (what == 0) p.dpre[c0 + t] = (float)all;
    else if (what == 1) p.dpost[c0 + t] = (float)all;
    else static_cast<TB *>(p.dgate)[(what - 2) * p.sgate + c0 + t] = (TB)(float)all;
}

// How rows of C channels are held.
struct Held {
    int wpr, nv, log_l;
    int rows; // a workgroup at once
};
Held held_of(int64_t C, int vec) {
    Held h{};
    h.nv = 8 / vec;
    h.log_l = 0;
    if (C <= 512) {
        h.wpr = 1;
        while ((8 << h.log_l) < C) ++h.log_l;
        h.rows = 256 >> h.log_l;
    } else {
        h.wpr = C <= 2048 ? 4 : 8;
        if (C > 4096) h.nv *= 2;
        h.rows = 1;
    }
    return h;
}

// Workgroups for each gate row of the backward: 768 in all, three a compute unit, while
// each has rows (8192 x 2048 bfloat16: 57.4 us; 1024: 58.0, 512: 60.0; 4 x 1999 x 320 f32:
// 27.5, 30.0 and 27.8), and enough that no f32 sum runs over more than kMostRows.
int64_t blocks_of(int64_t seg_rows, int64_t segs, const Held &h) {
    const int64_t most = (seg_rows + h.rows - 1) / h.rows;
    const int64_t least = (seg_rows + (int64_t)h.rows * kMostRows - 1) / ((int64_t)h.rows * kMostRows);
    return std::max<int64_t>(1, std::max(least, std::min(most, (768 + segs - 1) / segs)));
}

struct Segs {
    int64_t rows, n;
};
bool gate_summed(const gdn2_residual_norm_args &a) { return a.gate && a.gate_rows != GDN2_GATE_ROW; }
Segs segs_of(const gdn2_residual_norm_args &a) {
    if (gate_summed(a) && a.gate_rows == GDN2_GATE_SAMPLE) return {a.rows, a.samples};
    return {a.samples * a.rows, 1};
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
bool sizes_ok(const gdn2_residual_norm_args &a) {
    return a.channels <= kMostC && (double)a.samples * (double)a.rows < double(1 << 30) && a.samples < (1 << 30) && a.rows < (1 << 30);
}

template <typename TS, typename TB> constexpr int vec_of() { return sizeof(TB) == 2 ? 8 : 4; }

// The checks of both directions; GDN2_OK with *nothing where there is nothing to do.
gdn2_status check(const gdn2_residual_norm_args *a, const std::string &who, bool bwd, bool *nothing) {
    *nothing = false;
    if (!a) return fail(GDN2_EINVAL, who + "null args");
    if (a->samples < 0 || a->rows < 0 || a->channels < 0) return fail(GDN2_EINVAL, who + "negative dimension");
    if (a->activation < GDN2_GATE_NONE || a->activation > GDN2_GATE_SIGMOID) return fail(GDN2_EINVAL, who + "unknown activation");
    if (a->gate_rows < GDN2_GATE_ROW || a->gate_rows > GDN2_GATE_ALL) return fail(GDN2_EINVAL, who + "unknown gate_rows");
    if (!drop_ok(a->dropout)) return fail(GDN2_EINVAL, who + "p must be between 0 and 1");
    if (!(a->eps >= 0.)) return fail(GDN2_EINVAL, who + "eps must not be negative");
    if (!a->y && (a->gate || a->post_weight || a->dropout.p != 0.))
        return fail(GDN2_EINVAL, who + "a gate, a weight or dropout without y");
    if (a->channels == 0 || (!bwd && (a->samples == 0 || a->rows == 0))) {
        *nothing = true;
        return GDN2_OK;
    }
    return GDN2_OK;
}

ResParams params_of(const gdn2_residual_norm_args &a) {
    ResParams p{};
    p.x = a.x; p.y = a.y; p.gate = a.gate; p.post = a.post_weight; p.pre = a.pre_weight;
    p.out = a.out; p.normed = a.normed; p.stats = a.stats;
    p.sx = {a.stride_x_n, a.stride_x_s}; p.sy = {a.stride_y_n, a.stride_y_s};
    p.sgate = {a.gate_rows == GDN2_GATE_ALL ? 0 : a.stride_gate_n, a.gate_rows == GDN2_GATE_ROW ? a.stride_gate_s : 0};
    p.sout = {a.stride_out_n, a.stride_out_s}; p.snormed = {a.stride_normed_n, a.stride_normed_s};
    p.M = a.samples * a.rows;
    p.S = (int)a.rows; p.C = (int)a.channels; p.act = a.activation;
    p.quads = (uint32_t)((a.channels + 3) / 4);
    p.inv_c = 1.f / (float)a.channels; p.eps = (float)a.eps;
    p.alpha = (float)a.residual_scale;
    p.has_drop = a.dropout.p > 0.;
    p.drop = drop_of(a.dropout);
    p.sigma = a.dropout.p < 1. ? (float)(a.branch_scale / (1. - a.dropout.p)) : 0.f;
    return p;
}

// f(the kernels' NV and WPR)
#define GDN2_HELD(h, VEC, f)                                  \
    do {                                                      \
        if ((h).wpr == 1) f(8 / VEC, 1);                      \
        else if ((h).wpr == 4) f(8 / VEC, 4);                 \
        else if ((h).nv * VEC == 8) f(8 / VEC, 8);            \
        else f(16 / VEC, 8);                                  \
    } while (0)

template <typename TS, typename TB> gdn2_status forward(const gdn2_residual_norm_args *a, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    bool nothing;
    const gdn2_status st = check(a, who, false, &nothing);
    if (st != GDN2_OK || nothing) return st;
    if (!a->x) return fail(GDN2_EINVAL, who + "null pointer");
    if (!a->normed != !a->pre_weight) return fail(GDN2_EINVAL, who + "normed and pre_weight go together");
    if (!a->out && !a->normed) return fail(GDN2_EINVAL, who + "null pointer");
    if (!sizes_ok(*a)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    constexpr int VEC = vec_of<TS, TB>();
    const Held h = held_of(a->channels, VEC);
    ResParams p = params_of(*a);
    p.log_l = h.log_l;
    p.stream = (double)p.M * (double)p.C * sizeof(TB) >= kStreamBytes;
    const dim3 grid((unsigned)std::min<int64_t>((p.M + h.rows - 1) / h.rows, 1 << 21)), block(h.wpr == 8 ? 512 : 256);
#define GDN2_RUN(NV, WPR)                                                                                              \
    do {                                                                                                               \
        if (p.C % VEC == 0) hipLaunchKernelGGL((residual_norm_kernel<TS, TB, VEC, NV, WPR, true>), grid, block, 0, s, p); \
        else hipLaunchKernelGGL((residual_norm_kernel<TS, TB, VEC, NV, WPR, false>), grid, block, 0, s, p);            \
    } while (0)
    GDN2_HELD(h, VEC, GDN2_RUN);
#undef GDN2_RUN
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

struct BwdPlan {
    Held h;
    Segs seg;
    int64_t per, blocks;
    size_t each, bytes;
};
BwdPlan plan_of(const gdn2_residual_norm_args &a, int vec) {
    BwdPlan q{};
    q.h = held_of(a.channels, vec);
    q.seg = segs_of(a);
    q.per = blocks_of(q.seg.rows, q.seg.n, q.h);
    q.blocks = q.per * q.seg.n;
    q.each = align256(sizeof(float) * (size_t)q.blocks * (size_t)a.channels);
    q.bytes = q.each * ((a.pre_weight ? 1 : 0) + (a.post_weight ? 1 : 0) + (gate_summed(a) ? 1 : 0));
    return q;
}

template <typename TS, typename TB>
gdn2_status backward(const gdn2_residual_norm_bwd_args *b, hipStream_t s, const char *name) {
    const std::string who = std::string(name) + ": ";
    bool nothing;
    const gdn2_residual_norm_args *a = b ? &b->fwd : nullptr;
    const gdn2_status st = check(a, who, true, &nothing);
    if (st != GDN2_OK || nothing) return st;
    if (!b->dpre != !a->pre_weight || !b->dpost != !a->post_weight)
        return fail(GDN2_EINVAL, who + "a weight and its gradient go together");
    if (!b->dgate != !a->gate || !b->dy != !a->y) return fail(GDN2_EINVAL, who + "y, gate and their gradients go together");
    const bool some = a->samples > 0 && a->rows > 0;
    if (some) {
        if (!b->d_normed != !a->pre_weight) return fail(GDN2_EINVAL, who + "d_normed and pre_weight go together");
        if (a->pre_weight && !a->out) return fail(GDN2_EINVAL, who + "null pointer");
        if (!a->stats && (a->pre_weight || a->post_weight)) return fail(GDN2_EINVAL, who + "stats missing");
    }
    if (!sizes_ok(*a)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    const int64_t M = a->samples * a->rows; // (below 2^30)
    constexpr int VEC = vec_of<TS, TB>();
    const BwdPlan q = M > 0 ? plan_of(*a, VEC) : BwdPlan{};
    const bool gsum = gate_summed(*a) && (a->gate_rows == GDN2_GATE_ALL || a->samples > 0); // (no samples: no rows of dgate)
    ResParams p = params_of(*a);
    const int64_t wgs = (2 + (gsum ? (a->gate_rows == GDN2_GATE_SAMPLE ? a->samples : 1) : 0)) * (int64_t)((p.C + 31) / 32);
    if (q.blocks >= (1 << 22) || wgs >= (1 << 24)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    if (M == 0 && !a->pre_weight && !a->post_weight && !gsum) return GDN2_OK;
    if (M > 0) {
        if (q.bytes && (!b->workspace || b->workspace_bytes < q.bytes || reinterpret_cast<uintptr_t>(b->workspace) % 256))
            return fail(GDN2_EINVAL, who + "workspace missing, too small or not 256-byte aligned");
        char *ws = static_cast<char *>(b->workspace);
        if (a->pre_weight) p.part_pre = reinterpret_cast<float *>(ws), ws += q.each;
        if (a->post_weight) p.part_post = reinterpret_cast<float *>(ws), ws += q.each;
        if (gsum) p.part_gate = reinterpret_cast<float *>(ws);
        p.dr = b->d_out; p.dn = b->d_normed; p.dx = b->dx; p.dy = b->dy; p.dgate = b->dgate;
        p.sdr = {b->stride_d_out_n, b->stride_d_out_s}; p.sdn = {b->stride_d_normed_n, b->stride_d_normed_s};
        p.sdx = {b->stride_dx_n, b->stride_dx_s}; p.sdy = {b->stride_dy_n, b->stride_dy_s};
        p.sdgate = {b->stride_dgate_n, b->stride_dgate_s};
        p.log_l = q.h.log_l;
        p.seg_rows = q.seg.rows;
        p.blocks_a_seg = (int)q.per;
        const dim3 grid((unsigned)q.blocks), block(q.h.wpr == 8 ? 512 : 256);
#define GDN2_FORM(NV, WPR, WHOLE)                                                                                           \
    do {                                                                                                                    \
        if (gsum) hipLaunchKernelGGL((residual_norm_bwd_kernel<TS, TB, VEC, NV, WPR, WHOLE, true>), grid, block, 0, s, p);  \
        else hipLaunchKernelGGL((residual_norm_bwd_kernel<TS, TB, VEC, NV, WPR, WHOLE, false>), grid, block, 0, s, p);      \
    } while (0)
#define GDN2_RUN(NV, WPR)                      \
    do {                                       \
        if (p.C % VEC == 0) GDN2_FORM(NV, WPR, true); \
        else GDN2_FORM(NV, WPR, false);        \
    } while (0)
        GDN2_HELD(q.h, VEC, GDN2_RUN);
#undef GDN2_RUN
#undef GDN2_FORM
    }
    if (a->pre_weight || a->post_weight || gsum) {
        SumParams t{};
        t.C = p.C;
        t.tiles = (p.C + 31) / 32;
        t.blocks = M > 0 ? q.blocks : 0;
        t.blocks_a_seg = M > 0 ? q.per : 0;
        // (with no rows nothing of these is read)
        t.pre = M > 0 ? p.part_pre : reinterpret_cast<const float *>(a->pre_weight);
        t.post = M > 0 ? p.part_post : reinterpret_cast<const float *>(a->post_weight);
        t.gate = gsum ? (M > 0 ? p.part_gate : static_cast<const float *>(a->gate)) : nullptr;
        t.dpre = b->dpre; t.dpost = b->dpost; t.dgate = b->dgate; t.sgate = b->stride_dgate_n;
        hipLaunchKernelGGL((residual_sums_kernel<TB>), dim3((unsigned)wgs), dim3(256), 0, s, t);
    }
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

// (the same for every type: a lane holds 8 channels in each)
extern "C" size_t gdn2_residual_norm_bwd_workspace_bytes(const gdn2_residual_norm_bwd_args *b) {
    if (!b) return 0;
    const gdn2_residual_norm_args &a = b->fwd;
    if (a.samples <= 0 || a.rows <= 0 || a.channels <= 0 || !gdn2::sizes_ok(a)) return 0;
    return gdn2::plan_of(a, 8).bytes;
}

#define GDN2_ENTRY(suffix, TS, TB)                                                                                       \
    extern "C" gdn2_status gdn2_residual_norm_##suffix(const gdn2_residual_norm_args *args, gdn2_stream_t stream) {      \
        try { /* no exception leaves a C entry */                                                                        \
            return gdn2::forward<TS, TB>(args, (hipStream_t)stream, "gdn2_residual_norm_" #suffix);                      \
        } catch (const std::exception &) {                                                                               \
            return GDN2_EHIP;                                                                                            \
        }                                                                                                                \
    }                                                                                                                    \
    extern "C" gdn2_status gdn2_residual_norm_bwd_##suffix(const gdn2_residual_norm_bwd_args *args, gdn2_stream_t stream) { \
        try {                                                                                                            \
            return gdn2::backward<TS, TB>(args, (hipStream_t)stream, "gdn2_residual_norm_bwd_" #suffix);                 \
        } catch (const std::exception &) {                                                                               \
            return GDN2_EHIP;                                                                                            \
        }                                                                                                                \
    }
GDN2_ENTRY(f32, float, float)
GDN2_ENTRY(bf16, gdn2::bf16, gdn2::bf16)
GDN2_ENTRY(f32_bf16, float, gdn2::bf16)
