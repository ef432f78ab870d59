// gdn2_group_norm_act_*: group norm over channels-last rows with an activation
// (or an activated gate) in the same pass, and its adjoint.
//   n = (x - mean) rstd,  z = n weight + bias,  y = act(z) or z act(gate)
//   dz = dy act'(z) or dy act(gate),  dgate = dy z act'(gate),  dn = dz weight
//   dx = rstd (dn - mean(dn) - n mean(dn n)),  dweight = sum dz n,  dbias = sum dz
//
// S = 1 (a token's heads): L lanes hold a group in registers, so that everything
// is read once; the variance is taken about the mean.  A larger group is held by
// up to kMostParts workgroups: each publishes its part's sums, takes those of the
// others, and goes on with its registers, so that again everything is read
// once.  Sums that do not come in time it forms itself, so that no workgroup
// depends on another's being started.  Groups larger than that, and results in
// place of their input, take three passes: sums for every channel and chunk of
// rows, a join, and one that reads x again.  Every sum runs in a fixed order.
//
// Bound: HBM.  Rows: 32768 x 2048 bf16 gated 0.40 GB in 69.7 us (5.8 TB/s), the
// adjoint of 8192 x 2048 f32 gated 0.34 GB in 62 (5.4).  Held groups: 8 x 4096 x
// 1024 f32 in 32 groups 0.27 GB in 69 us (3.9 TB/s, the loads of a part and its
// stores do not overlap) where three passes take 76; 4 x 1999 x 320 bf16, adjoint,
// 15 MB in 22 us: three launches one after the other, the parts' exchange among them.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <exception>
#include <string>
#include <type_traits>

#include "common.hpp"
#include "gdn2_mixer.h"
#include "vec_io.hpp"

namespace gdn2 {
namespace {

struct GroupNormParams {
    const void *x, *gate, *dy;
    const float *weight, *bias;
    void *y; // forward: y; backward: dx
    void *dgate;
    float *stats; // [N][G] (mean, rstd); forward: NULL if not wanted
    float *dweight, *dbias;
    float *part;  // see the kernels
    float *sums;  // backward, S > 1: [N][G] means of dn and dn n
    int64_t sxn, sxs, sgn, sgs;
    int64_t N, S;
    int C, G, D, act;
    float eps;
    int log_l;         // rows kernels: lanes a group, as a power of two
    int row_blocks;    // backward rows kernel
    int lc;            // tile kernels: lanes along the channels (a power of two); held groups: any number
    int chunks, chunk; // row chunks of a sample, rows in one
    int spans, span;   // a group's chunks are joined in spans of `span` chunks
    float *joined;     // [N][G][spans][2] what they give, where they are several
    // held groups: channels a tile, tiles a set of groups, sets; a part: a chunk of rows by a tile
    int tile, tiles, sets, set_groups; // (sets: rows kernels, too)
    unsigned long long *words; // [sample][set][part][set_groups] what the parts publish
    int patience;              // looks at a word before its part's sums are formed here
};

// (v_rcp_f32 is within one unit in the last place)
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z)); }

template <int N> __device__ __forceinline__ void act_n(int act, const float *z, float *a) {
    if (act == GDN2_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = z[j] * sigmoid_f(z[j]);
    } else if (act == GDN2_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = 0.5f * z[j] * (1.f + erff(z[j] * 0.70710678118654752f));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = z[j];
    }
}
// a = act(z), d = act'(z)
template <int N> __device__ __forceinline__ void act_grad_n(int act, const float *z, float *a, float *d) {
    if (act == GDN2_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float s = sigmoid_f(z[j]);
            a[j] = z[j] * s;
            d[j] = s * __builtin_fmaf(z[j], 1.f - s, 1.f);
        }
    } else if (act == GDN2_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float c = 0.5f * (1.f + erff(z[j] * 0.70710678118654752f));
            a[j] = z[j] * c;
            d[j] = __builtin_fmaf(z[j] * 0.3989422804014327f, fast_exp2(-0.5f * kLog2e * z[j] * z[j]), c);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = z[j], d[j] = 1.f;
    }
}

// The place of a lane: VEC channels from c of the wave's groups, chunk k of NV.
template <int VEC, int NV> struct Lanes {
    int g, c[NV];
    bool ok[NV];
    __device__ Lanes(const GroupNormParams &p, int set, int lane) {
        const int l = 1 << p.log_l;
        g = set * (kWave >> p.log_l) + (lane >> p.log_l);
        const int first = lane & (l - 1);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int e = (k * l + first) * VEC;
            ok[k] = g < p.G && e < p.D; // (VEC divides D)
            c[k] = ok[k] ? g * p.D + e : 0;
        }
    }
};

// S = 1.  A wave takes U rows at a time of its groups.
template <typename T, int VEC, int NV, int U, bool GATE>
__global__ __launch_bounds__(256) void norm_rows_kernel(GroupNormParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lanes<VEC, NV> at(p, blockIdx.x % p.sets, lane); // (neighbours read neighbouring channels)
    const int64_t n0 = ((int64_t)(blockIdx.x / p.sets) * 4 + wave) * U;
    if (n0 >= p.N) return;
    Raw<T, VEC> rx[U][NV], rg[U][GATE ? NV : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t n = min(n0 + u, p.N - 1);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            rx[u][k] = raw_n<T, VEC>(static_cast<const T *>(p.x) + n * p.sxn + at.c[k]);
            if constexpr (GATE) rg[u][k] = raw_n<T, VEC>(static_cast<const T *>(p.gate) + n * p.sgn + at.c[k]);
        }
    }
    float wt[NV][VEC], bs[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) wt[k][j] = 1.f, bs[k][j] = 0.f;
        if (p.weight) load_n<float, VEC>(p.weight + at.c[k], wt[k]);
        if (p.bias) load_n<float, VEC>(p.bias + at.c[k], bs[k]);
    }
    const float inv_d = 1.f / p.D;
    float x[U][NV][VEC], mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        mean[u] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                x[u][k][j] = at.ok[k] ? (float)rx[u][k][j] : 0.f;
                mean[u] += x[u][k][j];
            }
    }
    lanes_sum<U>(mean, p.log_l);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        mean[u] *= inv_d;
        rstd[u] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                x[u][k][j] = at.ok[k] ? x[u][k][j] - mean[u] : 0.f;
                rstd[u] = __builtin_fmaf(x[u][k][j], x[u][k][j], rstd[u]);
            }
    }
    lanes_sum<U>(rstd, p.log_l);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        rstd[u] = 1.f / sqrtf(__builtin_fmaf(rstd[u], inv_d, p.eps));
        const int64_t n = n0 + u;
        if (n >= p.N) break;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float z[VEC], a[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[j] = __builtin_fmaf(x[u][k][j] * rstd[u], wt[k][j], bs[k][j]);
            if constexpr (GATE) {
                float gt[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) gt[j] = (float)rg[u][k][j];
                act_n<VEC>(p.act, gt, a);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] *= z[j];
            } else {
                act_n<VEC>(p.act, z, a);
            }
            if (at.ok[k]) stream_n<T, VEC>(static_cast<T *>(p.y) + n * p.sxn + at.c[k], a);
        }
        if (p.stats && at.g < p.G && (lane & ((1 << p.log_l) - 1)) == 0) {
            p.stats[(n * p.G + at.g) * 2] = mean[u];
            p.stats[(n * p.G + at.g) * 2 + 1] = rstd[u];
        }
    }
}

// S = 1, adjoint.  The waves of all workgroups walk the rows together, U at a time
// each (blocks of rows of their own, a power of two apart, meet in few memory
// channels: 94 against 66 us), the next ones' loads in flight, and keep dweight and dbias of its channels in registers; the
// workgroup's go to part [row_blocks][2][C].
template <typename T, int VEC, int NV, int U, bool GATE>
__global__ __launch_bounds__(256) void norm_rows_bwd_kernel(GroupNormParams p) {
    __shared__ float red[2][4][kWave * VEC * NV];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lanes<VEC, NV> at(p, blockIdx.x % p.sets, lane);
    const int64_t block = blockIdx.x / p.sets, n0 = block * 4 * U, step = (int64_t)p.row_blocks * 4 * U, n1 = p.N;
    float wt[NV][VEC], bs[NV][VEC], dwt[NV][VEC], dbs[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) wt[k][j] = 1.f, bs[k][j] = dwt[k][j] = dbs[k][j] = 0.f;
        if (p.weight) load_n<float, VEC>(p.weight + at.c[k], wt[k]);
        if (p.bias) load_n<float, VEC>(p.bias + at.c[k], bs[k]);
    }
    const float inv_d = 1.f / p.D;
    const int gs = min(at.g, p.G - 1);
    struct Rows {
        Raw<T, VEC> x[U][NV], dy[U][NV], gate[U][GATE ? NV : 1];
        float mean[U], rstd[U];
    };
    auto load = [&](int64_t first, Rows &r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = min(first + u, n1 - 1);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                r.x[u][k] = raw_n<T, VEC>(static_cast<const T *>(p.x) + n * p.sxn + at.c[k]);
                r.dy[u][k] = raw_n<T, VEC>(static_cast<const T *>(p.dy) + n * p.sxn + at.c[k]);
                if constexpr (GATE) r.gate[u][k] = raw_n<T, VEC>(static_cast<const T *>(p.gate) + n * p.sgn + at.c[k]);
            }
            r.mean[u] = p.stats[(n * p.G + gs) * 2];
            r.rstd[u] = p.stats[(n * p.G + gs) * 2 + 1];
        }
    };
    // The sums of kRowsAtOnce rows, those of the rest beside them: in registers all rows'
    // sums would be one chain of roundings.
    constexpr int kRowsAtOnce = 128;
    auto put_by = [&](bool start) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float *const a = &red[0][wave][(k * VEC + j) * kWave + lane], *const b = &red[1][wave][(k * VEC + j) * kWave + lane];
                *a = start ? 0.f : *a + dwt[k][j];
                *b = start ? 0.f : *b + dbs[k][j];
                dwt[k][j] = dbs[k][j] = 0.f;
            }
    };
    put_by(true);
    int taken = 0;
    Rows next;
    if (n0 + wave * U < n1) load(n0 + wave * U, next);
    for (int64_t first = n0 + wave * U; first < n1; first += step) {
        const Rows r = next;
        if ((taken += U) > kRowsAtOnce) {
            put_by(false);
            taken = U;
        }
        load(min(first + step, n1 - 1), next);
        float nn[U][NV][VEC], dn[U][NV][VEC], s[2 * U]; // sums of dn, of dn n
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = first + u;
            const bool in = n < n1;
            s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float z[VEC], a[VEC], d[VEC], dz[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    nn[u][k][j] = ((float)r.x[u][k][j] - r.mean[u]) * r.rstd[u];
                    z[j] = __builtin_fmaf(nn[u][k][j], wt[k][j], bs[k][j]);
                }
                if constexpr (GATE) {
                    float gt[VEC], dg[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) gt[j] = (float)r.gate[u][k][j];
                    act_grad_n<VEC>(p.act, gt, a, d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        dg[j] = (float)r.dy[u][k][j] * z[j] * d[j];
                        dz[j] = (float)r.dy[u][k][j] * a[j];
                    }
                    if (in && at.ok[k]) stream_n<T, VEC>(static_cast<T *>(p.dgate) + n * p.sgn + at.c[k], dg);
                } else {
                    act_grad_n<VEC>(p.act, z, a, d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dz[j] = (float)r.dy[u][k][j] * d[j];
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    dz[j] = in ? dz[j] : 0.f;
                    dwt[k][j] = in ? __builtin_fmaf(dz[j], nn[u][k][j], dwt[k][j]) : dwt[k][j];
                    dbs[k][j] += dz[j];
                    dn[u][k][j] = dz[j] * wt[k][j];
                    s[2 * u] += at.ok[k] ? dn[u][k][j] : 0.f;
                    s[2 * u + 1] = at.ok[k] ? __builtin_fmaf(dn[u][k][j], nn[u][k][j], s[2 * u + 1]) : s[2 * u + 1];
                }
            }
        }
        lanes_sum<2 * U>(s, p.log_l);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (first + u >= n1) break;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float dx[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) dx[j] = r.rstd[u] * (dn[u][k][j] - s[2 * u] * inv_d - nn[u][k][j] * (s[2 * u + 1] * inv_d));
                if (at.ok[k]) stream_n<T, VEC>(static_cast<T *>(p.y) + (first + u) * p.sxn + at.c[k], dx);
            }
        }
    }
    if (!p.part) return;
    put_by(false);
    __syncthreads();
    if (wave == 0) {
        float *out = p.part + block * 2 * p.C;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (at.ok[k]) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int i = (k * VEC + j) * kWave + lane;
                    out[at.c[k] + j] = (red[0][0][i] + red[0][1][i]) + (red[0][2][i] + red[0][3][i]);
                    out[p.C + at.c[k] + j] = (red[1][0][i] + red[1][1][i]) + (red[1][2][i] + red[1][3][i]);
                }
            }
    }
}

// dweight and dbias from the blocks' sums: part [blocks][2][C].  A workgroup
// takes 16 columns (of 2 C), 16 threads a column, which sum in 64 bits: there may be a
// million blocks.
__global__ __launch_bounds__(256) void column_sum_kernel(const float *part, int64_t blocks, int C, float *dweight, float *dbias) {
    __shared__ double red[16][17];
    const int col = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int64_t i = (int64_t)blockIdx.x * 16 + col;
    double sum = 0.;
    if (i < 2 * (int64_t)C)
#pragma unroll 4
        for (int64_t b = r; b < blocks; b += 16) sum += part[b * 2 * C + i];
    red[r][col] = sum;
    __syncthreads();
    if (r == 0 && i < 2 * (int64_t)C) {
        sum = 0.;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += red[k][col];
        float *out = i < C ? dweight : dbias;
        if (out) out[i < C ? i : i - C] = (float)sum;
    }
}

// The mean of n values and their squares about it, from sums about a value near the
// mean: what that one's roundings left (`rest`, sum d) and the squares (sum d^2).
struct Moments {
    float mean, squares;
    __device__ Moments(float about, float rest, float squares_about, float n) {
        mean = about + rest / n;
        const float q = __builtin_fmaf(-rest, rest / n, squares_about);
        squares = fmaxf(q, q - q); // (a NaN stays)
    }
};

// A workgroup's tile of the general form: lc lanes of VEC channels, 256 / lc rows
// at a time of a chunk of rows of sample n.
template <int VEC> struct TileAt {
    int c, rl, rows;
    bool ok;
    int64_t n, s0, s1;
    __device__ explicit TileAt(const GroupNormParams &p) {
        const int cl = threadIdx.x & (p.lc - 1);
        rl = threadIdx.x / p.lc;
        rows = 256 / p.lc;
        c = (blockIdx.y * p.lc + cl) * VEC;
        ok = c < p.C; // (VEC divides C)
        c = ok ? c : 0;
        n = blockIdx.x / p.chunks;
        s0 = (int64_t)(blockIdx.x % p.chunks) * p.chunk;
        s1 = min(s0 + p.chunk, p.S);
    }
};

// Sums over a chunk's rows of a pair of values a channel: every thread's over
// its rows are joined in LDS and go to part [N][chunks][2][C].
template <int VEC, typename F>
__device__ __forceinline__ void tile_pairs(const GroupNormParams &p, const TileAt<VEC> &at, const float *a, const float *b, F join) {
    __shared__ float red[2][VEC][256];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        red[0][j][threadIdx.x] = a[j];
        red[1][j][threadIdx.x] = b[j];
    }
    __syncthreads();
    if (at.rl == 0 && at.ok) {
        float *out = p.part + (int64_t)blockIdx.x * 2 * p.C + at.c;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float x, y;
            join(red[0][j], red[1][j], &x, &y);
            out[j] = x;
            out[p.C + j] = y;
        }
    }
}

// First pass, forward: the mean and the sum of squares about it of every channel
// over the chunk's rows.  A thread takes kBatch rows at a time, less its first one's
// value: their sum s and their squares q about their own mean in 32 bits, the batches'
// sum q, sum s and sum s^2 / n in 64, so that neither a large mean, nor a first value
// far from the others, nor many rows cost digits.
constexpr int kBatch = 8;
template <typename T, int VEC> __global__ __launch_bounds__(256) void norm_moments_kernel(GroupNormParams p) {
    const TileAt<VEC> at(p);
    double sum[VEC], sq[VEC], among[VEC]; // sum s, sum q, sum s^2 / n
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[j] = sq[j] = among[j] = 0.;
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c;
    int64_t row = at.s0 + at.rl, count = 0;
    float first[VEC];
    load_n<T, VEC>(x + min(row, at.s1 - 1) * p.sxs, first);
    auto batch = [&](auto rows) {
        constexpr int B = decltype(rows)::value;
        Raw<T, VEC> v[B];
#pragma unroll
        for (int i = 0; i < B; ++i) v[i] = raw_n<T, VEC>(x + (row + i * at.rows) * p.sxs);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float s = 0.f, q = 0.f;
#pragma unroll
            for (int i = 0; i < B; ++i) s += (float)v[i][j] - first[j];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float d = __builtin_fmaf(-s, 1.f / B, (float)v[i][j] - first[j]);
                q = __builtin_fmaf(d, d, q);
            }
            sum[j] += s;
            sq[j] += q;
            among[j] = __builtin_fma((double)s, (double)s * (1. / B), among[j]);
        }
        row += B * at.rows;
        count += B;
    };
    while (row + (kBatch - 1) * at.rows < at.s1) batch(std::integral_constant<int, kBatch>());
    while (row < at.s1) batch(std::integral_constant<int, 1>());
    const double inv = count ? 1. / (double)count : 0.;
    float mean_of[VEC], sq_of[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const double m = sum[j] * inv;
        mean_of[j] = (float)(first[j] + m);
        sq_of[j] = (float)(sq[j] + fmax(__builtin_fma(-m, sum[j], among[j]), 0.)); // (a NaN is in the mean)
    }
    const int64_t total = at.s1 - at.s0;
    tile_pairs<VEC>(p, at, mean_of, sq_of, [&](const float *m, const float *q, float *mean, float *m2) {
        const int cl = threadIdx.x & (p.lc - 1);
        float s = 0.f;
        for (int r = 0; r < at.rows; ++r) {
            const int64_t k = (total - r + at.rows - 1) / at.rows; // rows of thread r
            if (k > 0) s += (float)k * (m[r * p.lc + cl] - m[cl]);
        }
        const float about = m[cl] + s / (float)total;
        float rest = 0.f, t = 0.f; // (see Moments)
        for (int r = 0; r < at.rows; ++r) {
            const int64_t k = (total - r + at.rows - 1) / at.rows;
            const float d = m[r * p.lc + cl] - about;
            if (k > 0) {
                rest = __builtin_fmaf((float)k, d, rest);
                t += q[r * p.lc + cl] + (float)k * d * d;
            }
        }
        const Moments of(about, rest, t, (float)total);
        *mean = of.mean;
        *m2 = of.squares;
    });
}

__device__ __forceinline__ float block_sum(float v, float *red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// Second pass, forward: a group's mean and rstd from its channels' and chunks', or of
// a span of chunks the mean and the squares about it.
__global__ __launch_bounds__(256) void norm_join_kernel(GroupNormParams p) {
    __shared__ float red[4];
    const int64_t n = blockIdx.x / p.G;
    const int g = (int)(blockIdx.x % p.G), k0 = (int)blockIdx.y * p.span, k1 = min(k0 + p.span, p.chunks);
    const int entries = (k1 - k0) * p.D;
    const float *part = p.part + (n * p.chunks + k0) * 2 * p.C + g * p.D;
    auto rows = [&](int k) { return (float)min((int64_t)p.chunk, p.S - (int64_t)(k0 + k) * p.chunk); };
    const float base = part[0]; // a mean to sum about
    float s = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < entries; i += 256) {
        const int k = i / p.D;
        s = __builtin_fmaf(rows(k), part[(int64_t)k * 2 * p.C + i % p.D] - base, s);
    }
    const float size = (float)(min((int64_t)k1 * p.chunk, p.S) - (int64_t)k0 * p.chunk) * (float)p.D;
    const float about = base + block_sum(s, red) / size;
    float rest = 0.f, t = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < entries; i += 256) {
        const int k = i / p.D;
        const float *e = part + (int64_t)k * 2 * p.C + i % p.D;
        const float d = e[0] - about;
        rest = __builtin_fmaf(rows(k), d, rest);
        t += e[p.C] + rows(k) * d * d;
    }
    rest = block_sum(rest, red);
    const Moments of(about, rest, block_sum(t, red), size);
    if (threadIdx.x == 0) {
        float *out = p.spans > 1 ? p.joined + ((int64_t)blockIdx.x * p.spans + blockIdx.y) * 2 : p.stats + (int64_t)blockIdx.x * 2;
        out[0] = of.mean;
        out[1] = p.spans > 1 ? of.squares : 1.f / sqrtf(of.squares / size + p.eps);
    }
}
// ... the spans of a group: a wave each.
__global__ __launch_bounds__(64) void norm_join_spans_kernel(GroupNormParams p) {
    const float *e = p.joined + (int64_t)blockIdx.x * p.spans * 2;
    auto rows = [&](int k) { return (float)(min((int64_t)(k + 1) * p.span * p.chunk, p.S) - (int64_t)k * p.span * p.chunk); };
    const float base = e[0], size = (float)p.S * (float)p.D;
    float s = 0.f, rest = 0.f, t = 0.f;
    for (int k = threadIdx.x; k < p.spans; k += kWave) s = __builtin_fmaf(rows(k), e[2 * k] - base, s);
    const float about = base + wave_sum(s) / (float)p.S;
    for (int k = threadIdx.x; k < p.spans; k += kWave) {
        const float d = e[2 * k] - about, n = rows(k) * (float)p.D;
        rest = __builtin_fmaf(n, d, rest);
        t += __builtin_fmaf(n * d, d, e[2 * k + 1]);
    }
    const Moments of(about, wave_sum(rest), wave_sum(t), size);
    if (threadIdx.x == 0) {
        p.stats[(int64_t)blockIdx.x * 2] = of.mean;
        p.stats[(int64_t)blockIdx.x * 2 + 1] = 1.f / sqrtf(of.squares / size + p.eps);
    }
}

template <int VEC> struct Channels {
    float mean[VEC], rstd[VEC], wt[VEC], bs[VEC];
    __device__ Channels(const GroupNormParams &p, int64_t n, int c) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int64_t g = n * p.G + (c + j) / p.D;
            mean[j] = p.stats[g * 2];
            rstd[j] = p.stats[g * 2 + 1];
            wt[j] = 1.f;
            bs[j] = 0.f;
        }
        if (p.weight) load_n<float, VEC>(p.weight + c, wt);
        if (p.bias) load_n<float, VEC>(p.bias + c, bs);
    }
};

// Third pass, forward.
template <typename T, int VEC, bool GATE> __global__ __launch_bounds__(256) void norm_apply_kernel(GroupNormParams p) {
    const TileAt<VEC> at(p);
    if (!at.ok) return;
    const Channels<VEC> ch(p, at.n, at.c);
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c;
    const T *gate = static_cast<const T *>(p.gate) + at.n * p.sgn + at.c;
    T *y = static_cast<T *>(p.y) + at.n * p.sxn + at.c;
#pragma unroll 4
    for (int64_t s = at.s0 + at.rl; s < at.s1; s += at.rows) {
        float z[VEC], a[VEC];
        load_n<T, VEC>(x + s * p.sxs, z);
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[j] = __builtin_fmaf((z[j] - ch.mean[j]) * ch.rstd[j], ch.wt[j], ch.bs[j]);
        if constexpr (GATE) {
            float gt[VEC];
            load_n<T, VEC>(gate + s * p.sgs, gt);
            act_n<VEC>(p.act, gt, a);
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] *= z[j];
        } else {
            act_n<VEC>(p.act, z, a);
        }
        store_n<T, VEC>(y + s * p.sxs, a);
    }
}

// One element's adjoint up to dz and n.
template <typename T, int VEC, bool GATE>
__device__ __forceinline__ void dz_n(const GroupNormParams &p, const Channels<VEC> &ch, const float *x, const float *dy,
                                     const float *gt, float *n, float *dz, float *dg) {
    float z[VEC], a[VEC], d[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        n[j] = (x[j] - ch.mean[j]) * ch.rstd[j];
        z[j] = __builtin_fmaf(n[j], ch.wt[j], ch.bs[j]);
    }
    act_grad_n<VEC>(p.act, GATE ? gt : z, a, d);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        dz[j] = dy[j] * (GATE ? a[j] : d[j]);
        if constexpr (GATE) dg[j] = dy[j] * z[j] * d[j];
    }
}

// First pass, adjoint: sums of dz n and dz of every channel over the chunk's rows, four
// at a time in 32 bits and these in 64.
template <typename T, int VEC, bool GATE> __global__ __launch_bounds__(256) void norm_bwd_sums_kernel(GroupNormParams p) {
    const TileAt<VEC> at(p);
    const Channels<VEC> ch(p, at.n, at.c);
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c;
    const T *dy = static_cast<const T *>(p.dy) + at.n * p.sxn + at.c;
    const T *gate = static_cast<const T *>(p.gate) + at.n * p.sgn + at.c;
    double sum_a[VEC], sum_b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum_a[j] = sum_b[j] = 0.;
    int64_t row = at.s0 + at.rl;
    auto batch = [&](auto rows) {
        constexpr int B = decltype(rows)::value;
        float vx[B][VEC], vd[B][VEC], vg[B][VEC], a[VEC], b[VEC];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int64_t s = row + i * at.rows;
            load_n<T, VEC>(x + s * p.sxs, vx[i]);
            load_n<T, VEC>(dy + s * p.sxs, vd[i]);
            if constexpr (GATE) load_n<T, VEC>(gate + s * p.sgs, vg[i]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = b[j] = 0.f;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            float n[VEC], dz[VEC], dg[VEC];
            dz_n<T, VEC, GATE>(p, ch, vx[i], vd[i], vg[i], n, dz, dg);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a[j] = __builtin_fmaf(dz[j], n[j], a[j]);
                b[j] += dz[j];
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            sum_a[j] += a[j];
            sum_b[j] += b[j];
        }
        row += B * at.rows;
    };
    while (row + 3 * at.rows < at.s1) batch(std::integral_constant<int, 4>());
    while (row < at.s1) batch(std::integral_constant<int, 1>());
    float a[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = (float)sum_a[j], b[j] = (float)sum_b[j];
    tile_pairs<VEC>(p, at, a, b, [&](const float *u, const float *v, float *x0, float *x1) {
        const int cl = threadIdx.x & (p.lc - 1);
        float s = 0.f, t = 0.f;
        for (int r = 0; r < at.rows; ++r) {
            s += u[r * p.lc + cl];
            t += v[r * p.lc + cl];
        }
        *x0 = s;
        *x1 = t;
    });
}

// Second pass, adjoint: a group's means of dn n and dn, or a span of chunks' sums.
__global__ __launch_bounds__(256) void norm_bwd_join_kernel(GroupNormParams p) {
    __shared__ float red[4];
    const int64_t n = blockIdx.x / p.G;
    const int g = (int)(blockIdx.x % p.G), k0 = (int)blockIdx.y * p.span, k1 = min(k0 + p.span, p.chunks);
    const int entries = (k1 - k0) * p.D;
    const float *part = p.part + (n * p.chunks + k0) * 2 * p.C + g * p.D;
    float s = 0.f, t = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < entries; i += 256) {
        const float *e = part + (int64_t)(i / p.D) * 2 * p.C + i % p.D;
        const float w = p.weight ? p.weight[g * p.D + i % p.D] : 1.f;
        s = __builtin_fmaf(e[0], w, s);
        t = __builtin_fmaf(e[p.C], w, t);
    }
    s = block_sum(s, red);
    t = block_sum(t, red);
    if (threadIdx.x == 0) {
        const float size = p.spans > 1 ? 1.f : (float)p.S * (float)p.D;
        float *out = p.spans > 1 ? p.joined + ((int64_t)blockIdx.x * p.spans + blockIdx.y) * 2 : p.sums + (int64_t)blockIdx.x * 2;
        out[0] = s / size;
        out[1] = t / size;
    }
}
// ... the spans of a group: a wave each.
__global__ __launch_bounds__(64) void norm_bwd_join_spans_kernel(GroupNormParams p) {
    const float *e = p.joined + (int64_t)blockIdx.x * p.spans * 2;
    float s = 0.f, t = 0.f;
    for (int k = threadIdx.x; k < p.spans; k += kWave) {
        s += e[2 * k];
        t += e[2 * k + 1];
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (threadIdx.x == 0) {
        const float size = (float)p.S * (float)p.D;
        p.sums[(int64_t)blockIdx.x * 2] = s / size;
        p.sums[(int64_t)blockIdx.x * 2 + 1] = t / size;
    }
}

// Third pass, adjoint.
template <typename T, int VEC, bool GATE> __global__ __launch_bounds__(256) void norm_bwd_apply_kernel(GroupNormParams p) {
    const TileAt<VEC> at(p);
    if (!at.ok) return;
    const Channels<VEC> ch(p, at.n, at.c);
    float s2[VEC], s1[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int64_t g = at.n * p.G + (at.c + j) / p.D;
        s2[j] = p.sums[g * 2];
        s1[j] = p.sums[g * 2 + 1];
    }
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c;
    const T *dy = static_cast<const T *>(p.dy) + at.n * p.sxn + at.c;
    T *dx = static_cast<T *>(p.y) + at.n * p.sxn + at.c;
    const T *gate = static_cast<const T *>(p.gate) + at.n * p.sgn + at.c;
    T *dgate = static_cast<T *>(p.dgate) + at.n * p.sgn + at.c;
#pragma unroll 4
    for (int64_t s = at.s0 + at.rl; s < at.s1; s += at.rows) {
        float vx[VEC], vd[VEC], vg[VEC], n[VEC], dz[VEC], dg[VEC], o[VEC];
        load_n<T, VEC>(x + s * p.sxs, vx);
        load_n<T, VEC>(dy + s * p.sxs, vd);
        if constexpr (GATE) load_n<T, VEC>(gate + s * p.sgs, vg);
        dz_n<T, VEC, GATE>(p, ch, vx, vd, vg, n, dz, dg);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = ch.rstd[j] * (dz[j] * ch.wt[j] - s1[j] - n[j] * s2[j]);
        store_n<T, VEC>(dx + s * p.sxs, o);
        if constexpr (GATE) store_n<T, VEC>(dgate + s * p.sgs, dg);
    }
}

// -- groups that several workgroups hold ----------------------------------------

// All ones over the words that parts publish.
__global__ __launch_bounds__(256) void norm_prepare_kernel(uint4 *words, int64_t n16) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256)
        words[i] = uint4{~0u, ~0u, ~0u, ~0u};
}

// A part of a set of groups: E rows a thread of VEC channels, lc lanes along the
// tile's channels.
constexpr int kMostParts = 64;
constexpr int NT = 256;     // threads
constexpr int kTile = 256;  // channels a tile at most
constexpr int kSet = 128;   // groups a set at most
constexpr int kMostWords = 1024; // parts by groups of a set at most
template <int VEC, int E> struct Held {
    int c, in_tile, rl, rows; // the lane's first channel, that in its tile; its row and the rows at a time
    unsigned number;
    int set, part, parts, count; // rows of this chunk
    bool ok;
    int64_t n, s0;
    __device__ Held(const GroupNormParams &p, unsigned number) {
        parts = p.chunks * p.tiles;
        part = (int)(number % (unsigned)parts); // (a set's parts start together: the waits are shorter)
        const unsigned ns = number / (unsigned)parts;
        set = (int)(ns % (unsigned)p.sets);
        n = ns / (unsigned)p.sets;
        const int tl = part % p.tiles;
        this->number = number;
        rows = NT / p.lc;
        rl = (int)threadIdx.x / p.lc;
        const int cl = (int)threadIdx.x % p.lc;
        const int set_c = set * p.set_groups * p.D, most = min(p.set_groups * p.D, p.C - set_c);
        in_tile = cl * VEC;
        c = set_c + tl * p.tile + in_tile;
        ok = rl < rows && in_tile < p.tile && tl * p.tile + in_tile < most; // (VEC divides all of these)
        c = ok ? c : set_c;
        s0 = (int64_t)(part / p.tiles) * p.chunk;
        count = (int)min((int64_t)p.chunk, p.S - s0);
    }
    __device__ int64_t row(int i) const { return s0 + min(rl + i * rows, count - 1); }
    __device__ bool has(int i) const { return ok && rl + i * rows < count; }
    // channels of the tile, and groups of the set that are there
    __device__ int channels(const GroupNormParams &p) const {
        const int set_c = set * p.set_groups * p.D;
        return min(p.tile, min(p.set_groups * p.D, p.C - set_c) - (part % p.tiles) * p.tile);
    }
    __device__ int groups(const GroupNormParams &p) const { return min(p.set_groups, p.G - set * p.set_groups); }
};

// A published pair is never all ones.
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    const unsigned lo = __builtin_bit_cast(unsigned, a), hi = b != b ? 0x7FC00000u : __builtin_bit_cast(unsigned, b);
    return (unsigned long long)hi << 32 | lo;
}
// The threads that work on a group: `share` neighbouring lanes of a wave, a power
// of two.
struct GroupLanes {
    int share, g, t;
    bool ok;
    __device__ explicit GroupLanes(int ng) {
        share = 64;
        while (share * ng > NT) share /= 2; // (ng is the same in the workgroup, and at most kSet)
        share = __builtin_amdgcn_readfirstlane(share);
        g = (int)threadIdx.x / share;
        t = (int)threadIdx.x % share;
        ok = g < ng;
        g = ok ? g : 0;
    }
    __device__ float sum(float v) const { return lanes_sum(v, __builtin_ctz(share)); } // to all of them
};

// f(i) for E rows, unrolled where they are in registers
template <int E, bool ONCE, typename F> __device__ __forceinline__ void each_row(std::integral_constant<bool, ONCE>, F f) {
    if constexpr (ONCE) {
#pragma unroll
        for (int i = 0; i < E; ++i) f(i);
    } else {
#pragma unroll 1
        for (int i = 0; i < E; ++i) f(i);
    }
}

// Publishes the part's pair of every group and collects those of all parts in
// all[2][parts][groups] (each entry by the lane that reads it).  `form`(k) makes
// every thread of a group return the pair of part k, by the operations of its own
// workgroup.
template <typename Form>
__device__ __forceinline__ void collect(const GroupNormParams &p, const GroupLanes &gl, int64_t set, int part, int parts, int ng, float2 own,
                                        float *all, unsigned long long *missing, Form form) {
    unsigned long long *const w = p.words + set * parts * p.set_groups + gl.g;
    float *const a = all, *const b = all + kMostWords;
    auto look = [&](int k) { return __hip_atomic_load(w + (int64_t)k * p.set_groups, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto take = [&](int k, unsigned long long v) {
        a[k * ng + gl.g] = __builtin_bit_cast(float, (unsigned)v);
        b[k * ng + gl.g] = __builtin_bit_cast(float, (unsigned)(v >> 32));
    };
    if (gl.ok && parts > 1 && gl.t == 0)
        __hip_atomic_store(w + (int64_t)part * p.set_groups, pair(own.x, own.y), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    bool late = false;
    if (gl.ok)
        for (int k = gl.t; k < parts; k += gl.share) {
            unsigned long long v = pair(own.x, own.y);
            if (k != part) {
                v = look(k);
                for (int i = 0; i < p.patience && v == ~0ull; ++i) {
                    __builtin_amdgcn_s_sleep(1);
                    v = look(k);
                }
                if (v == ~0ull) {
                    late = true;
                    atomicOr(missing, 1ull << k);
                }
            }
            take(k, v);
        }
    if (parts == 1 || !__syncthreads_or(late)) return;
    const unsigned long long these = *missing;
    for (int k = 0; k < parts; ++k) {
        if (!(these >> k & 1)) continue;
        const float2 f = form(k);
        if (gl.ok && k % gl.share == gl.t) take(k, pair(f.x, f.y));
    }
}

template <typename T, int VEC, int E, bool GATE>
__global__ __launch_bounds__(NT) void norm_held_kernel(GroupNormParams p) {
    __shared__ float red[3][VEC * NT]; // a value, sums about it, and squares about their mean, of a thread's channels
    __shared__ float all[2][kMostWords], stat[2][kSet];
    __shared__ unsigned long long missing;
    const int tid = threadIdx.x;
    const Held<VEC, E> at(p, blockIdx.x);
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c;
    const T *gate = static_cast<const T *>(p.gate) + at.n * p.sgn + at.c;
    Raw<T, VEC> rx[E], rg[GATE ? E : 1];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        rx[i] = raw_n<T, VEC>(x + at.row(i) * p.sxs);
        if constexpr (GATE) rg[i] = raw_n<T, VEC>(gate + at.row(i) * p.sgs);
    }
    if (tid == 0) missing = 0;
    const int ng = at.groups(p);
    const GroupLanes gl(ng);
    float wt[VEC], bs[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) wt[j] = 1.f, bs[j] = 0.f;
    if (p.weight) load_n<float, VEC>(p.weight + at.c, wt);
    if (p.bias) load_n<float, VEC>(p.bias + at.c, bs);
    int group[VEC]; // of the set (the same in every part of it)
#pragma unroll
    for (int j = 0; j < VEC; ++j) group[j] = p.tiles == 1 && at.ok ? (at.in_tile + j) / p.D : 0;

    // The mean of a part and the squares about it.  A thread sums less its first value,
    // its squares are about its own mean, and both are joined about the part's: neither
    // a large mean nor a value far from the others costs digits.
    auto moments = [&](const Held<VEC, E> &h, auto at_once, auto value) { // value(i): the i-th row's; at_once: rows unrolled
        const int gc = min(p.D, h.channels(p)); // the tile's channels of a group
        auto rows_of = [&](int r) { return max(0, (h.count - r + h.rows - 1) / h.rows); }; // of a channel's r-th thread
        const int mine = h.ok ? rows_of(h.rl) : 0;
        const float inv = mine ? 1.f / mine : 0.f;
        float base[VEC], s[VEC], q[VEC];
        const Raw<T, VEC> v0 = value(0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) base[j] = (float)v0[j], s[j] = q[j] = 0.f;
        each_row<E>(at_once, [&](int i) {
            const Raw<T, VEC> v = value(i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j] += i < mine ? (float)v[j] - base[j] : 0.f;
        });
        each_row<E>(at_once, [&](int i) {
            const Raw<T, VEC> v = value(i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = i < mine ? __builtin_fmaf(-s[j], inv, (float)v[j] - base[j]) : 0.f;
                q[j] = __builtin_fmaf(d, d, q[j]);
            }
        });
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            red[0][j * NT + tid] = base[j];
            red[1][j * NT + tid] = s[j];
            red[2][j * NT + tid] = q[j];
        }
        __syncthreads();
        // channel c of the tile is at c % VEC of lane c / VEC, for every row of threads:
        // f(n, 1 / n, place, k) of those of them that hold rows, in four chains
        const int full = h.count / h.rows, more = h.count % h.rows; // rows of a thread; the first `more` have one more
        const int there = full ? h.rows : more;
        const float n0 = (float)full, n1 = (float)(full + 1), inv0 = 1.f / n0, inv1 = 1.f / n1;
        auto each = [&](auto f) {
            if (gl.ok)
                for (int c = gl.g * p.D + gl.t; c < gl.g * p.D + gc; c += gl.share) {
                    const int o = (c % VEC) * NT + c / VEC;
                    auto one = [&](int r, int k) {
                        f(r < more ? n1 : n0, r < more ? inv1 : inv0, o + r * p.lc, k);
                    };
                    int r = 0;
                    for (; r + 4 <= there; r += 4)
#pragma unroll
                        for (int k = 0; k < 4; ++k) one(r + k, k);
                    for (; r < there; ++r) one(r, 0);
                }
        };
        const float one = red[0][gl.g * p.D % VEC * NT + gl.g * p.D / VEC], size = (float)h.count * (float)gc;
        float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        each([&](float n, float, int at, int k) { t[k] += __builtin_fmaf(n, red[0][at] - one, red[1][at]); });
        const float about = one + gl.sum((t[0] + t[1]) + (t[2] + t[3])) / size;
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = 0.f;
        each([&](float n, float inv_n, int at, int k) {
            const float d = __builtin_fmaf(n, red[0][at] - about, red[1][at]);
            t[k] += d;
            t[4 + k] += __builtin_fmaf(d * d, inv_n, red[2][at]);
        });
        float two[2] = {(t[0] + t[1]) + (t[2] + t[3]), (t[4] + t[5]) + (t[6] + t[7])};
        lanes_sum<2>(two, __builtin_ctz(gl.share));
        const Moments of(about, two[0], two[1], size);
        const float2 m = {of.mean, of.squares};
        __syncthreads(); // (red may be written again)
        return m;
    };
    const float2 own = moments(at, std::true_type(), [&](int i) { return rx[i]; });
    collect(p, gl, at.n * p.sets + at.set, at.part, at.parts, ng, own, all[0], &missing, [&](int k) {
        const Held<VEC, E> other(p, at.number - at.part + k);
        const T *const y = static_cast<const T *>(p.x) + other.n * p.sxn + other.c;
        return moments(other, std::false_type(), [&](int i) { return raw_n<T, VEC>(y + other.row(i) * p.sxs); });
    });
    const float *const means = all[0], *const squares = all[1];
    auto size = [&](int k) { // elements of part k
        const int64_t rows = min((int64_t)p.chunk, p.S - (int64_t)(k / p.tiles) * p.chunk);
        return (float)rows * (float)(p.tiles == 1 ? p.D : min(p.tile, p.D - (k % p.tiles) * p.tile));
    };
    // (a lane reads what it wrote itself; sums about part 0's mean, the same in every part)
    const float one = __shfl(gl.t == 0 ? means[gl.g] : 0.f, 0, gl.share);
    float s = 0.f, about[2] = {0.f, 0.f};
    for (int k = gl.t; gl.ok && k < at.parts; k += gl.share) s = __builtin_fmaf(size(k), means[k * ng + gl.g] - one, s);
    const float total = (float)p.S * (float)p.D, near = one + gl.sum(s) / total;
    for (int k = gl.t; gl.ok && k < at.parts; k += gl.share) {
        const float d = means[k * ng + gl.g] - near;
        about[0] = __builtin_fmaf(size(k), d, about[0]);
        about[1] += __builtin_fmaf(size(k) * d, d, squares[k * ng + gl.g]);
    }
    lanes_sum<2>(about, __builtin_ctz(gl.share));
    const Moments of(near, about[0], about[1], total);
    const float mean = of.mean, rstd = 1.f / sqrtf(of.squares / total + p.eps);
    if (gl.ok && gl.t == 0) {
        stat[0][gl.g] = mean;
        stat[1][gl.g] = rstd;
        if (p.stats && at.part == 0) {
            float *st = p.stats + (at.n * p.G + at.set * p.set_groups + gl.g) * 2;
            st[0] = mean;
            st[1] = rstd;
        }
    }
    __syncthreads();
    if (!at.ok) return;
    float m[VEC], rs[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        m[j] = stat[0][group[j]];
        rs[j] = stat[1][group[j]];
    }
    T *y = static_cast<T *>(p.y) + at.n * p.sxn + at.c;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (!at.has(i)) break;
        float z[VEC], a[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[j] = __builtin_fmaf(((float)rx[i][j] - m[j]) * rs[j], wt[j], bs[j]);
        if constexpr (GATE) {
            float gt[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) gt[j] = (float)rg[i][j];
            act_n<VEC>(p.act, gt, a);
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] *= z[j];
        } else {
            act_n<VEC>(p.act, z, a);
        }
        stream_n<T, VEC>(y + at.row(i) * p.sxs, a);
    }
}

template <typename T, int VEC, int E, bool GATE>
__global__ __launch_bounds__(NT) void norm_held_bwd_kernel(GroupNormParams p) {
    __shared__ float red[2][VEC * NT]; // sums of dz n and dz of a thread's channels
    __shared__ float all[2][kMostWords], stat[2][kSet];
    __shared__ unsigned long long missing;
    const int tid = threadIdx.x;
    const Held<VEC, E> at(p, blockIdx.x);
    const T *x = static_cast<const T *>(p.x) + at.n * p.sxn + at.c, *dy = static_cast<const T *>(p.dy) + at.n * p.sxn + at.c;
    const T *gate = static_cast<const T *>(p.gate) + at.n * p.sgn + at.c;
    const Channels<VEC> ch(p, at.n, at.c);
    Raw<T, VEC> rx[E], ry[E], rg[GATE ? E : 1];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        rx[i] = raw_n<T, VEC>(x + at.row(i) * p.sxs);
        ry[i] = raw_n<T, VEC>(dy + at.row(i) * p.sxs);
        if constexpr (GATE) rg[i] = raw_n<T, VEC>(gate + at.row(i) * p.sgs);
    }
    if (tid == 0) missing = 0;
    const int ng = at.groups(p);
    const GroupLanes gl(ng);
    T *dgate = static_cast<T *>(p.dgate) + at.n * p.sgn + at.c;
    // n and dz (and the gate's gradient) of a row
    auto element = [&](const Channels<VEC> &ch, const Raw<T, VEC> &x, const Raw<T, VEC> &y, const Raw<T, VEC> &g, float *n, float *dz, float *dg) {
        float vx[VEC], vy[VEC], vg[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            vx[j] = (float)x[j];
            vy[j] = (float)y[j];
            if constexpr (GATE) vg[j] = (float)g[j];
        }
        dz_n<T, VEC, GATE>(p, ch, vx, vy, vg, n, dz, dg);
    };
    // The sums of a part: a group's of dn n and dn; a channel's of dz n and dz go to
    // part [sample][chunk][2][C] for the weights' gradients.
    auto sums = [&](const Held<VEC, E> &h, const Channels<VEC> &ch, auto at_once, auto value_x, auto value_y, auto value_g) {
        constexpr bool keep = decltype(at_once)::value; // this workgroup's own
        float a[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = b[j] = 0.f;
        each_row<E>(at_once, [&](int i) {
            if (!h.has(i)) return;
            float n[VEC], dz[VEC], dg[VEC];
            element(ch, value_x(i), value_y(i), value_g(i), n, dz, dg);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a[j] = __builtin_fmaf(dz[j], n[j], a[j]);
                b[j] += dz[j];
            }
            if constexpr (GATE && keep) stream_n<T, VEC>(dgate + h.row(i) * p.sgs, dg);
        });
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            red[0][j * NT + tid] = a[j];
            red[1][j * NT + tid] = b[j];
        }
        __syncthreads();
        const int c0 = h.set * p.set_groups * p.D + h.part % p.tiles * p.tile, gc = min(p.D, h.channels(p));
        float *out = p.part && keep ? p.part + (h.n * p.chunks + h.part / p.tiles) * 2 * p.C + c0 : nullptr;
        float t[2] = {0.f, 0.f};
        if (gl.ok)
            for (int c = gl.g * p.D + gl.t; c < gl.g * p.D + gc; c += gl.share) {
                const int o = (c % VEC) * NT + c / VEC;
                const float w = p.weight ? p.weight[c0 + c] : 1.f;
                float u = 0.f, v = 0.f;
#pragma unroll 4
                for (int r = 0; r < h.rows; ++r) {
                    u += red[0][o + r * p.lc];
                    v += red[1][o + r * p.lc];
                }
                if (out) {
                    out[c] = u;
                    out[p.C + c] = v;
                }
                t[0] = __builtin_fmaf(u, w, t[0]);
                t[1] = __builtin_fmaf(v, w, t[1]);
            }
        lanes_sum<2>(t, __builtin_ctz(gl.share));
        __syncthreads(); // (red may be written again)
        return float2{t[0], t[1]};
    };
    const float2 own = sums(at, ch, std::true_type(), [&](int i) { return rx[i]; }, [&](int i) { return ry[i]; },
                           [&](int i) { return rg[GATE ? i : 0]; });
    collect(p, gl, at.n * p.sets + at.set, at.part, at.parts, ng, own, all[0], &missing, [&](int k) {
        const Held<VEC, E> o(p, at.number - at.part + k);
        auto from = [&](const void *base, int64_t sn, int64_t ss, int i) {
            return raw_n<T, VEC>(static_cast<const T *>(base) + o.n * sn + o.row(i) * ss + o.c);
        };
        return sums(o, Channels<VEC>(p, o.n, o.c), std::false_type(), [&](int i) { return from(p.x, p.sxn, p.sxs, i); },
                    [&](int i) { return from(p.dy, p.sxn, p.sxs, i); },
                    [&](int i) { return GATE ? from(p.gate, p.sgn, p.sgs, i) : Raw<T, VEC>{}; });
    });
    float t[2] = {0.f, 0.f};
    for (int k = gl.t; gl.ok && k < at.parts; k += gl.share) { // (a lane reads what it wrote itself)
        t[0] += all[0][k * ng + gl.g];
        t[1] += all[1][k * ng + gl.g];
    }
    lanes_sum<2>(t, __builtin_ctz(gl.share));
    if (gl.ok && gl.t == 0) {
        const float size = (float)p.S * (float)p.D;
        stat[0][gl.g] = t[0] / size;
        stat[1][gl.g] = t[1] / size;
    }
    __syncthreads();
    if (!at.ok) return;
    float m2[VEC], m1[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int g = p.tiles == 1 ? (at.in_tile + j) / p.D : 0;
        m2[j] = stat[0][g];
        m1[j] = stat[1][g];
    }
    T *dx = static_cast<T *>(p.y) + at.n * p.sxn + at.c;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (!at.has(i)) break;
        float n[VEC], dz[VEC], dg[VEC], o[VEC];
        element(ch, rx[i], ry[i], rg[GATE ? i : 0], n, dz, dg);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = ch.rstd[j] * (dz[j] * ch.wt[j] - m1[j] - n[j] * m2[j]);
        stream_n<T, VEC>(dx + at.row(i) * p.sxs, o);
    }
}

// The statistics of groups of nothing.
__global__ __launch_bounds__(256) void norm_no_stats_kernel(float *stats, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) stats[i] = NAN;
}

// -- host ---------------------------------------------------------------------

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

struct Plan {
    bool rows; // S = 1 with groups that a wave holds
    bool held; // groups that up to kMostParts workgroups hold
    int e; // rows a thread
    int tile, set_groups;
    int64_t o_words, words; // bytes of the words that parts publish
    int vec, nv, u, log_l, sets;
    int row_blocks;
    int lc, tiles, chunks, chunk, spans, span;
    size_t o_stats, o_sums, o_joined, bytes; // workspace: part, then these
};

int up_log2(int64_t n) {
    int k = 0;
    while ((int64_t(1) << k) < n) ++k;
    return k;
}

// see gdn2_group_norm_patience; 512 looks are about half a millisecond
std::atomic<int> g_patience{512};

// The plan of a held group; false where it takes too many parts.
constexpr int kRows3 = 16, kRows3Bwd = 12; // rows a thread at most (as many as leave no register in memory)
bool hold(const gdn2_group_norm_args &a, bool bwd, int vec, Plan *q) {
    const int G = (int)a.groups, D = (int)a.channels / G;
    int unit = 1; // groups that make a multiple of vec channels
    while ((int64_t)unit * D % vec) unit *= 2;
    // Rows a thread, channels of a set of whole groups, parts at most.  Eight rows run
    // faster than four (8 x 4096 x 1024 f32 in 64 channels: 70 against 96 us) and than
    // sixteen (4 x 2000 x 2048 bf16 gated: 33 against 36 us); 128 channels faster
    // than 64 but for more than 32 parts (84 against 70 us).
    const int most = bwd ? kRows3Bwd : kRows3;
    const int forms[][3] = {{4, 128, 1}, {8, 128, 32}, {8, 64, 32}, {most, 64, 32}, {most, 128, kMostParts}, {most, 64, kMostParts}};
    for (const auto &f : forms) {
        const int sg = std::max(unit, f[1] / D / unit * unit);
        q->set_groups = std::min(sg, G);
        q->sets = (G + q->set_groups - 1) / q->set_groups;
        const int64_t set_c = (int64_t)q->set_groups * D;
        if (q->set_groups > 1 && set_c > kTile) return false;
        q->tile = (int)std::min<int64_t>(set_c, kTile);
        q->tiles = (int)((set_c + q->tile - 1) / q->tile);
        q->lc = q->tile / vec;
        const int64_t chunk = (int64_t)(NT / q->lc) * f[0], chunks = (a.rows + chunk - 1) / chunk, parts = chunks * q->tiles;
        if (parts > f[2] || parts * q->set_groups > kMostWords) continue;
        q->held = true;
        q->vec = vec;
        q->e = f[0];
        q->chunk = (int)std::min<int64_t>(chunk, a.rows);
        q->chunks = (int)chunks;
        return true;
    }
    return false;
}

constexpr int kJoin = 16384;
Plan plan_of(const gdn2_group_norm_args &a, bool bwd, bool vec4, bool sums_wanted, bool in_place) {
    Plan q{};
    const int64_t C = a.channels, D = C / a.groups, N = a.samples, S = a.rows;
    q.vec = vec4 && D % 4 == 0 ? 4 : 1;
    const int64_t lanes = (D + q.vec - 1) / q.vec;
    q.log_l = std::min(6, up_log2(lanes));
    const int64_t nv = (lanes + (1 << q.log_l) - 1) >> q.log_l;
    q.rows = S == 1 && nv <= (bwd && q.vec == 4 ? 8 : 16);
    if (q.rows) {
        q.nv = nv == 1 ? 1 : nv <= 4 ? 4 : bwd && q.vec == 4 ? 8 : 16;
        q.u = q.nv == 1 ? 4 : 1;
        const int gpw = 64 >> q.log_l;
        q.sets = (int)((a.groups + gpw - 1) / gpw);
        if (bwd) {
            // 512 workgroups, two a compute unit (1024: 67 against 62.5 us at 8192 x 2048
            // gated f32; more of them for 262144 rows: 1326 against 1195), of at least two rows
            // a wave
            q.row_blocks = (int)std::max<int64_t>(1, std::min<int64_t>((512 + q.sets - 1) / q.sets, (N + 7) / 8));
            q.bytes = sums_wanted ? up256(8 * (size_t)q.row_blocks * C) : 0;
        }
        return q;
    }
    q.vec = vec4 && C % 4 == 0 ? 4 : 1;
    if (!in_place && (hold(a, bwd, q.vec, &q) || (q.vec > 1 && hold(a, bwd, 1, &q)))) {
        size_t at = bwd && sums_wanted ? up256(8 * (size_t)(N * q.chunks) * C) : 0;
        q.o_words = (int64_t)at;
        q.words = q.chunks * q.tiles > 1 ? (int64_t)up256(8 * (size_t)(N * q.sets * q.chunks * q.tiles * q.set_groups)) : 0;
        q.bytes = at + (size_t)q.words;
        return q;
    }
    // the widest tile that wastes at most an eighth of its lanes, or the one that wastes least
    const int64_t need = (C + q.vec - 1) / q.vec;
    int64_t best = 0;
    for (int lc = 64; lc >= 8; lc /= 2) {
        const int64_t padded = (need + lc - 1) / lc * lc;
        if (best == 0 || padded < best) {
            best = padded;
            q.lc = lc;
        }
        if (8 * (padded - need) <= need) break;
    }
    q.tiles = (int)((need + q.lc - 1) / q.lc);
    // about 2048 workgroups, of at least four rows a thread
    const int64_t rows = 256 / q.lc;
    const int64_t most = std::max<int64_t>(1, S / (4 * rows)), want = std::max<int64_t>(1, 2048 / (N * q.tiles));
    // and as few as one workgroup of the join takes, where 512 or more remain (200000 x 64
    // f32 in two groups, 512 chunks and 2048: 76 and 89 us; 32768 x 512 in one, 32, 256 and
    // 1024 chunks: 162, 71 and 73; 50000 x 2048 in one, 8, 64 and 256: 1143, 311 and 282)
    const int64_t chunks = std::min({most, want, std::max<int64_t>({1, kJoin / D, (512 + N * q.tiles - 1) / (N * q.tiles)})});
    q.chunk = (int)((S + chunks - 1) / chunks);
    q.chunks = (int)((S + q.chunk - 1) / q.chunk);
    // joined by a workgroup for every kJoin channels of chunks of a group
    q.span = (int)std::min<int64_t>(q.chunks, std::max<int64_t>(1, kJoin / D));
    q.spans = (q.chunks + q.span - 1) / q.span;
    size_t at = up256(8 * (size_t)(N * q.chunks) * C);
    q.o_stats = at;
    if (!bwd) at += up256(8 * (size_t)(N * a.groups));
    q.o_sums = at;
    if (bwd) at += up256(8 * (size_t)(N * a.groups));
    q.o_joined = at;
    if (q.spans > 1) at += up256(8 * (size_t)(N * a.groups) * q.spans);
    q.bytes = at;
    return q;
}

const char *check(const gdn2_group_norm_args &a, bool *nothing, bool *limits) {
    *nothing = *limits = false;
    if (a.samples < 0 || a.rows < 0 || a.channels < 0 || a.groups < 0) return "negative dimension";
    if (a.activation < GDN2_ACT_NONE || a.activation > GDN2_ACT_GELU) return "unknown activation";
    if (!(a.eps >= 0.0) || !std::isfinite(a.eps)) return "eps must be finite and not negative";
    if (a.groups == 0 ? a.channels != 0 : a.channels % a.groups != 0) return "channels must be a multiple of groups";
    if (a.samples == 0 || a.rows == 0 || a.channels == 0) {
        *nothing = true;
        return nullptr;
    }
    const int64_t most = int64_t(1) << 30;
    // 2^24 workgroups of 256 threads, and 2^16 of them along the channels
    if (a.channels >= (1 << 24) || a.samples >= most || a.rows >= most || a.samples * a.groups >= (1 << 24) ||
        a.samples >= (1 << 24)) {
        *limits = true;
        return "sizes above the kernels' limits";
    }
    return nullptr;
}

bool mult4(int64_t s) { return s % 4 == 0; }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A dimension of one has no stride to speak of.
gdn2_group_norm_args tidy(gdn2_group_norm_args a) {
    if (a.samples == 1) a.stride_x_n = a.stride_gate_n = 0;
    if (a.rows == 1) a.stride_x_s = a.stride_gate_s = 0;
    return a;
}

template <typename T> bool can_vec(const gdn2_group_norm_args &a) {
    const size_t e = 4 * sizeof(T);
    return aligned(a.x, e) && aligned(a.gate, e) && aligned(a.y, e) && aligned(a.weight, 16) && aligned(a.bias, 16) &&
           mult4(a.stride_x_n) && mult4(a.stride_x_s) && (!a.gate || (mult4(a.stride_gate_n) && mult4(a.stride_gate_s)));
}

GroupNormParams fill(const gdn2_group_norm_args &a, const Plan &q, void *ws) {
    GroupNormParams p{};
    p.x = a.x; p.gate = a.gate; p.weight = a.weight; p.bias = a.bias; p.y = a.y; p.stats = a.stats;
    p.sxn = a.stride_x_n; p.sxs = a.stride_x_s; p.sgn = a.stride_gate_n; p.sgs = a.stride_gate_s;
    p.N = a.samples; p.S = a.rows; p.C = (int)a.channels; p.G = (int)a.groups; p.D = p.C / p.G;
    p.act = a.activation; p.eps = (float)a.eps;
    p.sets = q.sets; p.log_l = q.log_l; p.row_blocks = q.row_blocks; p.lc = q.lc; p.chunks = q.chunks; p.chunk = q.chunk;
    p.spans = q.spans; p.span = q.span;
    char *w = static_cast<char *>(ws);
    if (q.bytes) p.part = reinterpret_cast<float *>(w);
    if (q.spans > 1) p.joined = reinterpret_cast<float *>(w + q.o_joined);
    if (q.held) {
        p.tile = q.tile; p.tiles = q.tiles; p.set_groups = q.set_groups;
        if (q.words) {
            p.words = reinterpret_cast<unsigned long long *>(w + q.o_words);
            p.patience = g_patience.load(std::memory_order_relaxed);
        }
        if (q.o_words == 0) p.part = nullptr;
    }
    return p;
}

template <typename T, int VEC, bool GATE> hipError_t run_rows(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    const dim3 grid((unsigned)((p.N + 4 * q.u - 1) / (4 * q.u) * q.sets));
    if (q.nv == 1) hipLaunchKernelGGL((norm_rows_kernel<T, VEC, 1, 4, GATE>), grid, dim3(256), 0, s, p);
    else if (q.nv == 4) hipLaunchKernelGGL((norm_rows_kernel<T, VEC, 4, 1, GATE>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((norm_rows_kernel<T, VEC, 16, 1, GATE>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}
template <typename T, int VEC, bool GATE> hipError_t run_rows_bwd(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    const dim3 grid((unsigned)(q.row_blocks * q.sets));
    if (q.nv == 1) hipLaunchKernelGGL((norm_rows_bwd_kernel<T, VEC, 1, 2, GATE>), grid, dim3(256), 0, s, p);
    else if (q.nv == 4) hipLaunchKernelGGL((norm_rows_bwd_kernel<T, VEC, 4, 1, GATE>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((norm_rows_bwd_kernel<T, VEC, VEC == 4 ? 8 : 16, 1, GATE>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

template <typename T, int VEC, int E, bool GATE, bool BWD> void launch_held(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    const dim3 grid((unsigned)(p.N * q.sets * q.chunks * q.tiles));
    if constexpr (BWD) hipLaunchKernelGGL((norm_held_bwd_kernel<T, VEC, E, GATE>), grid, dim3(NT), 0, s, p);
    else hipLaunchKernelGGL((norm_held_kernel<T, VEC, E, GATE>), grid, dim3(NT), 0, s, p);
}
template <typename T, int VEC, bool GATE, bool BWD> hipError_t run_held(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    if (q.words) {
        const int64_t n16 = q.words / 16;
        hipLaunchKernelGGL(norm_prepare_kernel, dim3((unsigned)std::min<int64_t>((n16 + 255) / 256, 1024)), dim3(256), 0, s,
                           reinterpret_cast<uint4 *>(p.words), n16);
    }
    if (q.e == 4) launch_held<T, VEC, 4, GATE, BWD>(q, p, s);
    else if (q.e == 8) launch_held<T, VEC, 8, GATE, BWD>(q, p, s);
    else launch_held<T, VEC, BWD ? kRows3Bwd : kRows3, GATE, BWD>(q, p, s);
    return hipGetLastError();
}

gdn2_status refuse(const char *who, const char *what, gdn2_status st = GDN2_EINVAL) {
    return fail(st, std::string(who) + ": " + what);
}

template <typename T, int VEC> hipError_t run_forward(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    if (q.rows) return p.gate ? run_rows<T, VEC, true>(q, p, s) : run_rows<T, VEC, false>(q, p, s);
    if (q.held) return p.gate ? run_held<T, VEC, true, false>(q, p, s) : run_held<T, VEC, false, false>(q, p, s);
    const dim3 grid((unsigned)(p.N * q.chunks), (unsigned)q.tiles);
    hipLaunchKernelGGL((norm_moments_kernel<T, VEC>), grid, dim3(256), 0, s, p);
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(p.N * p.G), (unsigned)q.spans), dim3(256), 0, s, p);
    if (q.spans > 1) hipLaunchKernelGGL(norm_join_spans_kernel, dim3((unsigned)(p.N * p.G)), dim3(kWave), 0, s, p);
    if (p.gate) hipLaunchKernelGGL((norm_apply_kernel<T, VEC, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((norm_apply_kernel<T, VEC, false>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}
template <typename T, int VEC, bool GATE> hipError_t run_backward(const Plan &q, const GroupNormParams &p, hipStream_t s) {
    const bool sums = p.dweight || p.dbias;
    int64_t blocks = q.row_blocks;
    if (q.rows) {
        if (const hipError_t e = run_rows_bwd<T, VEC, GATE>(q, p, s); e != hipSuccess) return e;
    } else if (q.held) {
        if (const hipError_t e = run_held<T, VEC, GATE, true>(q, p, s); e != hipSuccess) return e;
        blocks = p.N * q.chunks;
    } else {
        const dim3 grid((unsigned)(p.N * q.chunks), (unsigned)q.tiles);
        hipLaunchKernelGGL((norm_bwd_sums_kernel<T, VEC, GATE>), grid, dim3(256), 0, s, p);
        hipLaunchKernelGGL(norm_bwd_join_kernel, dim3((unsigned)(p.N * p.G), (unsigned)q.spans), dim3(256), 0, s, p);
        if (q.spans > 1) hipLaunchKernelGGL(norm_bwd_join_spans_kernel, dim3((unsigned)(p.N * p.G)), dim3(kWave), 0, s, p);
        hipLaunchKernelGGL((norm_bwd_apply_kernel<T, VEC, GATE>), grid, dim3(256), 0, s, p);
        blocks = p.N * q.chunks;
    }
    if (sums)
        hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((2 * (int64_t)p.C + 15) / 16)), dim3(256), 0, s, p.part, blocks,
                           p.C, p.dweight, p.dbias);
    return hipGetLastError();
}

bool grid_fits(const gdn2_group_norm_args &a, const Plan &q) {
    if (q.rows) return (double)((a.samples + 3) / 4) * q.sets < 16777216.0;
    if (q.held) return (double)a.samples * q.sets * q.chunks * q.tiles < 16777216.0;
    return (double)a.samples * q.chunks < 16777216.0 && q.tiles < 65536;
}

template <typename T> gdn2_status forward(const char *who, const gdn2_group_norm_args *args, hipStream_t s) {
    if (!args) return refuse(who, "null args");
    const gdn2_group_norm_args tidied = tidy(*args), *const a = &tidied;
    bool nothing, limits;
    if (const char *e = check(*a, &nothing, &limits)) return refuse(who, e, limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL);
    if (nothing) {
        if (!a->stats || a->samples == 0 || a->groups == 0) return GDN2_OK;
        if (a->samples >= (1 << 24) || a->groups >= (1 << 24) || a->samples * a->groups >= (1 << 24))
            return refuse(who, "sizes above the kernels' limits", GDN2_NOT_APPLICABLE);
        const int64_t n = 2 * a->samples * a->groups;
        hipLaunchKernelGGL(norm_no_stats_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a->stats, n);
        GDN2_HIP_CHECK(hipGetLastError());
        return GDN2_OK;
    }
    if (!a->x || !a->y) return refuse(who, "null tensor pointer");
    if (a->y == a->gate && (a->stride_gate_n != a->stride_x_n || a->stride_gate_s != a->stride_x_s))
        return refuse(who, "y may be gate only with x's strides");
    const Plan q = plan_of(*a, false, can_vec<T>(*a), false, a->y == a->x || a->y == a->gate);
    if (!grid_fits(*a, q)) return refuse(who, "sizes above the kernels' limits", GDN2_NOT_APPLICABLE);
    if (q.bytes > 0 && (!a->workspace || a->workspace_bytes < q.bytes || !aligned(a->workspace, 256)))
        return refuse(who, "workspace missing, too small or not 256-byte aligned");
    GroupNormParams p = fill(*a, q, a->workspace);
    if (!q.rows && !q.held && !p.stats) p.stats = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + q.o_stats);
    GDN2_HIP_CHECK((q.vec == 4 ? run_forward<T, 4>(q, p, s) : run_forward<T, 1>(q, p, s)));
    return GDN2_OK;
}

template <typename T> gdn2_status backward(const char *who, const gdn2_group_norm_bwd_args *a, hipStream_t s) {
    if (!a) return refuse(who, "null args");
    const gdn2_group_norm_args f = tidy(a->fwd);
    bool nothing, limits;
    if (const char *e = check(f, &nothing, &limits)) return refuse(who, e, limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL);
    if (!nothing) {
        if (!f.x || !f.stats || !a->d_y || !a->dx) return refuse(who, "null tensor pointer");
        if (!f.gate != !a->dgate) return refuse(who, "dgate must be given exactly where gate is");
        for (const void *in : {f.x, f.gate})
            if (in && (a->dx == in || a->dgate == in)) return refuse(who, "dx and dgate must not be inputs");
        if (a->dgate && (a->dgate == a->d_y || a->dgate == a->dx)) return refuse(who, "dgate must not be another operand");
    }
    const bool sums = a->dweight || a->dbias;
    if (nothing) { // no rows: zero gradients of the weights
        if (sums && f.channels > 0) {
            if (f.channels >= (1 << 24)) return refuse(who, "sizes above the kernels' limits", GDN2_NOT_APPLICABLE);
            hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((2 * f.channels + 15) / 16)), dim3(256), 0, s, nullptr,
                               (int64_t)0, (int)f.channels, a->dweight, a->dbias);
            GDN2_HIP_CHECK(hipGetLastError());
        }
        return GDN2_OK;
    }
    const size_t e = 4 * sizeof(T);
    const bool vec4 = can_vec<T>(f) && aligned(a->d_y, e) && aligned(a->dx, e) && aligned(a->dgate, e);
    const Plan q = plan_of(f, true, vec4, sums, a->dx == a->d_y);
    if (!grid_fits(f, q)) return refuse(who, "sizes above the kernels' limits", GDN2_NOT_APPLICABLE);
    if (q.bytes > 0 && (!a->workspace || a->workspace_bytes < q.bytes || !aligned(a->workspace, 256)))
        return refuse(who, "workspace missing, too small or not 256-byte aligned");
    GroupNormParams p = fill(f, q, a->workspace);
    p.dy = a->d_y; p.y = a->dx; p.dgate = a->dgate; p.dweight = a->dweight; p.dbias = a->dbias;
    p.sums = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + q.o_sums);
    if (f.gate)
        GDN2_HIP_CHECK((q.vec == 4 ? run_backward<T, 4, true>(q, p, s) : run_backward<T, 1, true>(q, p, s)));
    else
        GDN2_HIP_CHECK((q.vec == 4 ? run_backward<T, 4, false>(q, p, s) : run_backward<T, 1, false>(q, p, s)));
    return GDN2_OK;
}

// (of either alignment, in place or not: the call knows them, the size does not)
size_t workspace_of(const gdn2_group_norm_args *a, bool bwd) {
    bool nothing, limits;
    if (!a || check(*a, &nothing, &limits) || nothing) return 0;
    size_t n = 0;
    for (const bool vec4 : {true, false})
        for (const bool in_place : {true, false}) n = std::max(n, plan_of(*a, bwd, vec4, true, in_place).bytes);
    return n;
}

// No exception leaves a C entry.
template <typename F> gdn2_status guarded(F f) {
    try {
        return f();
    } catch (const std::exception &) {
        return GDN2_EHIP;
    }
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" size_t gdn2_group_norm_act_workspace_bytes(const gdn2_group_norm_args *a) { return workspace_of(a, false); }
extern "C" size_t gdn2_group_norm_act_bwd_workspace_bytes(const gdn2_group_norm_bwd_args *a) {
    return a ? workspace_of(&a->fwd, true) : 0;
}
extern "C" gdn2_status gdn2_group_norm_act_f32(const gdn2_group_norm_args *a, gdn2_stream_t s) {
    return guarded([&] { return forward<float>("gdn2_group_norm_act_f32", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_group_norm_act_bf16(const gdn2_group_norm_args *a, gdn2_stream_t s) {
    return guarded([&] { return forward<bf16>("gdn2_group_norm_act_bf16", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_group_norm_act_bwd_f32(const gdn2_group_norm_bwd_args *a, gdn2_stream_t s) {
    return guarded([&] { return backward<float>("gdn2_group_norm_act_bwd_f32", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_group_norm_act_bwd_bf16(const gdn2_group_norm_bwd_args *a, gdn2_stream_t s) {
    return guarded([&] { return backward<bf16>("gdn2_group_norm_act_bwd_bf16", a, (hipStream_t)s); });
}
extern "C" int gdn2_group_norm_patience(int looks) { return g_patience.exchange(std::max(looks, 0), std::memory_order_relaxed); }
