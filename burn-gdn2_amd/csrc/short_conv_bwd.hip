// gdn2_short_conv_bwd_f32: the gradients of gdn2_short_conv_f32.
//   z_t = sum_i xpad[t + i] w_i,  out = silu(z),  xpad = cat(cache or 3 copies of x_0, x)
//   dz = dy silu'(z),  dxpad[j] = sum_i dz[j - i] w_i (+ d_cache[j - T] for j >= T),
//   dw_i = sum_t dz_t xpad[t + i]
// A thread walks R tokens of VEC channels with the last rows of xpad and dz in
// registers; the three tokens behind its run, whose dz its last outputs need, it
// computes again (x and dy from cache).  dw goes to a sum a workgroup, then to
// one over the workgroups in a fixed order.
//
// Bound: HBM, 12 bytes an element: 4 x 2048 x 2048 0.20 GB in 43.4 us (4.6 TB/s),
// 40 of them the walk (5.0) and 4 the second sum.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2.h"
#include "vec_io.hpp"

namespace gdn2 {
namespace {

constexpr int kCache = 3;
constexpr int kStep = 2; // tokens whose rows are loaded together (1 to 4 of 16 bytes, 2 to 4 of 8: all 44 to 45 us)

struct ConvGradParams {
    const float *x, *w, *cache, *dy, *dcache;
    float *dx, *dcache_in;
    float *part; // [B * blocks][C][4]
    int64_t T, C;
    int blocks, run; // workgroups along a sequence, tokens a wave
};

template <int VEC> __global__ __launch_bounds__(256) void short_conv_bwd_kernel(ConvGradParams p) {
    __shared__ floatx4 red[4][VEC][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t c0 = ((int64_t)blockIdx.y * kWave + lane) * VEC;
    const bool ok = c0 < p.C; // (VEC divides C)
    const int64_t c = ok ? c0 : 0, b = blockIdx.x / p.blocks;
    const int64_t t0 = ((int64_t)(blockIdx.x % p.blocks) * 4 + wave) * p.run, t1 = min(t0 + p.run, p.T);
    const float *x = p.x + b * p.T * p.C + c, *dy = p.dy + b * p.T * p.C + c;
    float *dx = p.dx + b * p.T * p.C + c;
    const float *cache = p.cache ? p.cache + b * kCache * p.C + c : nullptr;
    const float *dc = p.dcache ? p.dcache + b * kCache * p.C + c : nullptr;
    float w[VEC][4];
#pragma unroll
    for (int j = 0; j < VEC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = p.w[(c + j) * 4 + i];

    // rows from one in memory in any case; those past the end count for nothing
    auto row = [&](const float *a, int64_t t, float *v) { load_n<float, VEC>(a + min(t, p.T - 1) * p.C, v); };
    auto pad = [&](int64_t j, float *v) { // xpad[j]
        if (j >= kCache) row(x, j - kCache, v);
        else if (cache) load_n<float, VEC>(cache + j * p.C, v);
        else load_n<float, VEC>(x, v);
    };
    float xw[3][VEC], dz[3][VEC], dw[VEC][4]; // xpad[t .. t + 2]; dz of t - 1, t - 2, t - 3
#pragma unroll
    for (int j = 0; j < VEC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dw[j][i] = 0.f;
            if (i < 3) dz[i][j] = 0.f;
        }
    // token t with its rows of x and dy; own: of this run (its share of dw).  Leaves
    // dx of token t - 3 in out.
    auto token = [&](int64_t t, bool own, const float *xt, const float *dyt, float *out) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float z = __builtin_fmaf(xw[0][j], w[j][0], __builtin_fmaf(xw[1][j], w[j][1],
                            __builtin_fmaf(xw[2][j], w[j][2], xt[j] * w[j][3])));
            const float s = __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z)); // (within one unit in the last place)
            const float d = t < p.T ? dyt[j] * (s * __builtin_fmaf(z, 1.f - s, 1.f)) : 0.f;
            out[j] = __builtin_fmaf(d, w[j][0], __builtin_fmaf(dz[0][j], w[j][1],
                     __builtin_fmaf(dz[1][j], w[j][2], dz[2][j] * w[j][3])));
            const float o = own ? d : 0.f;
            dw[j][0] = __builtin_fmaf(o, xw[0][j], dw[j][0]);
            dw[j][1] = __builtin_fmaf(o, xw[1][j], dw[j][1]);
            dw[j][2] = __builtin_fmaf(o, xw[2][j], dw[j][2]);
            dw[j][3] = __builtin_fmaf(o, xt[j], dw[j][3]);
            dz[2][j] = dz[1][j];
            dz[1][j] = dz[0][j];
            dz[0][j] = d;
            xw[0][j] = xw[1][j];
            xw[1][j] = xw[2][j];
            xw[2][j] = xt[j];
        }
    };
    if (t0 < t1) {
        float xp[3][VEC], gp[3][VEC], xn[kStep][VEC], gn[kStep][VEC], out[VEC];
        auto load = [&](int64_t s0) { // the rows of tokens s0 + 3 .. s0 + 3 + kStep: outputs s0 ..
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                row(x, s0 + 3 + i, xn[i]);
                row(dy, s0 + 3 + i, gn[i]);
            }
        };
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            pad(t0 + i, xw[i]);
            row(x, t0 + i, xp[i]);
            row(dy, t0 + i, gp[i]);
        }
        load(t0);
        float first[VEC]; // dxpad[0 .. 2] where the run starts the sequence
#pragma unroll
        for (int j = 0; j < VEC; ++j) first[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            token(t0 + i, t0 + i < t1, xp[i], gp[i], out);
            if (t0 == 0) {
                if (dc && i >= p.T) {
                    float e[VEC];
                    load_n<float, VEC>(dc + (i - p.T) * p.C, e);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) out[j] += e[j];
                }
                if (cache) {
                    if (p.dcache_in && ok) store_n<float, VEC>(p.dcache_in + (b * kCache + i) * p.C + c, out);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) first[j] += out[j];
                }
            }
        }
        for (int64_t s0 = t0; s0 < t1; s0 += kStep) {
            float xs[kStep][VEC], gs[kStep][VEC];
#pragma unroll
            for (int i = 0; i < kStep; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) xs[i][j] = xn[i][j], gs[i][j] = gn[i][j];
            load(s0 + kStep); // in flight beside this step
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                const int64_t s = s0 + i;
                token(s + 3, s + 3 < t1, xs[i], gs[i], out);
                if (s >= t1) continue;
                if (dc && s + 3 >= p.T) {
                    float e[VEC];
                    load_n<float, VEC>(dc + (s + 3 - p.T) * p.C, e);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) out[j] += e[j];
                }
                if (s == 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) out[j] += first[j];
                }
                if (ok) stream_n<float, VEC>(dx + s * p.C, out);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) red[wave][j][lane] = floatx4{dw[j][0], dw[j][1], dw[j][2], dw[j][3]};
    __syncthreads();
    if (wave == 0 && ok) {
        floatx4 *out = reinterpret_cast<floatx4 *>(p.part) + (int64_t)blockIdx.x * p.C + c;
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = (red[0][j][lane] + red[1][j][lane]) + (red[2][j][lane] + red[3][j][lane]);
    }
}

// Sums over `blocks` rows of n columns; a workgroup takes 16 columns, 16 threads each,
// which sum in 64 bits: there may be tens of thousands of rows.
__global__ __launch_bounds__(256) void conv_weight_sum_kernel(const float *part, int64_t blocks, int64_t n, float *out) {
    __shared__ double red[16][17];
    const int col = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int64_t i = (int64_t)blockIdx.x * 16 + col;
    double sum = 0.;
    if (i < n)
#pragma unroll 4
        for (int64_t b = r; b < blocks; b += 16) sum += part[b * n + i];
    red[r][col] = sum;
    __syncthreads();
    if (r == 0 && i < n) {
        sum = 0.;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += red[k][col];
        out[i] = (float)sum;
    }
}

__global__ __launch_bounds__(256) void copy_cache_kernel(const float *in, float *out, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = in ? in[i] : 0.f;
}

struct ConvPlan {
    int vec, run;
    int64_t blocks, tiles;
    size_t bytes;
};
ConvPlan plan_of(int64_t B, int64_t T, int64_t C, bool vec4) {
    ConvPlan q{};
    q.vec = vec4 && C % 4 == 0 ? 4 : 1;
    q.tiles = (C + kWave * q.vec - 1) / (kWave * q.vec);
    // a wave's run: up to 32 tokens (3 of 35 computed twice; 16: 47.7 against 44 us)
    // while 2048 waves, eight a compute unit, remain (64: 30 against 26 us at 2 x 3000
    // x 1537)
    q.run = 32;
    while (q.run > 8 && B * q.tiles * ((T + q.run - 1) / q.run) < 2048) q.run -= 8;
    q.blocks = (T + 4 * q.run - 1) / (4 * q.run);
    q.bytes = (sizeof(float) * 4 * (size_t)(B * q.blocks) * C + 255) & ~(size_t)255;
    return q;
}
bool sizes_ok(int64_t B, int64_t T, int64_t C) {
    const double el = (double)B * (double)T * (double)C;
    return B < (1 << 24) && C < (1 << 22) && T < (int64_t(1) << 40) && el < 1e15 && (double)B * ((double)T / 32 + 1) < 16777216.0;
}

bool overlaps(const void *a, const void *b, size_t n) {
    const char *p = static_cast<const char *>(a), *q = static_cast<const char *>(b);
    return p < q + n && q < p + n;
}

gdn2_status run(const float *x, const float *weight, const float *cache_in, const float *d_out, const float *d_cache_out,
                float *dx, float *dweight, float *d_cache_in, int64_t B, int64_t T, int64_t C, void *workspace,
                size_t workspace_bytes, hipStream_t s) {
    const std::string who = "gdn2_short_conv_bwd_f32: ";
    if (B < 0 || T < 0 || C < 0) return fail(GDN2_EINVAL, who + "negative dimension");
    if (C == 0) return GDN2_OK;
    if (!dweight || (B > 0 && T > 0 && (!x || !weight || !d_out || !dx))) return fail(GDN2_EINVAL, who + "null pointer");
    if (d_cache_in && !cache_in) return fail(GDN2_EINVAL, who + "d_cache_in without cache_in");
    if (!sizes_ok(B, T, C)) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    if (B == 0 || T == 0) { // no tokens: the cache passes through
        hipLaunchKernelGGL(conv_weight_sum_kernel, dim3((unsigned)((4 * C + 15) / 16)), dim3(256), 0, s, nullptr, (int64_t)0,
                           4 * C, dweight);
        const int64_t n = B * kCache * C;
        if (n > 0 && d_cache_in && d_cache_in != d_cache_out)
            hipLaunchKernelGGL(copy_cache_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, d_cache_out, d_cache_in, n);
        GDN2_HIP_CHECK(hipGetLastError());
        return GDN2_OK;
    }
    const size_t nx = sizeof(float) * (size_t)(B * T) * C;
    if (overlaps(dx, x, nx) || overlaps(dx, d_out, nx)) return fail(GDN2_EINVAL, who + "dx must not overlap x or d_out");
    const size_t nc = sizeof(float) * (size_t)(B * kCache) * C;
    if (d_cache_in && (overlaps(d_cache_in, cache_in, nc) || (d_cache_out && overlaps(d_cache_in, d_cache_out, nc))))
        return fail(GDN2_EINVAL, who + "d_cache_in must not overlap cache_in or d_cache_out");
    uintptr_t bits = 0;
    for (const void *q : {(const void *)x, (const void *)cache_in, (const void *)d_out, (const void *)d_cache_out,
                          (const void *)dx, (const void *)d_cache_in})
        bits |= reinterpret_cast<uintptr_t>(q);
    const ConvPlan q = plan_of(B, T, C, bits % 16 == 0);
    if (!workspace || workspace_bytes < q.bytes || reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(GDN2_EINVAL, who + "workspace missing, too small or not 256-byte aligned");
    if ((double)B * q.blocks >= 16777216.0 || q.tiles >= 65536)
        return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    ConvGradParams p{};
    p.x = x; p.w = weight; p.cache = cache_in; p.dy = d_out; p.dcache = d_cache_out; p.dx = dx; p.dcache_in = d_cache_in;
    p.part = static_cast<float *>(workspace);
    p.T = T; p.C = C; p.blocks = (int)q.blocks; p.run = q.run;
    const dim3 grid((unsigned)(B * q.blocks), (unsigned)q.tiles);
    if (q.vec == 4) hipLaunchKernelGGL(short_conv_bwd_kernel<4>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(short_conv_bwd_kernel<1>, grid, dim3(256), 0, s, p);
    hipLaunchKernelGGL(conv_weight_sum_kernel, dim3((unsigned)((4 * C + 15) / 16)), dim3(256), 0, s, p.part, B * q.blocks, 4 * C,
                       dweight);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_short_conv_bwd_workspace_bytes(int64_t B, int64_t T, int64_t C) {
    if (B <= 0 || T <= 0 || C <= 0 || !gdn2::sizes_ok(B, T, C)) return 0;
    return std::max(gdn2::plan_of(B, T, C, true).bytes, gdn2::plan_of(B, T, C, false).bytes);
}

extern "C" gdn2_status gdn2_short_conv_bwd_f32(const float *x, const float *weight, const float *cache_in,
                                               const float *d_out, const float *d_cache_out, float *dx, float *dweight,
                                               float *d_cache_in, int64_t B, int64_t T, int64_t C, void *workspace,
                                               size_t workspace_bytes, gdn2_stream_t stream) {
    try { // no exception leaves a C entry
        return gdn2::run(x, weight, cache_in, d_out, d_cache_out, dx, dweight, d_cache_in, B, T, C, workspace,
                         workspace_bytes, (hipStream_t)stream);
    } catch (const std::exception &) {
        return GDN2_EHIP;
    }
}
