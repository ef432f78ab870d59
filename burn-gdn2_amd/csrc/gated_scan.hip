// gdn2_gated_scan_*: h_t = e^{g_t} h_{t-1} + u_t, u = w v, per channel, and its
// adjoint, in one pass over the data.
//
// A run of tokens acts on the state that enters it as h -> e^G h + X, with G
// the sum of its log decays and X what the run leaves of a zero state; two runs
// join as (G1, X1), (G2, X2) -> (G1 + G2, e^G2 X1 + X2).  A workgroup holds a
// tile of consecutive tokens by CH channels in registers, R tokens and VEC
// channels a thread, joins the threads' runs by lane shuffles and through LDS,
// gets the state entering the tile from the tiles before it, and writes h.
// The token that starts a sequence has G = -inf and u += e^g h0, so that
// nothing of the sequence before it, infinities and NaN included, comes through,
// and several sequences in a tile need no other care.  The adjoint is the same
// recurrence from the last token to the first,
//   D_t = dy_t + E_{t+1},  E_t = e^{g_t} D_t,  dv = w D, dw = v D, dg_t = E_t h_{t-1}.
//
// Decays above e^-0.34 are kept as expm1(g) and the state is advanced as
// h + (expm1(g) h + u): the error of a rounded e^g, the same at every token, would
// otherwise add up over the tokens that a slowly decaying state lives through.
//
// Tiles of one (row, CH channels) form a chain.  A tile publishes (G, X) once it
// is loaded, and its final state once it knows what enters it.  It looks at the
// TL tiles before it at once, takes the nearest final state among them and
// applies the (G, X) after it in order, which gives the same bits whichever of
// them that was.  Words carry their own readiness (all ones: not yet), so that no
// other memory has to be ordered with them.  A workgroup draws its tile's number
// when it starts: the tiles it waits for have then started too, and a tile
// publishes (G, X) without waiting for anything, so every wait ends.
//
// Bound: HBM, 16 bytes an element forward and 32 backward in f32.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2_mixer.h"
#include "vec_io.hpp"

namespace gdn2 {
namespace {

constexpr unsigned kNaN = 0x7FC00000u;

struct GatedScanParams {
    const float *g;
    const void *v, *w;
    const float *state_in;
    float *state_out; // forward: final states; backward: d_state0
    void *out;        // forward: written; backward: h, read
    const int *info;  // packed: the sequence of every token (-1: none), with a -1 before and after; else NULL
    const void *dy;
    const float *ds;
    float *dg;
    void *dv, *dw;
    float *dgp; // partial sums of dg over a unit's channel tiles, or NULL
    int64_t sgb, sgh, sgt, svb, svh, svt, sob, soh, sot;
    int T, H, V;
    int unit, units; // channels are tiled within runs of `unit`: the whole row, or a head
    unsigned tiles_c, chains;
    unsigned tiles_t;
    unsigned *tickets;
    unsigned *pre;           // [chain][tile][CH] final states
    unsigned long long *agg; // [chain][tile][CH] (G, X)
};

// A token's decay in a register.  Sign bit set: expm1(g), for -0.34 < g <= 0, by
// seven terms of its series (the rest is below 2^-26 of it).  Clear: e^g.
__device__ __forceinline__ float decay(float g) {
    float p = __builtin_fmaf(g, 1.f / 5040, 1.f / 720);
    p = __builtin_fmaf(p, g, 1.f / 120);
    p = __builtin_fmaf(p, g, 1.f / 24);
    p = __builtin_fmaf(p, g, 1.f / 6);
    p = __builtin_fmaf(p, g, 0.5f);
    p = __builtin_fmaf(p * g, g, g);
    return g > -0.34f && g <= 0.f ? -__builtin_fabsf(p) : fast_exp2(g * kLog2e);
}
// e^g s + u.  Nothing of s, an infinity or NaN either, passes an e^g of zero; an
// infinity passes any other.
__device__ __forceinline__ float advance(float c, float s, float u) {
    const int bits = __builtin_bit_cast(int, c);
    const float t = __builtin_fmaf(c, s, u);
    return bits == 0 ? u : bits < 0 ? s + (__builtin_isinf(s) ? u : t) : t;
}

// e^G h + X of a joined run.  e^G of a growing run can overflow where e^G h does not.
__device__ __forceinline__ float join(float G, float X, float h) {
    if (G > 80.f) {
        const float e = fast_exp2(G * (0.5f * kLog2e));
        return h == 0.f ? X : __builtin_fmaf(e * h, e, X);
    }
    const float e = fast_exp2(G * kLog2e);
    return e == 0.f ? X : __builtin_fmaf(e, h, X);
}

// A published word is never all ones.
__device__ __forceinline__ unsigned word(float x) { return x != x ? kNaN : __builtin_bit_cast(unsigned, x); }

template <typename W> __device__ __forceinline__ W peek(const W *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename W> __device__ __forceinline__ void publish(W *p, W v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// All ones over the chains' words, and the sequence of every token (a search of
// the offsets for each).
__global__ __launch_bounds__(256) void scan_prepare_kernel(uint4 *words, int64_t n16, const int *cu, int N, int T, int *info) {
    const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    for (int64_t i = i0; i < n16; i += step) words[i] = uint4{~0u, ~0u, ~0u, ~0u};
    if (!cu) return;
    for (int64_t i = i0; i < (int64_t)T + 2; i += step) {
        const int t = (int)i - 1;
        int lo = 0, hi = N + 1; // offsets [0, lo) are at most t, [hi, N + 1) are above
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (cu[mid] <= t) lo = mid + 1;
            else hi = mid;
        }
        info[i] = t >= 0 && t < T && lo <= N ? lo - 1 : -1;
    }
}

// States of sequences without tokens.
__global__ __launch_bounds__(256) void empty_states_kernel(const int *cu, int64_t N, int64_t n, const float *in, float *out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= N * n) return;
    const int64_t s = i / n;
    if (cu[s + 1] <= cu[s]) out[i] = in ? in[i] : 0.f;
}

template <typename T, int VEC, int LC, int R, int NW, bool BWD, bool HEAD, bool HASW>
__global__ __launch_bounds__(64 * NW) void gated_scan_kernel(GatedScanParams p) {
    constexpr int TL = 64 / LC, CH = LC * VEC, TT = TL * R * NW;
    __shared__ float tot[2][NW][CH]; // the waves' runs (G, X)
    __shared__ float enter[CH];
    __shared__ unsigned drawn;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cl = lane % LC, tl = lane / LC;

    const unsigned chain = blockIdx.x % p.chains;
    unsigned tile = 0;
    if (p.tiles_t > 1) {
        if (tid == 0) drawn = atomicAdd(p.tickets + chain, 1u) + 1u; // from all ones
        __syncthreads();
        tile = __builtin_amdgcn_readfirstlane(drawn);
    }
    const unsigned ct = chain % p.tiles_c;
    const unsigned bu = chain / p.tiles_c, b = bu / (unsigned)p.units, un = bu % (unsigned)p.units;
    const int in_unit = (int)ct * CH + cl * VEC; // (VEC divides V where it is not 1)
    const bool ok = in_unit < p.unit;
    const int ch = (int)un * p.unit + (ok ? in_unit : 0), h = ch / p.V, c = ch % p.V;

    const float *g = p.g + b * p.sgb + h * p.sgh + (HEAD ? 0 : c);
    const T *v = static_cast<const T *>(p.v) + b * p.svb + h * p.svh + c;
    const T *w = static_cast<const T *>(p.w) + b * p.svb + h * p.svh + c;
    const int64_t oo = b * p.sob + h * p.soh + c;

    // p0: the run's first token in the direction of the recurrence; token(i) its i-th
    const int p0 = (int)tile * TT + (wave * TL + tl) * R;
    auto token = [&](int i) { return BWD ? p.T - 1 - (p0 + i) : p0 + i; };

    // masks of the run's tokens: present, first of a sequence, last of one
    unsigned have = 0, first = 0, last = 0;
    int seq[R];
    if (p.info) {
        int near[R + 2]; // the tokens around and in the run, in its direction
#pragma unroll
        for (int i = 0; i < R + 2; ++i) {
            const int t = token(i - 1);
            near[i] = t >= -1 && t <= p.T ? p.info[t + 1] : -1;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            seq[i] = near[i + 1];
            const bool in = near[i + 1] >= 0;
            have |= (unsigned)in << i;
            first |= (unsigned)(in && near[BWD ? i + 2 : i] != near[i + 1]) << i;
            last |= (unsigned)(in && near[BWD ? i : i + 2] != near[i + 1]) << i;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            seq[i] = (int)b;
            have |= (unsigned)(p0 + i < p.T) << i;
            first |= (unsigned)(token(i) == 0) << i;
            last |= (unsigned)(token(i) == p.T - 1) << i;
        }
    }
    if (!ok) have = first = last = 0;
    auto state_at = [&](int n) { return ((int64_t)n * p.H + h) * p.V + c; };

    // All loads of the run, from a row of the tensor in any case (what an absent
    // token's row holds is dropped), so that they are in flight together.
    // Backward: u is dy, hb the state before the token.
    constexpr int GV = HEAD ? 1 : VEC;
    Raw<float, GV> rg[R];
    Raw<T, VEC> ru[R], rw[HASW ? R : 1], rv[BWD && HASW ? R : 1], rh[BWD ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t t = min(max(token(i), 0), p.T - 1);
        rg[i] = raw_n<float, GV>(g + t * p.sgt);
        if constexpr (!BWD) {
            ru[i] = raw_n<T, VEC>(v + t * p.svt);
        } else {
            ru[i] = raw_n<T, VEC>(static_cast<const T *>(p.dy) + oo + t * p.sot);
            rh[i] = raw_n<T, VEC>(static_cast<const T *>(p.out) + oo + max(t - 1, (int64_t)0) * p.sot);
            if constexpr (HASW) rv[i] = raw_n<T, VEC>(v + t * p.svt);
        }
        if constexpr (HASW) rw[i] = raw_n<T, VEC>(w + t * p.svt);
    }
    float em[R][GV], u[R][VEC];

    // the run
    float G[VEC], X[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) G[j] = X[j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const bool in = have >> i & 1;
        float g0 = 0.f;
        if constexpr (HEAD) em[i][0] = decay(g0 = in ? rg[i][0] : 0.f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            u[i][j] = (float)ru[i][j];
            if constexpr (HASW && !BWD) u[i][j] *= (float)rw[i][j];
            u[i][j] = in ? u[i][j] : 0.f;
        }
        const bool cut = (BWD ? last : first) >> i & 1; // nothing comes from the token before in this direction
        float s0[VEC]; // forward: the state before a sequence; backward: the gradient of the one after it
#pragma unroll
        for (int j = 0; j < VEC; ++j) s0[j] = 0.f;
        if (cut) {
            const float *s = BWD ? p.ds : p.state_in;
            if (s) load_n<float, VEC>(s + state_at(seq[i]), s0);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float gj = HEAD ? g0 : in ? rg[i][HEAD ? 0 : j] : 0.f;
            if constexpr (!HEAD) em[i][j] = decay(gj);
            const float dec = em[i][HEAD ? 0 : j];
            if constexpr (!BWD) {
                if (cut) u[i][j] = advance(dec, s0[j], u[i][j]);
                X[j] = cut ? u[i][j] : advance(dec, X[j], u[i][j]);
            } else {
                if (cut) u[i][j] += s0[j];
                X[j] = advance(dec, cut ? u[i][j] : u[i][j] + X[j], 0.f);
            }
            G[j] = cut ? -INFINITY : G[j] + gj;
        }
    }

    // runs before this one: in the wave ...
    float Gw[VEC], Xw[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) Gw[j] = G[j], Xw[j] = X[j];
#pragma unroll
    for (int o = 1; o < TL; o <<= 1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float Gp = __shfl_up(Gw[j], o * LC, 64), Xp = __shfl_up(Xw[j], o * LC, 64);
            if (tl >= o) {
                Xw[j] = join(Gw[j], Xw[j], Xp);
                Gw[j] = Gw[j] == -INFINITY ? -INFINITY : Gw[j] + Gp;
            }
        }
    }
    if (tl == TL - 1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            tot[0][wave][cl * VEC + j] = Gw[j];
            tot[1][wave][cl * VEC + j] = Xw[j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float Gp = __shfl_up(Gw[j], LC, 64), Xp = __shfl_up(Xw[j], LC, 64);
        Gw[j] = tl ? Gp : 0.f;
        Xw[j] = tl ? Xp : 0.f;
    }
    __syncthreads();

    // ... and before the tile
    if (p.tiles_t > 1) {
        if (wave == 0) {
            const int64_t at = ((int64_t)chain * p.tiles_t + tile) * CH;
            float Gt[VEC], Xt[VEC], hin[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                Gt[j] = 0.f;
                Xt[j] = 0.f;
#pragma unroll
                for (int k = 0; k < NW; ++k) {
                    const float Gk = tot[0][k][cl * VEC + j], Xk = tot[1][k][cl * VEC + j];
                    Xt[j] = join(Gk, Xk, Xt[j]);
                    Gt[j] = Gk == -INFINITY ? -INFINITY : Gt[j] + Gk;
                }
                hin[j] = 0.f;
            }
            if (tl == 0 && tile + 1 < p.tiles_t) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    publish(p.agg + at + cl * VEC + j, (unsigned long long)word(Gt[j]) | (unsigned long long)word(Xt[j]) << 32);
            }
            if (tile > 0) {
                const bool there = (int)tile - 1 - tl >= 0;
                const int64_t from = at - (int64_t)(there ? tl + 1 : 0) * CH + cl * VEC;
                unsigned P[VEC];
                unsigned long long A[VEC];
                int nearest;
                for (;;) {
                    bool hasP = there, hasA = there;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        P[j] = peek(p.pre + from + j);
                        A[j] = peek(p.agg + from + j);
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        hasP = hasP && P[j] != ~0u;
                        hasA = hasA && A[j] != ~0ull;
                    }
                    const unsigned long long mp = __ballot(hasP) >> cl, ma = __ballot(hasA || hasP) >> cl;
                    nearest = -1;
                    bool all = true;
#pragma unroll
                    for (int k = 0; k < TL; ++k) {
                        if (nearest < 0 && all && (mp >> (k * LC) & 1)) nearest = k;
                        all = all && (ma >> (k * LC) & 1);
                    }
                    if (__all(nearest >= 0)) break;
                    __builtin_amdgcn_s_sleep(1);
                }
#pragma unroll
                for (int k = TL - 1; k >= 0; --k) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int src = k * LC + cl;
                        const float Pk = __builtin_bit_cast(float, (unsigned)__shfl((int)P[j], src, 64));
                        const float Gk = __builtin_bit_cast(float, (unsigned)__shfl((int)(unsigned)A[j], src, 64));
                        const float Xk = __builtin_bit_cast(float, (unsigned)__shfl((int)(unsigned)(A[j] >> 32), src, 64));
                        hin[j] = k > nearest ? 0.f : k == nearest ? Pk : join(Gk, Xk, hin[j]);
                    }
                }
            }
            if (tl == 0) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (tile + 1 < p.tiles_t) publish(p.pre + at + cl * VEC + j, word(join(Gt[j], Xt[j], hin[j])));
                    enter[cl * VEC + j] = hin[j];
                }
            }
        }
        __syncthreads();
    }

    float s[VEC]; // the state (or gradient) entering this thread's run
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        float x = p.tiles_t > 1 ? enter[cl * VEC + j] : 0.f;
        for (int k = 0; k < wave; ++k) x = join(tot[0][k][cl * VEC + j], tot[1][k][cl * VEC + j], x);
        s[j] = join(Gw[j], Xw[j], x);
    }

#pragma unroll
    for (int i = 0; i < R; ++i) {
        const bool in = have >> i & 1, cut = (BWD ? last : first) >> i & 1;
        const int64_t t = token(i);
        if constexpr (!BWD) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                s[j] = cut ? u[i][j] : advance(em[i][HEAD ? 0 : j], s[j], u[i][j]);
            }
            if (in) store_n<T, VEC>(static_cast<T *>(p.out) + oo + t * p.sot, s);
            if ((last >> i & 1) && p.state_out) store_n<float, VEC>(p.state_out + state_at(seq[i]), s);
        } else {
            float dg[VEC], dv[VEC], dw[VEC], hb[VEC]; // hb: the state before the token
#pragma unroll
            for (int j = 0; j < VEC; ++j) hb[j] = first >> i & 1 ? 0.f : (float)rh[i][j];
            if ((first >> i & 1) && p.state_in) load_n<float, VEC>(p.state_in + state_at(seq[i]), hb);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = cut ? u[i][j] : u[i][j] + s[j];
                s[j] = advance(em[i][HEAD ? 0 : j], d, 0.f);
                dg[j] = s[j] * hb[j];
                dv[j] = d;
                if constexpr (HASW) {
                    dv[j] *= (float)rw[i][j];
                    dw[j] = (float)rv[i][j] * d;
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) { // rows outside every sequence have no part in L
                dg[j] = in ? dg[j] : 0.f;
                dv[j] = in ? dv[j] : 0.f;
                if constexpr (HASW) dw[j] = in ? dw[j] : 0.f;
            }
            const bool row = ok && p0 + i < p.T;
            if (row) {
                store_n<T, VEC>(static_cast<T *>(p.dv) + (v - static_cast<const T *>(p.v)) + t * p.svt, dv);
                if constexpr (HASW)
                    store_n<T, VEC>(static_cast<T *>(p.dw) + (v - static_cast<const T *>(p.v)) + t * p.svt, dw);
                if constexpr (!HEAD) store_n<float, VEC>(p.dg + (g - p.g) + t * p.sgt, dg);
            }
            if ((first >> i & 1) && p.state_out) store_n<float, VEC>(p.state_out + state_at(seq[i]), s);
            if constexpr (HEAD) { // the tile's channels are of one head
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum += dg[j];
#pragma unroll
                for (int o = 1; o < LC; o <<= 1) sum += __shfl_xor(sum, o, 64);
                if (cl == 0 && row) {
                    if (p.dgp) p.dgp[(((int64_t)b * p.units + un) * p.T + t) * p.tiles_c + ct] = sum;
                    else p.dg[b * p.sgb + h * p.sgh + t * p.sgt] = sum;
                }
            }
        }
    }
}

// dg of a head from its channel tiles' sums.
__global__ __launch_bounds__(256) void dg_sum_kernel(GatedScanParams p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t t = i % p.T, h = i / p.T % p.H, b = i / p.T / p.H;
    float sum = 0.f;
    for (unsigned k = 0; k < p.tiles_c; ++k) sum += p.dgp[i * p.tiles_c + k];
    p.dg[b * p.sgb + h * p.sgh + t * p.sgt] = sum;
}

// A few tokens: a thread walks its channels through them.
template <typename T, int VEC, bool HEAD, bool HASW>
__global__ __launch_bounds__(256) void gated_step_kernel(GatedScanParams p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t e = i * VEC, c = e % p.V, h = e / p.V % p.H, b = e / p.V / p.H;
    const float *g = p.g + b * p.sgb + h * p.sgh + (HEAD ? 0 : c);
    const T *v = static_cast<const T *>(p.v) + b * p.svb + h * p.svh + c;
    const T *w = static_cast<const T *>(p.w) + b * p.svb + h * p.svh + c;
    T *out = static_cast<T *>(p.out) + b * p.sob + h * p.soh + c;
    float s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = 0.f;
    if (p.state_in) load_n<float, VEC>(p.state_in + e, s);
    for (int t = 0; t < p.T; ++t) {
        float x[VEC], y[VEC], gg[HEAD ? 1 : VEC];
        load_n<float, HEAD ? 1 : VEC>(g + t * p.sgt, gg);
        load_n<T, VEC>(v + t * p.svt, x);
        if constexpr (HASW) load_n<T, VEC>(w + t * p.svt, y);
        float dec = 0.f;
        if constexpr (HEAD) dec = decay(gg[0]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (!HEAD) dec = decay(gg[j]);
            s[j] = advance(dec, s[j], HASW ? x[j] * y[j] : x[j]);
        }
        store_n<T, VEC>(out + t * p.sot, s);
    }
    if (p.state_out) store_n<float, VEC>(p.state_out + e, s);
}

// -- host ---------------------------------------------------------------------

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr int kWalk = 8; // tokens that gated_step_kernel takes

struct Plan {
    bool vec, walk;
    int ch, tt;
    int unit, units;
    int64_t tiles_c, tiles_t, chains;
    size_t o_pre, o_agg, words, o_info, o_dgp, bytes; // workspace: tickets, pre, agg; the tokens' sequences; dg sums
};

Plan plan_of(const gdn2_gated_scan_args &a, bool bwd, bool vec) {
    Plan q{};
    q.vec = vec;
    const int64_t T = a.seq_len, HV = a.num_heads * a.head_v_dim;
    q.walk = !bwd && !a.cu_seqlens && T <= kWalk;
    if (q.walk) return q;
    q.ch = 32;
    q.tt = vec ? (bwd ? 128 : 256) : 64;
    const bool heads = bwd && a.g_per_head;
    q.unit = (int)(heads ? a.head_v_dim : HV);
    q.units = (int)(heads ? a.num_heads : 1);
    q.tiles_c = (q.unit + q.ch - 1) / q.ch;
    q.tiles_t = (T + q.tt - 1) / q.tt;
    q.chains = a.batch * q.units * q.tiles_c;
    size_t at = 0;
    if (q.tiles_t > 1) {
        at = up256(4 * (size_t)q.chains);
        q.o_pre = at;
        at += up256(4 * (size_t)(q.chains * q.tiles_t * q.ch));
        q.o_agg = at;
        at += up256(8 * (size_t)(q.chains * q.tiles_t * q.ch));
        q.words = at;
    }
    q.o_info = at;
    if (a.cu_seqlens) at += up256(4 * (size_t)(T + 2));
    q.o_dgp = at;
    if (heads && q.tiles_c > 1) at += up256(4 * (size_t)(a.batch * a.num_heads * T * q.tiles_c));
    q.bytes = at;
    return q;
}

const char *check(const gdn2_gated_scan_args &a, bool *nothing, bool *limits) {
    *nothing = *limits = false;
    if (a.batch < 0 || a.num_heads < 0 || a.seq_len < 0 || a.head_v_dim < 0 || a.num_seqs < 0) return "negative dimension";
    if (a.cu_seqlens && a.batch != 1) return "packed sequences need batch 1";
    if (a.batch == 0 || a.num_heads == 0 || a.head_v_dim == 0 || (a.cu_seqlens && a.num_seqs == 0)) {
        *nothing = true;
        return nullptr;
    }
    const int64_t most = int64_t(1) << 30;
    if (a.seq_len >= most || a.num_heads >= most || a.head_v_dim >= most || a.num_heads * a.head_v_dim >= most ||
        a.num_seqs >= most || a.batch >= most) {
        *limits = true;
        return "sizes above the kernels' limits";
    }
    // 2^24 workgroups of 256 threads; tiles hold 64 tokens by 32 channels at least
    const double N = (double)(a.cu_seqlens ? a.num_seqs : a.batch), HV = (double)a.num_heads * a.head_v_dim;
    const double tiles = (double)a.batch * a.num_heads * ((a.head_v_dim + 31) / 32) * ((a.seq_len + 63) / 64);
    if (tiles >= 16777216.0 || N * HV >= 4294967040.0 || (double)a.batch * a.num_heads * a.seq_len >= 4294967040.0) {
        *limits = true;
        return "sizes above the kernels' limits";
    }
    return nullptr;
}

bool mult(int64_t s, int64_t m) { return s % m == 0; }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T> bool can_vec(const gdn2_gated_scan_args &a) {
    const size_t e = 4 * sizeof(T);
    bool ok = a.head_v_dim % 4 == 0 && mult(a.stride_vw_b, 4) && mult(a.stride_vw_h, 4) && mult(a.stride_vw_t, 4) &&
              mult(a.stride_o_b, 4) && mult(a.stride_o_h, 4) && mult(a.stride_o_t, 4) && aligned(a.v, e) &&
              aligned(a.w, e) && aligned(a.out, e) && aligned(a.state_in, 16) && aligned(a.state_out, 16);
    if (!a.g_per_head)
        ok = ok && mult(a.stride_g_b, 4) && mult(a.stride_g_h, 4) && mult(a.stride_g_t, 4) && aligned(a.g, 16);
    return ok;
}

void fill(const gdn2_gated_scan_args &a, const Plan &q, void *workspace, GatedScanParams *p) {
    p->g = a.g; p->v = a.v; p->w = a.w; p->state_in = a.state_in; p->state_out = a.state_out; p->out = a.out;
    p->sgb = a.stride_g_b; p->sgh = a.stride_g_h; p->sgt = a.stride_g_t;
    p->svb = a.stride_vw_b; p->svh = a.stride_vw_h; p->svt = a.stride_vw_t;
    p->sob = a.stride_o_b; p->soh = a.stride_o_h; p->sot = a.stride_o_t;
    p->T = (int)a.seq_len; p->H = (int)a.num_heads; p->V = (int)a.head_v_dim;
    if (q.walk) return;
    p->unit = q.unit; p->units = q.units;
    p->tiles_c = (unsigned)q.tiles_c; p->chains = (unsigned)q.chains; p->tiles_t = (unsigned)q.tiles_t;
    char *ws = static_cast<char *>(workspace);
    if (q.tiles_t > 1) {
        p->tickets = reinterpret_cast<unsigned *>(ws);
        p->pre = reinterpret_cast<unsigned *>(ws + q.o_pre);
        p->agg = reinterpret_cast<unsigned long long *>(ws + q.o_agg);
    }
    if (a.cu_seqlens) p->info = reinterpret_cast<const int *>(ws + q.o_info);
}

template <typename T, bool BWD, bool HEAD, bool HASW>
hipError_t launch_tiles(const Plan &q, const GatedScanParams &p, hipStream_t s) {
    const dim3 grid((unsigned)(q.chains * q.tiles_t));
    if (q.vec) hipLaunchKernelGGL((gated_scan_kernel<T, 4, 8, BWD ? 4 : 8, 4, BWD, HEAD, HASW>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gated_scan_kernel<T, 1, 32, 8, 4, BWD, HEAD, HASW>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}
template <typename T, bool HEAD, bool HASW>
hipError_t launch_walk(const gdn2_gated_scan_args &a, const Plan &q, const GatedScanParams &p, hipStream_t s) {
    const int64_t n = a.batch * a.num_heads * a.head_v_dim / (q.vec ? 4 : 1);
    const dim3 grid((unsigned)((n + 255) / 256));
    if (q.vec) hipLaunchKernelGGL((gated_step_kernel<T, 4, HEAD, HASW>), grid, dim3(256), 0, s, p, n);
    else hipLaunchKernelGGL((gated_step_kernel<T, 1, HEAD, HASW>), grid, dim3(256), 0, s, p, n);
    return hipGetLastError();
}

hipError_t prepare(const gdn2_gated_scan_args &a, const Plan &q, void *ws, hipStream_t s) {
    if (q.words == 0 && !a.cu_seqlens) return hipSuccess;
    const int64_t n16 = (int64_t)(q.words / 16), n = std::max<int64_t>(n16, a.cu_seqlens ? a.seq_len + 2 : 0);
    const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 2048);
    hipLaunchKernelGGL(scan_prepare_kernel, dim3(blocks), dim3(256), 0, s, reinterpret_cast<uint4 *>(ws), n16, a.cu_seqlens,
                       (int)a.num_seqs, (int)a.seq_len, reinterpret_cast<int *>(static_cast<char *>(ws) + q.o_info));
    return hipGetLastError();
}

hipError_t empty_states(const gdn2_gated_scan_args &a, const float *in, float *out, hipStream_t s) {
    if (!a.cu_seqlens || !out) return hipSuccess;
    const int64_t n = a.num_heads * a.head_v_dim;
    hipLaunchKernelGGL(empty_states_kernel, dim3((unsigned)((a.num_seqs * n + 255) / 256)), dim3(256), 0, s, a.cu_seqlens,
                       a.num_seqs, n, in, out);
    return hipGetLastError();
}

gdn2_status bad_workspace(const char *who) {
    return fail(GDN2_EINVAL, std::string(who) + ": workspace missing, too small or not 256-byte aligned");
}

// The states of a call without tokens.
__global__ __launch_bounds__(256) void copy_states_kernel(const float *in, float *out, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = in ? in[i] : 0.f;
}

gdn2_status no_tokens(const gdn2_gated_scan_args &a, const float *in, float *out, hipStream_t s) {
    const int64_t n = (a.cu_seqlens ? a.num_seqs : a.batch) * a.num_heads * a.head_v_dim;
    if (!out || out == in) return GDN2_OK;
    hipLaunchKernelGGL(copy_states_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, in, out, n);
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

template <typename T> gdn2_status forward(const char *who, const gdn2_gated_scan_args *a, hipStream_t s) {
    if (!a) return fail(GDN2_EINVAL, std::string(who) + ": null args");
    bool nothing, limits;
    if (const char *e = check(*a, &nothing, &limits))
        return fail(limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL, std::string(who) + ": " + e);
    if (nothing) return GDN2_OK;
    if (a->seq_len == 0) return no_tokens(*a, a->state_in, a->state_out, s);
    if (!a->g || !a->v || !a->out) return fail(GDN2_EINVAL, std::string(who) + ": null tensor pointer");
    const Plan q = plan_of(*a, false, can_vec<T>(*a));
    if (q.bytes > 0 && (!a->workspace || a->workspace_bytes < q.bytes || !aligned(a->workspace, 256))) return bad_workspace(who);
    GatedScanParams p{};
    fill(*a, q, a->workspace, &p);
    if (q.walk) {
        GDN2_HIP_CHECK(a->g_per_head ? (a->w ? launch_walk<T, true, true>(*a, q, p, s) : launch_walk<T, true, false>(*a, q, p, s))
                                     : (a->w ? launch_walk<T, false, true>(*a, q, p, s) : launch_walk<T, false, false>(*a, q, p, s)));
        return GDN2_OK;
    }
    GDN2_HIP_CHECK(prepare(*a, q, a->workspace, s));
    GDN2_HIP_CHECK(a->g_per_head
                       ? (a->w ? launch_tiles<T, false, true, true>(q, p, s) : launch_tiles<T, false, true, false>(q, p, s))
                       : (a->w ? launch_tiles<T, false, false, true>(q, p, s) : launch_tiles<T, false, false, false>(q, p, s)));
    GDN2_HIP_CHECK(empty_states(*a, a->state_in, a->state_out, s));
    return GDN2_OK;
}

template <typename T> gdn2_status backward(const char *who, const gdn2_gated_scan_bwd_args *a, hipStream_t s) {
    if (!a) return fail(GDN2_EINVAL, std::string(who) + ": null args");
    const gdn2_gated_scan_args &f = a->fwd;
    bool nothing, limits;
    if (const char *e = check(f, &nothing, &limits))
        return fail(limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL, std::string(who) + ": " + e);
    if (nothing) return GDN2_OK;
    if (f.seq_len == 0) return no_tokens(f, a->d_state_out, a->d_state0, s);
    if (!f.g || !f.out || !a->d_out || !a->dg || !a->dv || (f.w && !f.v))
        return fail(GDN2_EINVAL, std::string(who) + ": null tensor pointer");
    if (!f.w != !a->dw) return fail(GDN2_EINVAL, std::string(who) + ": dw must be given exactly where w is");
    const size_t e = 4 * sizeof(T);
    const bool vec = can_vec<T>(f) && aligned(a->d_out, e) && aligned(a->dv, e) && aligned(a->dw, e) &&
                     aligned(a->d_state_out, 16) && aligned(a->d_state0, 16) && (f.g_per_head || aligned(a->dg, 16));
    const Plan q = plan_of(f, true, vec);
    if (q.bytes > 0 && (!a->workspace || a->workspace_bytes < q.bytes || !aligned(a->workspace, 256))) return bad_workspace(who);
    GatedScanParams p{};
    fill(f, q, a->workspace, &p);
    p.state_out = a->d_state0;
    p.dy = a->d_out; p.ds = a->d_state_out; p.dg = a->dg; p.dv = a->dv; p.dw = a->dw;
    if (f.g_per_head && q.tiles_c > 1) p.dgp = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + q.o_dgp);
    GDN2_HIP_CHECK(prepare(f, q, a->workspace, s));
    GDN2_HIP_CHECK(f.g_per_head
                       ? (f.w ? launch_tiles<T, true, true, true>(q, p, s) : launch_tiles<T, true, true, false>(q, p, s))
                       : (f.w ? launch_tiles<T, true, false, true>(q, p, s) : launch_tiles<T, true, false, false>(q, p, s)));
    if (p.dgp) {
        const int64_t n = f.batch * f.num_heads * f.seq_len;
        hipLaunchKernelGGL(dg_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, n);
        GDN2_HIP_CHECK(hipGetLastError());
    }
    GDN2_HIP_CHECK(empty_states(f, a->d_state_out, a->d_state0, s));
    return GDN2_OK;
}

size_t workspace_of(const gdn2_gated_scan_args *a, bool bwd) {
    bool nothing, limits;
    if (!a || check(*a, &nothing, &limits) || nothing || a->seq_len == 0) return 0;
    return std::max(plan_of(*a, bwd, true).bytes, plan_of(*a, bwd, false).bytes);
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

extern "C" size_t gdn2_gated_scan_workspace_bytes(const gdn2_gated_scan_args *a) { return workspace_of(a, false); }
extern "C" size_t gdn2_gated_scan_bwd_workspace_bytes(const gdn2_gated_scan_bwd_args *a) {
    return a ? workspace_of(&a->fwd, true) : 0;
}
extern "C" gdn2_status gdn2_gated_scan_fwd_f32(const gdn2_gated_scan_args *a, gdn2_stream_t s) {
    return guarded([&] { return forward<float>("gdn2_gated_scan_fwd_f32", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_gated_scan_fwd_bf16(const gdn2_gated_scan_args *a, gdn2_stream_t s) {
    return guarded([&] { return forward<bf16>("gdn2_gated_scan_fwd_bf16", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_gated_scan_bwd_f32(const gdn2_gated_scan_bwd_args *a, gdn2_stream_t s) {
    return guarded([&] { return backward<float>("gdn2_gated_scan_bwd_f32", a, (hipStream_t)s); });
}
extern "C" gdn2_status gdn2_gated_scan_bwd_bf16(const gdn2_gated_scan_bwd_args *a, gdn2_stream_t s) {
    return guarded([&] { return backward<bf16>("gdn2_gated_scan_bwd_bf16", a, (hipStream_t)s); });
}
