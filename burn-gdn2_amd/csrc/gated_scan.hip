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
// Decays above e^-1/8 are kept as expm1(g) and the state is advanced as
// h + (expm1(g) h + u): the error of a rounded e^g, the same at every token, would
// otherwise add up over the tokens that a slowly decaying state lives through.
//
// Tiles of one (row, CH channels) form a chain (a scan in a single pass, by decoupled
// look-back).  A tile publishes (G, X) once it
// is loaded, and its final state once it knows what enters it.  It looks at
// several tiles before it at once, takes the nearest final state among them and
// applies the (G, X) after it in order, which gives the same bits whichever of
// them that was.  Words carry their own readiness (all ones: not yet), so that no
// other memory has to be ordered with them.  A workgroup draws its tile's number
// when it is about to start on it: of the tiles that were drawn and are not
// finished, the one of the lowest number waits for none, so every wait ends.
//
// Bound: HBM, 16 bytes an element forward and 32 backward in f32.  (8 x 4096 x
// 2048 f32, decays per channel: 1.07 GB in 194 us, 5.5 TB/s, where torch's
// elementwise kernel of three reads and a write reaches 5.8; backward of 4 x 2048
// x 2048, 0.54 GB in 103 us, 5.2 TB/s.)  One packed row of bf16, decays
// per head, has few chains, and long ones: 65536 tokens 219 us (3.7 TB/s), of which
// waiting for the tiles before is 32; backward of 32767 187 us (4.3 TB/s), 9.
// Prepare beside them is 3 to 6 us.
#include <algorithm>
#include <exception>
#include <initializer_list>
#include <string>
#include <type_traits>

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
    const int *cu, *info; // packed: the N + 1 offsets; the sequence of every token (-1: none), a -1 before and after
    const void *dy;
    const float *ds;
    float *dg;
    void *dv, *dw;
    float *dgp; // partial sums of dg over a unit's channel tiles, or NULL
    int64_t sgb, sgh, sgt, svb, svh, svt, sob, soh, sot;
    int T, H, V, N;
    int unit, units; // channels are tiled within runs of `unit`: the whole row, or a head
    unsigned tiles_c, chains;
    unsigned tiles_t;
    unsigned *ticket; // the next tile
    unsigned *pre;           // [chain][tile][CH] final states
    unsigned long long *agg; // [chain][tile][CH] (G, X)
};

// A token's decay in a register.  Sign bit set: expm1(g), for -1/8 < g < 0, by
// four terms of its series (the rest is below 2^-24 of it).  Clear: e^g (of -0,
// too: its series ends in a zero whose sign says e^g).
__device__ __forceinline__ float decay(float g) {
    const float p = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(g, 1.f / 120, 1.f / 24), g, 1.f / 6), g, 0.5f);
    return __builtin_bit_cast(unsigned, g) - 0x80000001u < 0x3DFFFFFFu ? __builtin_fmaf(p * g, g, g) : fast_exp2(g * kLog2e);
}
// Whether e^g is zero: nothing passes that token, and of its run, whatever decays lie
// before it, NaN too, G is -inf.
__device__ __forceinline__ bool forgets(float c) { return __builtin_bit_cast(int, c) == 0; }
// e^g s + u for finite s
__device__ __forceinline__ float advance(float c, float s, float u) {
    const int mask = __builtin_bit_cast(int, c) >> 31;
    return __builtin_fmaf(c, s, u) + __builtin_bit_cast(float, __builtin_bit_cast(int, s) & mask);
}
// ... for any s.  Nothing of s, an infinity or NaN either, passes an e^g of zero;
// an infinity passes any other.
__device__ __forceinline__ float advance_any(float c, float s, float u) {
    const int bits = __builtin_bit_cast(int, c);
    const float t = __builtin_fmaf(c, s, u);
    return forgets(c) ? u : bits < 0 ? s + (__builtin_isinf(s) ? u : t) : t;
}

// A run's G is kept as G log2(e) / 2, so that e^G h can be formed in two steps
// where e^G alone overflows.
constexpr float kHalf = 0.5f * kLog2e;
// e^G h + X of a joined run, e = growth(G).  Nothing of h passes e = 0, which is that
// of G = -inf alone: an infinite or NaN h passes any product of decays, as it passes
// each.  (Of a finite one 2^-252 may be left where it should be less, below 2^-124.)
__device__ __forceinline__ float growth(float G) {
    return G == -INFINITY ? 0.f : fast_exp2(__builtin_amdgcn_fmed3f(G, -126.f, 127.f));
}
__device__ __forceinline__ float join(float e, float X, float h) { return e == 0.f ? X : __builtin_fmaf(e * h, e, X); }

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

// A tile: NW waves of LC lanes along the channels, VEC each, and 64 / LC along
// the tokens, R each.
template <int VEC_, int LC_, int R_, int NW_> struct Form {
    static constexpr bool NEAR = VEC_ > 1; // 32-bit offsets within a wave, see near_rows
    static constexpr int VEC = VEC_, LC = LC_, R = R_, NW = NW_, TL = 64 / LC, CH = LC * VEC, TT = TL * R * NW;
};
// (how much each takes of the registers goes by the types and by what is loaded:
// these are the largest without registers in memory)
template <typename T, bool BWD, bool HEAD> struct FormOf;
template <> struct FormOf<float, false, false> : Form<4, 32, 4, 8> {};
template <> struct FormOf<float, false, true> : Form<4, 32, 4, 8> {};
template <> struct FormOf<bf16, false, false> : Form<8, 16, 4, 8> {};
template <> struct FormOf<bf16, false, true> : Form<8, 16, 8, 8> {};
template <> struct FormOf<float, true, false> : Form<4, 32, 4, 8> {};
template <> struct FormOf<float, true, true> : Form<4, 32, 4, 8> {};
template <> struct FormOf<bf16, true, false> : Form<8, 16, 2, 8> {};
template <> struct FormOf<bf16, true, true> : Form<8, 16, 4, 8> {};
// The same for few chains: of fewer channels, so that a look reaches over four
// times the tokens (see plan_of).
template <typename T, bool BWD, bool HEAD> struct NarrowOf : Form<4, 8, 4, 8> {};
template <bool BWD, bool HEAD> struct NarrowOf<bf16, BWD, HEAD> : Form<8, 4, BWD && !HEAD ? 2 : 4, 8> {};
// Rows that are no multiple of 16 bytes, or not aligned to them.
typedef Form<4, 16, 4, 8> HalfForm;
typedef Form<1, 32, 8, 4> OddForm;

// A workgroup takes tile after tile: the number of the next one is drawn while
// this one's run is computed, and its loads are in flight from there on.
template <typename T, typename F, bool BWD, bool HEAD, bool HASW>
__global__ __launch_bounds__(64 * F::NW) void gated_scan_kernel(GatedScanParams p) {
    constexpr int VEC = F::VEC, LC = F::LC, R = F::R, NW = F::NW, TL = F::TL, CH = F::CH, TT = F::TT;
    constexpr int GV = HEAD ? 1 : VEC; // decays a token
    constexpr int LOOK = (CH + 63) / 64; // waves that join the tiles, a lane a channel
    static_assert(LOOK <= NW && R <= 32, "a bit a token of the run");
    __shared__ float tot[2][NW][CH]; // the waves' runs (G, X)
    __shared__ float enter[NW][CH];  // the states entering them
    __shared__ unsigned first_drawn, drawn;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cl = lane % LC, tl = lane / LC;
    const bool chained = p.tiles_t > 1;
    const unsigned tiles = p.chains * p.tiles_t;

    struct Place {
        unsigned number, chain, tile, ct; // tile number; its chain, place along the tokens and the channels
        int b, un, hu, h, c; // batch row, unit; the tile's first head, the lane's, its channel there
        int w0;              // the wave's first token in the direction of the recurrence
        bool ok;    // the lane's channels are there
        bool plain; // see below
        int p0;     // the run's first token
        unsigned have, first, last; // masks of the run's tokens: there, first of a sequence, last of one
    };
    auto token = [&](const Place &q, int i) { return BWD ? p.T - 1 - (q.p0 + i) : q.p0 + i; };
    auto place = [&](unsigned number) {
        Place q;
        q.number = number;
        q.tile = number / p.chains;
        q.chain = number % p.chains;
        q.ct = q.chain % p.tiles_c;
        const unsigned bu = q.chain / p.tiles_c;
        q.b = (int)(bu / (unsigned)p.units);
        q.un = (int)(bu % (unsigned)p.units);
        const int in_unit = (int)q.ct * CH + cl * VEC; // (VEC divides the unit)
        q.ok = in_unit < p.unit;
        const int ch0 = q.un * p.unit + (int)q.ct * CH; // (uniform)
        q.h = q.hu = ch0 / p.V;
        q.c = ch0 % p.V + (q.ok ? cl * VEC : 0);
        while (q.c >= p.V) { // (once at most where a head fills a tile)
            q.c -= p.V;
            ++q.h;
        }
        const int w0 = q.w0 = (int)q.tile * TT + wave * TL * R;
        q.p0 = w0 + tl * R;
        // Whether the wave's tokens are all there and of one sequence that neither
        // starts nor ends among them (for any offsets: all reads stay in bounds).
        bool plain = (int)(q.ct + 1) * CH <= p.unit && w0 + TL * R <= p.T;
        if (p.info) {
            if (plain) {
                const int lo = BWD ? p.T - w0 - TL * R : w0; // first token of the wave
                const int n = p.info[lo + 1];
                plain = n >= 0 && n == p.info[lo] && n == p.info[lo + TL * R + 1] && n == p.info[lo + TL * R];
            }
        } else {
            plain = plain && w0 > 0 && w0 + TL * R < p.T;
        }
        q.plain = __builtin_amdgcn_readfirstlane((int)plain);
        q.have = q.plain ? ~0u : 0u;
        q.first = q.last = 0;
        if (!q.plain && q.ok) {
#pragma unroll 1
            for (int i = 0; i < R; ++i) {
                const int t = token(q, i);
                bool in = t >= 0 && t < p.T, f = t == 0, l = t == p.T - 1;
                if (p.info && in) {
                    const int n = p.info[t + 1];
                    in = n >= 0;
                    f = in && p.info[t] != n;
                    l = in && p.info[t + 2] != n;
                }
                q.have |= (unsigned)in << i;
                q.first |= (unsigned)(in && f) << i;
                q.last |= (unsigned)(in && l) << i;
            }
        }
        return q;
    };

    // Channel `chan` of the lane's head at token(i) - shift of a tensor (the nearest
    // row where that is outside it): an address that the wave shares and 32 bits a
    // lane beside it, the same for every i of a plain run (`quick`).  Only rows too
    // far apart for that take 64 bits a lane.
    auto at = [&](const Place &q, auto quick, int i, const void *base, int size, int64_t sb, int64_t sh, int64_t st, int chan,
                  int shift) {
        const int t = min(max(token(q, i) - shift, 0), p.T - 1);
        const char *x = static_cast<const char *>(base);
        if constexpr (!F::NEAR) return x + size * (q.b * sb + q.h * sh + chan + t * st);
        constexpr bool Q = decltype(quick)::value;
        const int low = BWD ? max(p.T - q.w0 - TL * R, 0) : min(q.w0, p.T - 1); // the wave's lowest token
        const int row = Q ? low - shift + (BWD ? R - 1 - i : i) : max(low - shift, 0);
        const int lane_row = Q ? (BWD ? TL - 1 - tl : tl) * R : t - row;
        return x + size * (q.b * sb + q.hu * sh + row * st) +
               (unsigned)size * ((unsigned)(q.h - q.hu) * (unsigned)sh + (unsigned)chan + (unsigned)lane_row * (unsigned)st);
    };
    auto at_g = [&](const Place &q, auto quick, int i, const float *g) {
        return (float *)at(q, quick, i, g, 4, p.sgb, p.sgh, p.sgt, HEAD ? 0 : q.c, 0);
    };
    auto at_v = [&](const Place &q, auto quick, int i, const void *v) {
        return (T *)at(q, quick, i, v, sizeof(T), p.svb, p.svh, p.svt, q.c, 0);
    };
    auto at_o = [&](const Place &q, auto quick, int i, const void *o, int shift) {
        return (T *)at(q, quick, i, o, sizeof(T), p.sob, p.soh, p.sot, q.c, shift);
    };

    // All loads of a run, so that they are in flight together.  What is not there
    // reads some row of the tensor and is dropped.
    Raw<float, GV> rg[R];
    Raw<T, VEC> ru[R], rw[HASW ? R : 1], rv[BWD && HASW ? R : 1], rh[BWD ? R : 1];
    auto load_run = [&](const Place &q, auto quick) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            rg[i] = raw_n<float, GV>(at_g(q, quick, i, p.g));
            ru[i] = raw_n<T, VEC>(BWD ? at_o(q, quick, i, p.dy, 0) : at_v(q, quick, i, p.v)); // backward: dy
            if constexpr (BWD) rh[i] = raw_n<T, VEC>(at_o(q, quick, i, p.out, 1)); // the state before the token
            if constexpr (BWD && HASW) rv[i] = raw_n<T, VEC>(at_v(q, quick, i, p.v));
            if constexpr (HASW) rw[i] = raw_n<T, VEC>(at_v(q, quick, i, p.w));
        }
    };
    auto load = [&](const Place &q) {
        if (q.plain) load_run(q, std::true_type());
        else load_run(q, std::false_type());
    };

    unsigned number = blockIdx.x;
    if (chained) {
        if (tid == 0) first_drawn = atomicAdd(p.ticket, 1u) + 1u; // from all ones
        __syncthreads();
        number = __builtin_amdgcn_readfirstlane(first_drawn);
    }
    if (number >= tiles) return; // (the same for the whole workgroup)
    Place q = place(number);
    load(q);
    for (;;) {
        unsigned after = q.number + gridDim.x;
        if (chained && tid == 0) after = atomicAdd(p.ticket, 1u) + 1u;
        auto state_at = [&](int i) {
            return ((int64_t)(p.info ? p.info[token(q, i) + 1] : q.b) * p.H + q.h) * p.V + q.c;
        };
        const unsigned cut = BWD ? q.last : q.first; // nothing comes from the token before in this direction

        // decays, u (backward: dy), G
        float em[R][GV], u[R][VEC], G[GV], X[VEC];
#pragma unroll
        for (int j = 0; j < GV; ++j) G[j] = 0.f;
        if (q.plain) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int j = 0; j < GV; ++j) {
                    em[i][j] = decay(rg[i][j]);
                    G[j] = forgets(em[i][j]) ? -INFINITY : __builtin_fmaf(rg[i][j], kHalf, G[j]);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    u[i][j] = (float)ru[i][j];
                    if constexpr (HASW && !BWD) u[i][j] *= (float)rw[i][j];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool in = q.have >> i & 1, ct_i = cut >> i & 1;
#pragma unroll
                for (int j = 0; j < GV; ++j) {
                    const float gj = in ? rg[i][j] : 0.f;
                    em[i][j] = decay(gj);
                    G[j] = ct_i || forgets(em[i][j]) ? -INFINITY : __builtin_fmaf(gj, kHalf, G[j]);
                }
                float s0[VEC]; // forward: the state before a sequence; backward: the gradient of the one after it
#pragma unroll
                for (int j = 0; j < VEC; ++j) s0[j] = 0.f;
                const float *s = BWD ? p.ds : p.state_in;
                if (ct_i && s) load_n<float, VEC>(s + state_at(i), s0);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    u[i][j] = (float)ru[i][j];
                    if constexpr (HASW && !BWD) u[i][j] *= (float)rw[i][j];
                    u[i][j] = in ? u[i][j] : 0.f;
                    if (ct_i) u[i][j] = BWD ? u[i][j] + s0[j] : advance_any(em[i][HEAD ? 0 : j], s0[j], u[i][j]);
                }
            }
        }

        // the run, from a zero state
        bool finite = q.plain;
        if (q.plain) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) X[j] = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float e = em[i][HEAD ? 0 : j];
                    X[j] = BWD ? advance(e, u[i][j] + X[j], 0.f) : advance(e, X[j], u[i][j]);
                }
#pragma unroll
            for (int j = 0; j < VEC; ++j) finite = finite && __builtin_isfinite(X[j]);
        }
        if (!__all(finite)) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) X[j] = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float e = em[i][HEAD ? 0 : j];
                    const bool fresh = cut >> i & 1;
                    X[j] = BWD ? advance_any(e, fresh ? u[i][j] : u[i][j] + X[j], 0.f)
                               : fresh ? u[i][j] : advance_any(e, X[j], u[i][j]);
                }
        }

        // runs before this one: in the wave ...
        float Gw[GV], Xw[VEC];
#pragma unroll
        for (int j = 0; j < GV; ++j) Gw[j] = G[j];
#pragma unroll
        for (int j = 0; j < VEC; ++j) Xw[j] = X[j];
#pragma unroll
        for (int o = 1; o < TL; o <<= 1) {
            float e[GV];
#pragma unroll
            for (int j = 0; j < GV; ++j) {
                e[j] = growth(Gw[j]);
                const float Gp = __shfl_up(Gw[j], o * LC, 64);
                Gw[j] = tl >= o && Gw[j] != -INFINITY ? Gw[j] + Gp : Gw[j];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float Xp = __shfl_up(Xw[j], o * LC, 64);
                Xw[j] = tl >= o ? join(e[HEAD ? 0 : j], Xw[j], Xp) : Xw[j];
            }
        }
        if (tl == TL - 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                tot[0][wave][cl * VEC + j] = Gw[HEAD ? 0 : j];
                tot[1][wave][cl * VEC + j] = Xw[j];
            }
        }
#pragma unroll
        for (int j = 0; j < GV; ++j) {
            const float Gp = __shfl_up(Gw[j], LC, 64);
            Gw[j] = tl ? Gp : 0.f;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float Xp = __shfl_up(Xw[j], LC, 64);
            Xw[j] = tl ? Xp : 0.f;
        }
        if (tid == 0) drawn = after;
        __syncthreads();
        const unsigned next_number = __builtin_amdgcn_readfirstlane(drawn);
        const bool more = next_number < tiles;
        Place next = q;

        // what the backward still needs of this tile's rows
        Raw<T, VEC> kw[BWD && HASW ? R : 1], kv[BWD && HASW ? R : 1], kh[BWD ? R : 1];
        if constexpr (BWD) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                kh[i] = rh[i];
                if constexpr (HASW) kw[i] = rw[i], kv[i] = rv[i];
            }
        }

        // ... and before the tile
        if (wave < LOOK) {
            const int me = LOOK == 1 ? lane % CH : wave * 64 + lane;
            float hin = 0.f;
            if (chained) {
                const int tile = (int)q.tile;
                const int64_t at = (int64_t)q.chain * p.tiles_t * CH + me;
                float Gt = 0.f, Xt = 0.f;
#pragma unroll
                for (int k = 0; k < NW; ++k) {
                    const float Gk = tot[0][k][me];
                    Xt = join(growth(Gk), tot[1][k][me], Xt);
                    Gt = Gk == -INFINITY ? Gk : Gt + Gk;
                }
                const bool follows = q.tile + 1 < p.tiles_t && (LOOK > 1 || lane < CH);
                if (follows) publish(p.agg + at + (int64_t)tile * CH, (unsigned long long)word(Gt) | (unsigned long long)word(Xt) << 32);
                if (tile > 0) {
                    // Looks at the W tiles before this one (tile 0 stands in for any before it):
                    // a state passes W tiles a look.  4 take 1 % less where the chip is full
                    // (65536 x 2048 bf16) and 20 to 40 % more for a few channels (32318 x 128: 65
                    // against 52 us); looks by all waves, 16 tiles at a time, crowd the memory (87).
                    constexpr int W = VEC == 8 && !HEAD ? 6 : 8; // (as many as the registers hold)
                    for (;;) {
                        unsigned P[W];
                        unsigned long long A[W];
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            const int64_t from = at + (int64_t)max(tile - 1 - j, 0) * CH;
                            P[j] = peek(p.pre + from);
                            A[j] = peek(p.agg + from);
                        }
                        int nearest = W; // the nearest with its final state
                        bool gap = false;
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            nearest = nearest == W && !gap && P[j] != ~0u ? j : nearest;
                            gap = gap || A[j] == ~0ull;
                        }
                        if (__all(nearest < W)) {
#pragma unroll
                            for (int j = W - 1; j >= 0; --j) {
                                if (!__any(nearest >= j)) continue;
                                const float Gj = __builtin_bit_cast(float, (unsigned)A[j]), Xj = __builtin_bit_cast(float, (unsigned)(A[j] >> 32));
                                hin = j == nearest ? __builtin_bit_cast(float, P[j]) : j < nearest ? join(growth(Gj), Xj, hin) : hin;
                            }
                            break;
                        }
                        __builtin_amdgcn_s_sleep(1);
                    }
                }
                if (follows) publish(p.pre + at + (int64_t)tile * CH, word(join(growth(Gt), Xt, hin)));
            }
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                if (LOOK > 1 || lane < CH) enter[k][me] = hin;
                hin = join(growth(tot[0][k][me]), tot[1][k][me], hin);
            }
        }
        // (the waves above only now: their looks would wait for these loads)
        if (more) {
            next = place(next_number);
            load(next);
        }
        __syncthreads();

        float s[VEC]; // the state (or gradient) entering this thread's run
        float eg[GV];
#pragma unroll
        for (int j = 0; j < GV; ++j) eg[j] = growth(Gw[j]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = join(eg[HEAD ? 0 : j], Xw[j], enter[wave][cl * VEC + j]);
        // Whether the run stays finite from there: its recurrence ahead of the results, of
        // which no step makes a value finite again that is not (c inf + inf with c < 0
        // and 0 inf are NaN).
        finite = q.plain;
        if (q.plain) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float t = s[j];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float e = em[i][HEAD ? 0 : j];
                    t = BWD ? advance(e, u[i][j] + t, 0.f) : advance(e, t, u[i][j]);
                }
                finite = finite && __builtin_isfinite(t);
            }
        }

        // The results.  Each token's go out as soon as they are known.
        auto results = [&](auto quick) {
            constexpr bool QUICK = decltype(quick)::value;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool in = QUICK || (q.have >> i & 1), fresh = !QUICK && (cut >> i & 1);
                const bool row = QUICK || (q.ok && q.p0 + i < p.T);
                if constexpr (!BWD) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float e = em[i][HEAD ? 0 : j];
                        s[j] = QUICK ? advance(e, s[j], u[i][j]) : fresh ? u[i][j] : advance_any(e, s[j], u[i][j]);
                    }
                    if (in) stream_n<T, VEC>(at_o(q, quick, i, p.out, 0), s);
                    if (!QUICK && (q.last >> i & 1) && p.state_out) store_n<float, VEC>(p.state_out + state_at(i), s);
                } else {
                    float xg[VEC], xv[VEC], xw[VEC], hb[VEC]; // hb: the state before the token
                    const bool start = !QUICK && (q.first >> i & 1);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) hb[j] = start ? 0.f : (float)kh[i][j];
                    if (start && p.state_in) load_n<float, VEC>(p.state_in + state_at(i), hb);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float e = em[i][HEAD ? 0 : j], d = fresh ? u[i][j] : u[i][j] + s[j];
                        s[j] = QUICK ? advance(e, d, 0.f) : advance_any(e, d, 0.f);
                        // (rows outside every sequence have no part in L, nor has a state that is forgotten)
                        xg[j] = in && !forgets(e) ? s[j] * hb[j] : 0.f;
                        xv[j] = in ? (HASW ? (float)kw[HASW ? i : 0][j] * d : d) : 0.f;
                        if constexpr (HASW) xw[j] = in ? (float)kv[i][j] * d : 0.f;
                    }
                    if (row) {
                        stream_n<T, VEC>(at_v(q, quick, i, p.dv), xv);
                        if constexpr (HASW) stream_n<T, VEC>(at_v(q, quick, i, p.dw), xw);
                        if constexpr (!HEAD) stream_n<float, VEC>(at_g(q, quick, i, p.dg), xg);
                    }
                    if (start && p.state_out) store_n<float, VEC>(p.state_out + state_at(i), s);
                    if constexpr (HEAD) { // the tile's channels are of one head
                        float sum = 0.f;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) sum += xg[j];
                        sum = lanes_sum(sum, __builtin_ctz(LC));
                        if (cl == 0 && row) {
                            if (p.dgp) p.dgp[(((int64_t)q.b * p.units + q.un) * p.T + token(q, i)) * p.tiles_c + q.ct] = sum;
                            else *at_g(q, quick, i, p.dg) = sum;
                        }
                    }
                }
            }
        };
        if (__all(finite)) results(std::true_type());
        else results(std::false_type());

        // the states of sequences without tokens, some a tile
        if (p.cu && p.state_out) {
            const float *in = BWD ? p.ds : p.state_in;
            for (int n = (int)q.tile * (64 * NW / CH) + tid / CH; n < p.N; n += (int)p.tiles_t * (64 * NW / CH)) {
                const int at = (int)q.ct * CH + tid % CH;
                if (at < p.unit && p.cu[n + 1] <= p.cu[n]) {
                    const int64_t e = (int64_t)n * p.H * p.V + (int64_t)q.un * p.unit + at;
                    p.state_out[e] = in ? in[e] : 0.f;
                }
            }
        }
        if (!more) break;
        q = next;
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

// A few tokens: a thread walks its channels through them.  (64 x 16 heads of 128,
// one token: 3.1 MB in 3.6 us, one trip to memory and the launch.)
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
            s[j] = advance_any(dec, s[j], HASW ? x[j] * y[j] : x[j]);
        }
        store_n<T, VEC>(out + t * p.sot, s);
    }
    if (p.state_out) store_n<float, VEC>(p.state_out + e, s);
}

// -- host ---------------------------------------------------------------------

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Tokens that gated_step_kernel takes: up to kWalk; up to kWalkMany where there are
// more tiles of one than run at once (an almost empty tile costs its workgroup
// 7 us whatever it holds).  Rows of 2048 channels in f32, walked and in tiles:
// B = 1: 5.4 and 7.5 us at T = 8, 7.1 and 7.6 at 12, 8.7 and 7.6 at 16;
// B = 64: 6 and 27 us at T = 8, 25 and 31 at 32, 36 and 34 at 48.
constexpr int kWalk = 12, kWalkMany = 32;
constexpr int kFewChains = 4;   // see plan_of
constexpr int kResident = 1024; // workgroups, four a compute unit
constexpr int kMostTokens = 64, kMostChannels = 128; // of a wave, of a tile

struct Plan {
    int vec;
    bool walk, narrow;
    int ch, tt;
    int unit, units;
    int64_t tiles_c, tiles_t, chains;
    size_t o_pre, o_agg, words, o_info, o_dgp, bytes; // workspace: the ticket, pre, agg; the tokens' sequences; dg sums
};

// f(form) for the form that `vec` values a lane, and a plan's `narrow`, stand for
template <typename T, bool BWD, bool HEAD, typename Fn> auto with_form(int vec, bool narrow, Fn f) {
    if (vec == FormOf<T, BWD, HEAD>::VEC && narrow) return f(NarrowOf<T, BWD, HEAD>());
    if (vec == FormOf<T, BWD, HEAD>::VEC) return f(FormOf<T, BWD, HEAD>());
    if constexpr (FormOf<T, BWD, HEAD>::VEC == 8)
        if (vec == 4) return f(HalfForm());
    return f(OddForm());
}

template <typename T, bool BWD> Plan plan_of(const gdn2_gated_scan_args &a, int vec) {
    constexpr bool bwd = BWD;
    Plan q{};
    q.vec = vec;
    const int64_t len = a.seq_len, HV = a.num_heads * a.head_v_dim;
    const bool heads = bwd && a.g_per_head;
    q.unit = (int)(heads ? a.head_v_dim : HV);
    q.units = (int)(heads ? a.num_heads : 1);
    auto size = [&](bool narrow) {
        auto set = [&](auto form) {
            static_assert(form.TL * form.R <= kMostTokens && form.CH <= kMostChannels, "near_rows");
            q.ch = form.CH;
            q.tt = form.TT;
        };
        if (a.g_per_head) with_form<T, BWD, true>(vec, narrow, set);
        else with_form<T, BWD, false>(vec, narrow, set);
        q.tiles_c = (q.unit + q.ch - 1) / q.ch;
        q.tiles_t = (len + q.tt - 1) / q.tt;
        q.chains = a.batch * q.units * q.tiles_c;
    };
    size(false);
    // Up to four chains of more than one look are bound by what passes along them.
    // 32 channels a tile against 128: one row of 32318 x 128 bf16 30 and 57 us, 39921
    // x 200 f32 58 and 101, 8192 x 512 25 and 31 (adjoint 30 and 36); but 65536 x 2048
    // bf16 312 and 218, and equal at 8192 x 1024.
    q.narrow = q.chains <= kFewChains && q.tiles_t > 8;
    if (q.narrow) size(true);
    q.walk = !bwd && !a.cu_seqlens && len <= (q.chains > kResident ? kWalkMany : kWalk);
    if (q.walk) return q;
    size_t at = 0;
    if (q.tiles_t > 1) {
        at = 256;
        q.o_pre = at;
        at += up256(4 * (size_t)(q.chains * q.tiles_t * q.ch));
        q.o_agg = at;
        at += up256(8 * (size_t)(q.chains * q.tiles_t * q.ch));
        q.words = at;
    }
    q.o_info = at;
    if (a.cu_seqlens) at += up256(4 * (size_t)(len + 2));
    q.o_dgp = at;
    if (heads && q.tiles_c > 1) at += up256(4 * (size_t)(a.batch * a.num_heads * len * q.tiles_c));
    q.bytes = at;
    return q;
}

const char *check(const gdn2_gated_scan_args &a, bool *nothing, bool *limits) {
    *nothing = *limits = false;
    if (a.batch < 0 || a.num_heads < 0 || a.seq_len < 0 || a.head_v_dim < 0 || a.num_seqs < 0) return "negative dimension";
    if (a.cu_seqlens && a.batch != 1) return "packed sequences need batch 1";
    if (a.batch == 0 || a.num_heads == 0 || a.head_v_dim == 0) {
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

// A dimension of one has no stride to speak of.
gdn2_gated_scan_args tidy(gdn2_gated_scan_args a) {
    if (a.batch == 1) a.stride_g_b = a.stride_vw_b = a.stride_o_b = 0;
    if (a.num_heads == 1) a.stride_g_h = a.stride_vw_h = a.stride_o_h = 0;
    if (a.seq_len == 1) a.stride_g_t = a.stride_vw_t = a.stride_o_t = 0;
    return a;
}
// Whether the offsets within a wave's tokens and a tile's heads fit 31 bits.
bool near_rows(const gdn2_gated_scan_args &a) {
    const int64_t heads = std::min<int64_t>(a.num_heads, kMostChannels / a.head_v_dim + 2), most = (int64_t(1) << 29) - kMostChannels;
    auto fits = [&](int64_t sh, int64_t st) { // (each below 2^29 first, so that the sum is exact)
        return sh >= 0 && st >= 0 && sh < most && st < most && heads * sh + kMostTokens * st < most;
    };
    return fits(a.stride_g_h, a.stride_g_t) && fits(a.stride_vw_h, a.stride_vw_t) && fits(a.stride_o_h, a.stride_o_t);
}
// Values a lane: 16 bytes of T, half of them, or one, as the rows' lengths,
// strides and addresses allow; `more`: f32 and T pointers beside those of a.
template <typename T>
int vec_of(const gdn2_gated_scan_args &a, std::initializer_list<const void *> more_t, std::initializer_list<const void *> more_f) {
    int64_t s = a.head_v_dim | a.stride_vw_b | a.stride_vw_h | a.stride_vw_t | a.stride_o_b | a.stride_o_h | a.stride_o_t;
    uintptr_t t = reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.out);
    uintptr_t f = reinterpret_cast<uintptr_t>(a.state_in) | reinterpret_cast<uintptr_t>(a.state_out);
    for (const void *q : more_t) t |= reinterpret_cast<uintptr_t>(q);
    for (const void *q : more_f) f |= reinterpret_cast<uintptr_t>(q);
    if (!a.g_per_head) {
        s |= a.stride_g_b | a.stride_g_h | a.stride_g_t;
        f |= reinterpret_cast<uintptr_t>(a.g);
    }
    if (!near_rows(a)) return 1;
    for (int n = 16 / (int)sizeof(T); n >= 4; n /= 2)
        if (s % n == 0 && t % (n * sizeof(T)) == 0 && f % (4 * n) == 0) return n;
    return 1;
}
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

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
        p->ticket = reinterpret_cast<unsigned *>(ws);
        p->pre = reinterpret_cast<unsigned *>(ws + q.o_pre);
        p->agg = reinterpret_cast<unsigned long long *>(ws + q.o_agg);
    }
    if (a.cu_seqlens) {
        p->cu = a.cu_seqlens;
        p->N = (int)a.num_seqs;
        p->info = reinterpret_cast<const int *>(ws + q.o_info);
    }
}

template <typename T, bool BWD, bool HEAD, bool HASW>
hipError_t launch_tiles(const Plan &q, const GatedScanParams &p, hipStream_t s) {
    // as many workgroups as run at once
    const dim3 grid((unsigned)std::min<int64_t>(q.chains * q.tiles_t, kResident));
    with_form<T, BWD, HEAD>(q.vec, q.narrow, [&](auto form) {
        hipLaunchKernelGGL((gated_scan_kernel<T, decltype(form), BWD, HEAD, HASW>), grid, dim3(64 * form.NW), 0, s, p);
    });
    return hipGetLastError();
}
template <typename T, bool HEAD, bool HASW>
hipError_t launch_walk(const gdn2_gated_scan_args &a, const Plan &q, const GatedScanParams &p, hipStream_t s) {
    const int64_t n = a.batch * a.num_heads * a.head_v_dim / (q.vec > 1 ? 4 : 1);
    const dim3 grid((unsigned)((n + 255) / 256));
    if (q.vec > 1) hipLaunchKernelGGL((gated_step_kernel<T, 4, HEAD, HASW>), grid, dim3(256), 0, s, p, n);
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

template <typename T> gdn2_status forward(const char *who, const gdn2_gated_scan_args *args, hipStream_t s) {
    if (!args) return fail(GDN2_EINVAL, std::string(who) + ": null args");
    const gdn2_gated_scan_args tidied = tidy(*args), *const a = &tidied;
    bool nothing, limits;
    if (const char *e = check(*a, &nothing, &limits))
        return fail(limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL, std::string(who) + ": " + e);
    if (nothing || (a->cu_seqlens && a->num_seqs == 0)) return GDN2_OK;
    if (a->seq_len == 0) return no_tokens(*a, a->state_in, a->state_out, s);
    if (!a->g || !a->v || !a->out) return fail(GDN2_EINVAL, std::string(who) + ": null tensor pointer");
    if (a->out == a->v || a->out == a->w || a->out == a->g) return fail(GDN2_EINVAL, std::string(who) + ": out must not be an input");
    const Plan q = plan_of<T, false>(*a, vec_of<T>(*a, {}, {}));
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
    return GDN2_OK;
}

template <typename T> gdn2_status backward(const char *who, const gdn2_gated_scan_bwd_args *a, hipStream_t s) {
    if (!a) return fail(GDN2_EINVAL, std::string(who) + ": null args");
    const gdn2_gated_scan_args f = tidy(a->fwd);
    bool nothing, limits;
    if (const char *e = check(f, &nothing, &limits))
        return fail(limits ? GDN2_NOT_APPLICABLE : GDN2_EINVAL, std::string(who) + ": " + e);
    if (nothing) { // (heads of no channels still have a log decay)
        const double all = f.g_per_head ? (double)f.batch * f.num_heads * f.seq_len : 0;
        if (all == 0) return GDN2_OK;
        if (f.num_heads >= (1 << 30) || f.seq_len >= (1 << 30) || all >= 4294967040.0)
            return fail(GDN2_NOT_APPLICABLE, std::string(who) + ": sizes above the kernels' limits");
        const int64_t n = f.batch * f.num_heads * f.seq_len;
        if (!a->dg) return fail(GDN2_EINVAL, std::string(who) + ": null tensor pointer");
        GatedScanParams p{};
        p.dg = a->dg;
        p.sgb = f.stride_g_b; p.sgh = f.stride_g_h; p.sgt = f.stride_g_t;
        p.T = (int)f.seq_len; p.H = (int)f.num_heads;
        hipLaunchKernelGGL(dg_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, n);
        GDN2_HIP_CHECK(hipGetLastError());
        return GDN2_OK;
    }
    if (f.seq_len == 0) return f.cu_seqlens && f.num_seqs == 0 ? GDN2_OK : no_tokens(f, a->d_state_out, a->d_state0, s);
    if (!f.g || !f.out || !a->d_out || !a->dg || !a->dv || (f.w && !f.v))
        return fail(GDN2_EINVAL, std::string(who) + ": null tensor pointer");
    if (!f.w != !a->dw) return fail(GDN2_EINVAL, std::string(who) + ": dw must be given exactly where w is");
    for (const void *r : {(const void *)a->dg, (const void *)a->dv, (const void *)a->dw})
        for (const void *q : {(const void *)f.g, f.v, f.w, (const void *)f.out, a->d_out})
            if (r && r == q) return fail(GDN2_EINVAL, std::string(who) + ": dg, dv and dw must not be inputs");
    const int vec = vec_of<T>(f, {a->d_out, a->dv, a->dw}, {a->d_state_out, a->d_state0, f.g_per_head ? nullptr : a->dg});
    const Plan q = plan_of<T, true>(f, vec);
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
    return GDN2_OK;
}

// (of either type and alignment: the call knows them, the size does not)
template <bool BWD> size_t workspace_of(const gdn2_gated_scan_args *a) {
    bool nothing, limits;
    if (!a || check(*a, &nothing, &limits) || nothing || a->seq_len == 0) return 0;
    if (!BWD && a->cu_seqlens && a->num_seqs == 0) return 0;
    size_t n = 0;
    for (const int vec : {8, 4, 1})
        n = std::max({n, plan_of<float, BWD>(*a, vec).bytes, plan_of<bf16, BWD>(*a, vec).bytes});
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

extern "C" size_t gdn2_gated_scan_workspace_bytes(const gdn2_gated_scan_args *a) { return workspace_of<false>(a); }
extern "C" size_t gdn2_gated_scan_bwd_workspace_bytes(const gdn2_gated_scan_bwd_args *a) {
    return a ? workspace_of<true>(&a->fwd) : 0;
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
