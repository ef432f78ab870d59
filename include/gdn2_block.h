/*
 * gdn2_block.h -- C ABI of what stands around the mixer in a block that is
 * trained and served: dropout, the residual path with the norms behind one
 * block and before the next, and low-rank adapters beside a projection that
 * many requests share, each with its backward.  No reference counterpart.
 *
 * Status codes and gdn2_last_error() are those of gdn2.h, and so are its
 * rules: caller-owned device pointers of the current device, no allocation,
 * asynchronous launches on `stream`, re-entrant across streams (calls that may
 * overlap need a workspace each).  Each call prepares its workspace itself and
 * leaves nothing in it for a later one, and may be captured into a graph (no
 * memset, copy or host node).  The suffix names the types of the tensors
 * declared void *; everything else is f32.  Arithmetic, sums and statistics are
 * f32 or wider, and a bfloat16 result is rounded once, to nearest even.  The
 * last dimension of every tensor is contiguous, strides are in elements.
 * Results do not depend on timing: the same call gives the same bits.
 */
#ifndef GDN2_BLOCK_H_
#define GDN2_BLOCK_H_

#include "gdn2.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * The random words of dropout.  Row r, channel c of a tensor of rows of C
 * channels takes word c % 4 of Philox-4x32 with 7 rounds (Salmon, Moraes, Dror
 * and Shaw, 2011; 7 is the least number of rounds that they found to pass all of
 * their tests) under the key `seed` at the counter (modulo 2^64)
 *   offset + r ceil(C / 4) + c / 4.
 * The element is dropped where word >> 8 < round(p 2^24), so that p = 1 drops
 * all.  A call takes rows ceil(C / 4) counters; one that is to be independent of
 * it starts behind them.  The mask is a function of place alone: never stored,
 * the same in the backward, and the same whatever the strides and types.
 * rng: device pointer to two words, or NULL.  They give the seed in place of
 * `seed` and are added to `offset`, so that a captured graph can be replayed with
 * another mask.
 * ---------------------------------------------------------------------- */
typedef struct gdn2_dropout {
    double p; /* 0 <= p <= 1 */
    uint64_t seed, offset;
    const uint64_t *rng;
} gdn2_dropout;

/* y = x / (1 - p) where the element is kept, 0 where it is dropped (whatever x
 * holds).  x, y: rows of C channels, `stride_x` and `stride_y` apart.  y may be x with
 * the same stride and must not overlap it otherwise.  The gradient of x for dy is
 * the same call on dy.
 * Limits (else GDN2_NOT_APPLICABLE): C < 2^31, rows < 2^40; where C is a multiple of 8
 * and the rows lie together, rows C <= 2^34 - 2^10 in f32 and 2^35 - 2^11 in bf16;
 * elsewhere rows ceil(C / 4) < 2^32 - 2^8. */
GDN2_API gdn2_status gdn2_dropout_f32(const void *x, void *y, int64_t rows, int64_t channels, int64_t stride_x,
                                      int64_t stride_y, const gdn2_dropout *drop, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_dropout_bf16(const void *x, void *y, int64_t rows, int64_t channels, int64_t stride_x,
                                       int64_t stride_y, const gdn2_dropout *drop, gdn2_stream_t stream);

/* ------------------------------------------------------------------------
 * The residual path between two blocks, for every row of C channels of
 * [N, S, C]:
 *   p = y rstd(y) post_weight      (y itself without post_weight)
 *   r = residual_scale x + branch_scale dropout(act(gate) p)
 *   n = r rstd(r) pre_weight
 *   rstd(t) = 1 / sqrt(mean(t^2) + eps)
 * x, out (r)       the residual stream
 * y, gate, normed  the block's output, its gate, the next block's input
 * y NULL: no branch (r = residual_scale x; gate and post_weight must be NULL, p 0).
 * gate NULL: 1.  gate_rows: whether each row has a gate of its own, each sample
 * has one (stride_gate_s unused), or there is one for all (neither stride used).
 * normed NULL iff pre_weight is NULL: that norm is not taken; out may be NULL
 * (not wanted) only with it.
 * stats [N, S, 2] contiguous, or NULL: rstd(y) and rstd(r), which the backward
 * takes; 0 for a norm that is not taken.  rstd(r) and n are of r before its
 * rounding.  Without channels nothing is written.
 * out may be x and normed may be y, with the same strides; nothing else may
 * overlap.
 * _f32, _bf16: all of them; _f32_bf16: x and out f32; y, gate and normed bf16.
 * Limits (else GDN2_NOT_APPLICABLE): C <= 8192, N S < 2^30.
 * ---------------------------------------------------------------------- */
typedef enum gdn2_gate {
    GDN2_GATE_NONE = 0, /* z */
    GDN2_GATE_SILU = 1, /* z / (1 + e^-z) */
    GDN2_GATE_SIGMOID = 2,
} gdn2_gate;

typedef enum gdn2_gate_rows {
    GDN2_GATE_ROW = 0,
    GDN2_GATE_SAMPLE = 1,
    GDN2_GATE_ALL = 2,
} gdn2_gate_rows;

typedef struct gdn2_residual_norm_args {
    const void *x, *y, *gate;
    const float *post_weight, *pre_weight;
    void *out, *normed;
    float *stats;
    int64_t samples, rows, channels;
    int64_t stride_x_n, stride_x_s;
    int64_t stride_y_n, stride_y_s;
    int64_t stride_gate_n, stride_gate_s;
    int64_t stride_out_n, stride_out_s;
    int64_t stride_normed_n, stride_normed_s;
    double eps, residual_scale, branch_scale;
    int32_t activation; /* gdn2_gate */
    int32_t gate_rows;  /* gdn2_gate_rows */
    gdn2_dropout dropout;
} gdn2_residual_norm_args;

GDN2_API gdn2_status gdn2_residual_norm_f32(const gdn2_residual_norm_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_residual_norm_bf16(const gdn2_residual_norm_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_residual_norm_f32_bf16(const gdn2_residual_norm_args *args, gdn2_stream_t stream);

/* The gradients of L = <d_out, out> + <d_normed, normed> of that call.
 *   fwd       its arguments, with out and stats as it wrote them (x and normed
 *             unused)
 *   d_out     or NULL (zero); d_normed NULL iff pre_weight is
 *   dx        or NULL (not wanted); dy and dgate NULL iff y and gate are.  dgate has
 *             gate's rows: one a sample, or one, are sums over the rows that share it
 *   dpost, dpre  [C]; NULL iff the weight is
 * dx may be d_out and dy may be d_normed with the same strides; nothing else may
 * overlap.  Sums over rows run in a fixed order: in f32 over at most 128 of them,
 * those in f64 (of a workgroup's rows, rounded to f32, and of all workgroups).
 * Limits besides (else GDN2_NOT_APPLICABLE): N S < 2^28; where samples have a gate each,
 * N < 2^21 and N ceil(C / 32) < 2^23.
 * workspace: gdn2_residual_norm_bwd_workspace_bytes(args) bytes, 256-byte aligned: a row
 * of C f32 a workgroup for each weight and for a gate that rows share.  Workgroups: up to
 * 768, more only for more than 98304 rows; where samples have a gate each, at least one a
 * sample (32768 samples of two rows of 2048 channels, both weights: 805 MB). */
typedef struct gdn2_residual_norm_bwd_args {
    gdn2_residual_norm_args fwd;
    const void *d_out, *d_normed;
    void *dx, *dy, *dgate;
    float *dpost, *dpre;
    int64_t stride_d_out_n, stride_d_out_s;
    int64_t stride_d_normed_n, stride_d_normed_s;
    int64_t stride_dx_n, stride_dx_s;
    int64_t stride_dy_n, stride_dy_s;
    int64_t stride_dgate_n, stride_dgate_s;
    void *workspace;
    size_t workspace_bytes;
} gdn2_residual_norm_bwd_args;

GDN2_API size_t gdn2_residual_norm_bwd_workspace_bytes(const gdn2_residual_norm_bwd_args *args);
GDN2_API gdn2_status gdn2_residual_norm_bwd_f32(const gdn2_residual_norm_bwd_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_residual_norm_bwd_bf16(const gdn2_residual_norm_bwd_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_residual_norm_bwd_f32_bf16(const gdn2_residual_norm_bwd_args *args, gdn2_stream_t stream);

/* ------------------------------------------------------------------------
 * Low-rank adapters of many requests beside a projection that they share: for
 * every row x of a request with adapter l
 *   h = x a_l^T,  out = y + scale_l h b_l
 * x        [B, T, D];  y, out [B, T, O] (y: the shared projection's output)
 * a        [L, R, D];  b [L, R, O]: each rank's vectors contiguous
 * adapters device, int32, one of each request; outside [0, L): none, and out = y
 * scale    [L], or NULL (1)
 * hidden   [B, T, R] contiguous f32, or NULL: h (0 without an adapter), which the
 *          backward takes.  h is not rounded on its way to b.
 * Without cu_seqlens the requests are the batch entries.  With cu_seqlens (device,
 * int32, num_seqs + 1 token offsets, not decreasing) batch must be 1, and request n
 * is tokens cu_seqlens[n] .. cu_seqlens[n + 1] - 1 of the one row; rows outside all
 * of them have no adapter.  Offsets outside [0, T] or decreasing ones give
 * unspecified results, never an access out of bounds.
 * out may be y with the same strides, nothing else may overlap.
 * workspace: gdn2_low_rank_add_workspace_bytes(args) bytes, 256-byte aligned.
 * Limits (else GDN2_NOT_APPLICABLE): R <= 512; D, O, L, num_seqs < 2^24; fewer than 2^22
 * tiles of 16 rows of one request (B ceil(T / 16); packed: T / 16 + num_seqs + 2), which
 * for R > 64 and R = 0 by ceil(O / 256) are fewer than 2^24; strides of tokens and ranks < 2^24
 * (none negative: GDN2_EINVAL).
 * ---------------------------------------------------------------------- */
typedef struct gdn2_low_rank_args {
    const void *x, *a, *b, *y;
    void *out;
    const int32_t *adapters, *cu_seqlens;
    const float *scale;
    float *hidden;
    int64_t batch, seq_len, in_features, out_features, rank, num_adapters, num_seqs;
    int64_t stride_x_b, stride_x_t;
    int64_t stride_y_b, stride_y_t;
    int64_t stride_out_b, stride_out_t;
    int64_t stride_a_l, stride_a_r;
    int64_t stride_b_l, stride_b_r;
    void *workspace;
    size_t workspace_bytes;
} gdn2_low_rank_args;

GDN2_API size_t gdn2_low_rank_add_workspace_bytes(const gdn2_low_rank_args *args);
GDN2_API gdn2_status gdn2_low_rank_add_f32(const gdn2_low_rank_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_low_rank_add_bf16(const gdn2_low_rank_args *args, gdn2_stream_t stream);

/* The gradients of L = <d_out, out> of that call (y's is d_out itself):
 *   dh = scale_l d_out b_l^T,  dx = dh a_l,  da_l = sum dh^T x,  db_l = scale_l sum h^T d_out
 *   fwd    its arguments, with hidden as it wrote it; y, out and workspace unused
 *   d_out  [B, T, O];  dx [B, T, D], or NULL (not wanted).  Rows without an adapter: 0.
 *          accumulate_dx: added to what dx holds (the shared projection's gradient)
 *   da     [L, R, D], db [L, R, O] f32 contiguous, either NULL (not wanted): sums over
 *          all rows of an adapter's requests, 0 for one without any; in a fixed order,
 *          in f32 over at most 4096 rows, those in f64
 * Nothing may overlap.
 * Limits besides, the forward's for D in place of O (else GDN2_NOT_APPLICABLE):
 * (B T / 4096 + requests + 2) ((D + O) / 64 + 2) < 2^23, L R (D + O) < 2^31.
 * workspace: gdn2_low_rank_add_bwd_workspace_bytes(args) bytes, 256-byte aligned. */
typedef struct gdn2_low_rank_bwd_args {
    gdn2_low_rank_args fwd;
    const void *d_out;
    void *dx;
    float *da, *db;
    int32_t accumulate_dx;
    int64_t stride_d_out_b, stride_d_out_t;
    int64_t stride_dx_b, stride_dx_t;
    void *workspace;
    size_t workspace_bytes;
} gdn2_low_rank_bwd_args;

GDN2_API size_t gdn2_low_rank_add_bwd_workspace_bytes(const gdn2_low_rank_bwd_args *args);
GDN2_API gdn2_status gdn2_low_rank_add_bwd_f32(const gdn2_low_rank_bwd_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_low_rank_add_bwd_bf16(const gdn2_low_rank_bwd_args *args, gdn2_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GDN2_BLOCK_H_ */
