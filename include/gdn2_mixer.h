/*
 * gdn2_mixer.h -- C ABI of the operators of a gated recurrent mixer that
 * stands beside the GDN-2 layer: the diagonal gated recurrence with its
 * backward, and the group norm with an activation with its backward.  (The
 * short conv in front of them is gdn2_short_conv_f32 of gdn2.h, its gradient
 * gdn2_short_conv_bwd_f32.)  No reference counterpart.
 *
 * Status codes and gdn2_last_error() are those of gdn2.h, and so are its
 * rules: caller-owned device pointers of the current device, no allocation,
 * asynchronous launches on `stream`, re-entrant across streams (calls that may
 * overlap need a workspace each).  Each call prepares its workspace itself and
 * leaves nothing in it for a later one, and may be captured into a graph (no
 * memset, copy or host node).  _f32: every tensor f32.  _bf16: the tensors
 * declared void * are bfloat16, everything else is f32; arithmetic, running
 * states and statistics are f32 in both, and a bfloat16 result is rounded once,
 * to nearest even.
 */
#ifndef GDN2_MIXER_H_
#define GDN2_MIXER_H_

#include "gdn2.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Gated scan: the recurrence of gdn2_recurrent_fwd_f32 with one state per
 * channel (K = 1, k = q = 1, no erase gate),
 *   h_t = e^{g_t} h_{t-1} + w_t v_t,   out_t = h_t.
 * g     log decay, f32 in both forms (a rounded log decay is off by the same
 *       factor at every token that the state lives through): [B, H, T, V], or
 *       [B, H, T] with g_per_head (one value per head and token).  Ordinary
 *       values are <= 0; where e^g is 0 in f32 (-inf, too) the state is
 *       forgotten, whatever it held; an infinity or a NaN lasts until then.  (An e^g
 *       below 2^-126 may count as 0.)
 *       A state that leaves f32's range is infinite; the ones after it are
 *       infinite or what the recurrence gives in a wider range.
 * v, w  [B, H, T, V]; w NULL means 1
 * out   [B, H, T, V], not overlapping the inputs
 * state_in [N, H, V] contiguous, or NULL (zeros); state_out likewise, or NULL
 *       (not wanted).  They may be the same buffer.
 * The last dimension is contiguous; strides are in elements for (batch, head,
 * time), any sign and order.
 * Without cu_seqlens N = batch.  With cu_seqlens (device, int32, num_seqs + 1
 * token offsets, not decreasing) batch must be 1 and N = num_seqs: sequence n
 * is tokens cu_seqlens[n] .. cu_seqlens[n + 1] - 1 of the one row, each with its
 * own state.  An empty sequence hands its state on.  Rows of out outside every
 * sequence are left as they were.  Offsets outside [0, seq_len] or decreasing
 * ones give unspecified results, never an access out of bounds.
 * workspace: gdn2_gated_scan_workspace_bytes(args) bytes, 256-byte aligned (0
 * for up to 12 tokens without cu_seqlens).
 * Results do not depend on timing: the same call gives the same bits.
 * Limits (else GDN2_NOT_APPLICABLE): every size < 2^30, H V < 2^30, N H V and
 * B H seq_len < 2^32 - 256, and B H ceil(V / 32) ceil(seq_len / 64) < 2^24.
 * ---------------------------------------------------------------------- */
typedef struct gdn2_gated_scan_args {
    const float *g;
    const void *v, *w;
    const float *state_in;
    float *state_out;
    void *out;
    const int32_t *cu_seqlens;
    int64_t batch, num_heads, seq_len, head_v_dim, num_seqs;
    int32_t g_per_head;
    int64_t stride_g_b, stride_g_h, stride_g_t;
    int64_t stride_vw_b, stride_vw_h, stride_vw_t;
    int64_t stride_o_b, stride_o_h, stride_o_t;
    void *workspace;
    size_t workspace_bytes;
} gdn2_gated_scan_args;

GDN2_API size_t gdn2_gated_scan_workspace_bytes(const gdn2_gated_scan_args *args);
GDN2_API gdn2_status gdn2_gated_scan_fwd_f32(const gdn2_gated_scan_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_gated_scan_fwd_bf16(const gdn2_gated_scan_args *args, gdn2_stream_t stream);

/* The gradients of L = <d_out, out> + <d_state_out, state_out> of that call:
 *   D_t = d_out_t + e^{g_{t+1}} D_{t+1}  (last token of a sequence: + d_state_out)
 *   dv = w D,  dw = v D,  dg_t = e^{g_t} D_t h_{t-1},  d_state0 = e^{g_0} D_0
 * (where e^{g_t} is 0, nothing of D passes it, and dg_t is 0 for any h_{t-1})
 *   fwd          the forward's arguments: g, v, w, state_in, cu_seqlens, shapes
 *                and strides; out as the forward wrote it (read: h_{t-1});
 *                state_out and workspace unused.  v is read only with w.
 *   d_out        strided like out
 *   d_state_out  [N, H, V] contiguous, or NULL (zero)
 *   dg           strided like g, f32; with g_per_head the sum over the head's
 *                channels (in a fixed order)
 *   dv, dw       strided like v; dw NULL iff w is
 *   d_state0     [N, H, V] contiguous, or NULL (not wanted); d_state_out may be
 *                the same buffer
 * Nothing else may overlap.  Rows of dg, dv and dw outside every
 * sequence are zero.
 * workspace: gdn2_gated_scan_bwd_workspace_bytes(args) bytes, 256-byte aligned.
 * Limits: those of the forward. */
typedef struct gdn2_gated_scan_bwd_args {
    gdn2_gated_scan_args fwd;
    const void *d_out;
    const float *d_state_out;
    float *dg;
    void *dv, *dw;
    float *d_state0;
    void *workspace;
    size_t workspace_bytes;
} gdn2_gated_scan_bwd_args;

GDN2_API size_t gdn2_gated_scan_bwd_workspace_bytes(const gdn2_gated_scan_bwd_args *args);
GDN2_API gdn2_status gdn2_gated_scan_bwd_f32(const gdn2_gated_scan_bwd_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_gated_scan_bwd_bf16(const gdn2_gated_scan_bwd_args *args, gdn2_stream_t stream);

/* ------------------------------------------------------------------------
 * Group norm with an activation, channels last.  x [N, S, C] has its channels
 * in `groups` runs of D = C / groups; a group's statistics are over the S rows
 * and D channels of one sample (S = 1: each token and head by itself, as
 * gdn2_rms_norm_gate_f32 normalises).
 *   n = (x - mean) / sqrt(var + eps),  z = n weight + bias
 *   y = act(z), or z act(gate) when a gate [N, S, C] is given
 * weight, bias [C] f32, either NULL (1, 0).  Rows are C contiguous elements;
 * strides in elements for (sample, row), one set for x and one for gate, y
 * and x share theirs.  y may be x, or gate where their strides are equal, and
 * must not overlap them otherwise.
 * stats [N, groups, 2] f32 contiguous, or NULL: mean and 1 / sqrt(var + eps),
 * what the backward takes (NaN for groups of no rows or channels).
 * workspace: gdn2_group_norm_act_workspace_bytes(args) bytes (0 for S = 1 and
 * ordinary groups), 256-byte aligned.
 * Limits (else GDN2_NOT_APPLICABLE): C < 2^24, S < 2^30, N and N groups < 2^24.
 * ---------------------------------------------------------------------- */
typedef enum gdn2_activation {
    GDN2_ACT_NONE = 0,
    GDN2_ACT_SILU = 1, /* z / (1 + e^-z) */
    GDN2_ACT_GELU = 2, /* z (1 + erf(z / sqrt 2)) / 2 */
} gdn2_activation;

typedef struct gdn2_group_norm_args {
    const void *x, *gate;
    const float *weight, *bias;
    void *y;
    float *stats;
    int64_t samples, rows, channels, groups;
    int64_t stride_x_n, stride_x_s;
    int64_t stride_gate_n, stride_gate_s;
    double eps;
    int32_t activation; /* gdn2_activation */
    void *workspace;
    size_t workspace_bytes;
} gdn2_group_norm_args;

GDN2_API size_t gdn2_group_norm_act_workspace_bytes(const gdn2_group_norm_args *args);
GDN2_API gdn2_status gdn2_group_norm_act_f32(const gdn2_group_norm_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_group_norm_act_bf16(const gdn2_group_norm_args *args, gdn2_stream_t stream);

/* A group that several workgroups hold is normalised once each has the others'
 * sums.  One that has looked `looks` times for another's forms them itself: the
 * results are the same bits.  Sets that number for calls that follow (512 in the
 * beginning; 0: hardly ever waits) and returns the one before; for tests. */
GDN2_API int gdn2_group_norm_patience(int looks);

/* The gradients of L = <d_y, y> of that call.  fwd: its arguments with the
 * stats it wrote (y unused).  d_y and dx strided like x, dgate like gate (NULL
 * iff gate is); dweight, dbias [C], either NULL (not wanted).  Every output is
 * overwritten; dx may be d_y, nothing else may overlap.  Sums
 * over samples and rows run in a fixed order.
 * workspace: gdn2_group_norm_act_bwd_workspace_bytes(args) bytes. */
typedef struct gdn2_group_norm_bwd_args {
    gdn2_group_norm_args fwd;
    const void *d_y;
    void *dx, *dgate;
    float *dweight, *dbias;
    void *workspace;
    size_t workspace_bytes;
} gdn2_group_norm_bwd_args;

GDN2_API size_t gdn2_group_norm_act_bwd_workspace_bytes(const gdn2_group_norm_bwd_args *args);
GDN2_API gdn2_status gdn2_group_norm_act_bwd_f32(const gdn2_group_norm_bwd_args *args, gdn2_stream_t stream);
GDN2_API gdn2_status gdn2_group_norm_act_bwd_bf16(const gdn2_group_norm_bwd_args *args, gdn2_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GDN2_MIXER_H_ */
