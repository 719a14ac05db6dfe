/*
 * remora_b200_seq.h — operators of a sequence block, beside the hot-path
 * entry points of remora_b200.h: root-mean-square norm (beside the row folds),
 * depthwise causal convolution (beside the convolutions) and the selective
 * state space scan (beside the scans), each forward, backward and for single
 * tokens.  None has a counterpart in the reference, whose scans are + and *
 * only (remora/lowering/tensor_ops.py:2301-2482) and whose convolution is the
 * single-channel im2col one (examples/crater_train.py:30-36).
 *
 * Conventions are those of remora_b200.h: descriptors by host pointer with any
 * element strides, f32 data unless an argument says otherwise, caller-owned
 * buffers, asynchronous on the given stream, a status code per call.  And:
 *  - The calling thread's current device is left as it was.
 *  - Nothing is allocated.  Calls that need scratch take it as (scratch,
 *    scratch_bytes), 16-byte aligned device memory that only this call uses
 *    until it has run; the matching _scratch entry point gives its size.  So a
 *    call can be captured into a CUDA graph, and two graphs share nothing
 *    that the caller did not share.
 *  - `lengths` (int32, one per sequence, may be NULL): sequence b is
 *    lengths[b] positions long, taken as 0 below 0 and as L above L.  Rows
 *    behind a sequence's end are never read; in outputs and gradients they
 *    stay as they were, or become zero where the spec's zero_rest is set.
 *  - Outputs must not overlap inputs or each other, except where an entry
 *    point says so, nor share addresses among their own elements; views that
 *    interleave (columns of one wider array) do not count as overlapping.  Input gradients of one array passed twice are two
 *    separate outputs.
 *  - Results do not depend on timing: sums run in a fixed order.
 */
#ifndef REMORA_B200_SEQ_H
#define REMORA_B200_SEQ_H

#include "remora_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------ */
/* Root-mean-square norm of the last axis                                   */
/* ------------------------------------------------------------------------ */
typedef struct {
  float eps;     /* >= 0                                                     */
  int32_t group; /* quant: columns per scale, 32, 64 or 128 dividing the
                    row; 0: one scale per row.  Others ignore it             */
} RemoraNormSpec;

/* s = x + residual (s = x without one); y = s / sqrt(mean(s^2) + eps) * w over
   the last axis.  x, residual, y and sum have rank `rank` (1..4); w has rank
   1.  residual may be NULL; sum (gets s) may be NULL, and must be without a
   residual.  y or sum may be exactly x or exactly residual (in place). */
int remora_b200_rms_norm_fwd(RemoraB200Ctx *ctx, const RemoraNormSpec *spec,
                             const void *x, const void *residual,
                             const RemoraMemRef1 *w, void *y, void *sum,
                             int32_t rank, remora_stream_t stream);

/* The same y in 8 bits: per row or per group of columns
   scale = max(max|y| / 448, 2^-126), q = the f32 quotient y / scale rounded to
   the nearest e4m3 value (4 exponent and 3 fraction bits, largest 448, ties to
   even), one byte each.  q has x's shape, scales x's leading axes and one last axis of
   dim / group (1 for group 0).  A NaN in a row gives NaN scales there. */
int remora_b200_rms_norm_quant(RemoraB200Ctx *ctx, const RemoraNormSpec *spec,
                               const void *x, const void *residual,
                               const RemoraMemRef1 *w, void *q, void *scales,
                               void *sum, int32_t rank, remora_stream_t stream);

/* Gradients of rms_norm_fwd from its s: with xh = s / sqrt(mean(s^2) + eps),
   dx = (w dy - xh mean(w dy xh)) / sqrt(mean(s^2) + eps) + dsum, the gradient
   of x and of the residual alike; dw = sum over rows of dy xh.  dsum (the
   gradient that reaches s itself) may be NULL.  dx may be exactly dy, dsum or
   s (in place). */
int remora_b200_rms_norm_bwd_scratch(RemoraB200Ctx *ctx, int64_t rows,
                                     int64_t dim, size_t *bytes);
int remora_b200_rms_norm_bwd(RemoraB200Ctx *ctx, const RemoraNormSpec *spec,
                             const void *s, const RemoraMemRef1 *w,
                             const void *dy, const void *dsum, void *dx,
                             RemoraMemRef1 *dw, int32_t rank, void *scratch,
                             size_t scratch_bytes, remora_stream_t stream);

/* ------------------------------------------------------------------------ */
/* Depthwise causal convolution along time                                  */
/* ------------------------------------------------------------------------ */
typedef struct {
  int32_t silu;      /* 1: y = p / (1 + exp(-p)) of the convolution's p     */
  int32_t zero_rest; /* 1: rows of y and dx that belong to no sequence
                        (behind an end; of a token left out) are set to zero */
} RemoraCausalConvSpec;

/* p[b,t,d] = bias[d] + sum_k w[d,k] x[b, t - (W-1) + k, d], W taps (2..8), x
   and y [B,L,D], w [D,W], bias [D] or NULL.  Rows before the first are
   state [B,W-1,D], or zeros when NULL.  state_out [B,W-1,D] (may be NULL, may
   be exactly state) gets the last W-1 rows of state followed by the
   sequence: the state of the call that continues it. */
int remora_b200_causal_conv_fwd(RemoraB200Ctx *ctx,
                                const RemoraCausalConvSpec *spec,
                                const RemoraMemRef3 *x, const RemoraMemRef2 *w,
                                const RemoraMemRef1 *bias,
                                const RemoraMemRef3 *state,
                                const RemoraMemRef1 *lengths, RemoraMemRef3 *y,
                                RemoraMemRef3 *state_out,
                                remora_stream_t stream);

/* Its gradients: dx [B,L,D], dw [D,W], dbias [D] (NULL: not wanted), dstate
   [B,W-1,D] (NULL: not wanted).  dstate_out (may be NULL) is the gradient
   that reaches state_out. */
int remora_b200_causal_conv_bwd_scratch(RemoraB200Ctx *ctx, int64_t batch,
                                        int64_t length, int64_t dim,
                                        int64_t width, size_t *bytes);
int remora_b200_causal_conv_bwd(
    RemoraB200Ctx *ctx, const RemoraCausalConvSpec *spec,
    const RemoraMemRef3 *x, const RemoraMemRef2 *w, const RemoraMemRef1 *bias,
    const RemoraMemRef3 *state, const RemoraMemRef1 *lengths,
    const RemoraMemRef3 *dy, const RemoraMemRef3 *dstate_out, RemoraMemRef3 *dx,
    RemoraMemRef2 *dw, RemoraMemRef1 *dbias, RemoraMemRef3 *dstate,
    void *scratch, size_t scratch_bytes, remora_stream_t stream);

/* One token per row: x and y [B,D].  Row i's state is row slots[i] of state
   [S,W-1,D] (slots int32 [B]; NULL: row i, B <= S); state_out [S,W-1,D]
   (exactly state for an update in place) gets the moved window in the same
   row, its other rows stay as they were.  A row whose slot is outside 0..S-1
   (-1 for padding) or was named by an earlier row is left out: all states and,
   without zero_rest, its y stay as they were.  B is at most 65535; each block
   of a row reads the slots ahead of it, so with slots the time has a part that
   grows with B squared (conv step of 4096 channels, 4 taps: 4096 rows 152 us
   without slots and 163 with; scan step of 4096 channels, 16 states: 1024 rows
   130 and 168 us, 4096 rows 504 and 1101). */
int remora_b200_causal_conv_step(RemoraB200Ctx *ctx,
                                 const RemoraCausalConvSpec *spec,
                                 const RemoraMemRef2 *x,
                                 const RemoraMemRef3 *state,
                                 const RemoraMemRef2 *w,
                                 const RemoraMemRef1 *bias,
                                 const RemoraMemRef1 *slots, RemoraMemRef2 *y,
                                 RemoraMemRef3 *state_out,
                                 remora_stream_t stream);

/* ------------------------------------------------------------------------ */
/* Selective state space scan                                               */
/* ------------------------------------------------------------------------ */
typedef struct {
  int32_t softplus;  /* 1: the step is softplus(delta + delta_bias)          */
  int32_t zero_rest; /* 1: rows of y, du, ddelta, dz, db and dc that belong to
                        no sequence are set to zero                          */
} RemoraSelectiveScanSpec;

/* Inputs of the scan over [B,L,D] with N states (1..64) per channel:
     s[t,d]   = f(delta[t,d] + delta_bias[d]), f softplus or the identity
     h[t,d,n] = exp(s[t,d] a[d,n]) h[t-1,d,n] + s[t,d] u[t,d] b[t,g,n]
     p[t,d]   = sum_n c[t,g,n] h[t,d,n] + d[d] u[t,d]
     y[t,d]   = p[t,d] z[t,d] / (1 + exp(-z[t,d]))   (y = p without z)
   for every sequence of the batch; channel d reads group g = d / (D / G) of
   b and c, G dividing D.  Members marked (NULL) may be NULL. */
typedef struct {
  const RemoraMemRef3 *u;          /* [B,L,D]                                */
  const RemoraMemRef3 *delta;      /* [B,L,D]                                */
  const RemoraMemRef2 *a;          /* [D,N]                                  */
  const RemoraMemRef4 *b;          /* [B,L,G,N]                              */
  const RemoraMemRef4 *c;          /* [B,L,G,N]                              */
  const RemoraMemRef1 *d;          /* [D] (NULL: 0)                          */
  const RemoraMemRef3 *z;          /* [B,L,D] (NULL: no gate)                */
  const RemoraMemRef1 *delta_bias; /* [D] (NULL: 0)                          */
  const RemoraMemRef3 *h0;         /* [B,D,N] state ahead of t = 0 (NULL: 0) */
  const RemoraMemRef1 *lengths;    /* int32 [B] (NULL: all L)                */
} RemoraSelectiveScanIn;

/* y [B,L,D]; h_last [B,D,N] (may be NULL, may be exactly h0) gets the state
   behind each sequence's last position.  saved (may be NULL): f32 memory of
   remora_b200_selective_scan_saved bytes, 16-byte aligned, that gets the
   states the backward pass starts from: those ahead of every 4th position (8th
   above 16 states, 16th above 32), N rounded up to a power of two, at least 4.
   That is N bytes per element of u for 4, 8 and 16 states and 16 bytes for more. */
int remora_b200_selective_scan_saved(int64_t batch, int64_t length, int64_t dim,
                                     int64_t states, size_t *bytes);
int remora_b200_selective_scan_fwd_scratch(RemoraB200Ctx *ctx, int64_t batch,
                                           int64_t length, int64_t dim,
                                           int64_t states, int64_t groups,
                                           size_t *bytes);
int remora_b200_selective_scan_fwd(RemoraB200Ctx *ctx,
                                   const RemoraSelectiveScanSpec *spec,
                                   const RemoraSelectiveScanIn *in,
                                   RemoraMemRef3 *y, RemoraMemRef3 *h_last,
                                   void *saved, size_t saved_bytes,
                                   void *scratch, size_t scratch_bytes,
                                   remora_stream_t stream);

/* Gradients; each shaped as its input.  dd, dz, ddelta_bias and dh0 may be
   NULL (not wanted; dz must be NULL without z). */
typedef struct {
  RemoraMemRef3 *du;
  RemoraMemRef3 *ddelta;
  RemoraMemRef2 *da;
  RemoraMemRef4 *db;
  RemoraMemRef4 *dc;
  RemoraMemRef1 *dd;
  RemoraMemRef3 *dz;
  RemoraMemRef1 *ddelta_bias;
  RemoraMemRef3 *dh0;
} RemoraSelectiveScanGrads;

/* Backward pass of selective_scan_fwd on the same inputs, from dy [B,L,D],
   the gradient dh_last [B,D,N] that reaches h_last (may be NULL) and the
   forward's `saved`. */
int remora_b200_selective_scan_bwd_scratch(RemoraB200Ctx *ctx, int64_t batch,
                                           int64_t length, int64_t dim,
                                           int64_t states, int64_t groups,
                                           size_t *bytes);
int remora_b200_selective_scan_bwd(RemoraB200Ctx *ctx,
                                   const RemoraSelectiveScanSpec *spec,
                                   const RemoraSelectiveScanIn *in,
                                   const RemoraMemRef3 *dy,
                                   const RemoraMemRef3 *dh_last,
                                   const void *saved, size_t saved_bytes,
                                   const RemoraSelectiveScanGrads *grads,
                                   void *scratch, size_t scratch_bytes,
                                   remora_stream_t stream);

/* Inputs of one token per row: as RemoraSelectiveScanIn without the time
   axis.  Row i's state is row slots[i] of `state`, with the rules of
   remora_b200_causal_conv_step. */
typedef struct {
  const RemoraMemRef3 *state;      /* [S,D,N]                                */
  const RemoraMemRef2 *u;          /* [B,D]                                  */
  const RemoraMemRef2 *delta;      /* [B,D]                                  */
  const RemoraMemRef2 *a;          /* [D,N]                                  */
  const RemoraMemRef3 *b;          /* [B,G,N]                                */
  const RemoraMemRef3 *c;          /* [B,G,N]                                */
  const RemoraMemRef1 *d;          /* [D] (NULL: 0)                          */
  const RemoraMemRef2 *z;          /* [B,D] (NULL: no gate)                  */
  const RemoraMemRef1 *delta_bias; /* [D] (NULL: 0)                          */
  const RemoraMemRef1 *slots;      /* int32 [B] (NULL: row i, B <= S)        */
} RemoraSelectiveStepIn;

/* y [B,D]; state_out [S,D,N], exactly `state` for an update in place. */
int remora_b200_selective_scan_step(RemoraB200Ctx *ctx,
                                    const RemoraSelectiveScanSpec *spec,
                                    const RemoraSelectiveStepIn *in,
                                    RemoraMemRef2 *y, RemoraMemRef3 *state_out,
                                    remora_stream_t stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* REMORA_B200_SEQ_H */
