/*
 * astra_sequence.h -- C ABI of the sequence operators on MI355X (gfx950): the layer of a
 * recurrent policy that plays and learns the games of this library. It has no counterpart
 * in nlyu1/astra-cuda's C++ (its policies are PyTorch modules, python/src/high_low/agent.py).
 *
 *   short_conv   y[b,t,d] = act(bias[d] + sum_k weight[d,k] x[b,t-K+1+k,d])
 *   state_scan   dt = softplus(dt_raw + dt_bias);  h_t = exp(dt_t A) h_{t-1} + dt_t x_t (x) B_t
 *                y_t = h_t C_t + D x_t               (per head; x_t [P], B_t and C_t [N], h [P,N])
 *   join_norm    r' = r + scale * gate * rms(block) * post;  n = rms(r') * next
 *
 * All pointers are device pointers; work is queued on `stream` and nothing synchronises or
 * allocates. "Type" arguments are ASTRA_SEQ_F32 or ASTRA_SEQ_BF16. Strides count elements;
 * the last dimension of every tensor is contiguous. A length array (int32 [B], may be NULL)
 * says how many positions of each row count: those after it are not read, their outputs and
 * gradients are zero, and a row of length 0 keeps its initial state; values outside [0,T]
 * are clamped. Return values and astra_last_error() are those of astra_market.h.
 */
#ifndef ASTRA_SEQUENCE_H
#define ASTRA_SEQUENCE_H

#include <stddef.h>
#include <stdint.h>

#include "astra_market.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ASTRA_SEQ_F32 0
#define ASTRA_SEQ_BF16 1

#define ASTRA_SEQ_LINEAR 0 /* short_conv's activation: none */
#define ASTRA_SEQ_SILU 1

#define ASTRA_SEQ_MAX_TAPS 4
#define ASTRA_SEQ_MAX_STATE 128
#define ASTRA_SEQ_MAX_NORM_WIDTH 16384

/* ---- short_conv ------------------------------------------------------------------- */

/* Forward. x [B,T,D] of `type` with strides; weight float [D,K] and bias float [D] (may be
 * NULL); window [B,K-1,D] (may be NULL: zeros) holds the K-1 inputs before x; y [B,T,D]
 * contiguous; last [B,K-1,D] (may be NULL) gets the K-1 inputs before position length[b],
 * i.e. the window for what follows. 2 <= K <= ASTRA_SEQ_MAX_TAPS. */
typedef struct astra_short_conv {
  const void *x;
  const float *weight, *bias;
  const void *window;
  const int32_t *lengths;
  void *y, *last;
  int64_t batch, length, x_stride_b, x_stride_t;
  int32_t width, taps, type, activation;
} astra_short_conv;
int astra_short_conv_forward(const astra_short_conv *a, void *stream);

/* Backward: `f` as in the forward call (y and last are not used). dy [B,T,D] contiguous,
 * dlast [B,K-1,D] (may be NULL); dx [B,T,D] contiguous, dwindow [B,K-1,D], dweight
 * float [D,K] and dbias float [D]: each may be NULL if not wanted. The workspace holds the
 * partial sums of dweight and dbias. */
typedef struct astra_short_conv_grad {
  astra_short_conv f;
  const void *dy, *dlast;
  void *dx, *dwindow;
  float *dweight, *dbias;
  void *workspace;
  size_t workspace_bytes;
} astra_short_conv_grad;
int astra_short_conv_workspace_size(const astra_short_conv *f, size_t *bytes);
int astra_short_conv_backward(const astra_short_conv_grad *a, void *stream);

/* One position: x and y [B,D] (x with a row stride, `x_stride_b`), `window` [B,K-1,D] is
 * moved on by one input in place. */
typedef struct astra_short_conv_one {
  const void *x;
  const float *weight, *bias;
  void *window, *y;
  int64_t batch, x_stride_b;
  int32_t width, taps, type, activation;
} astra_short_conv_one;
int astra_short_conv_step(const astra_short_conv_one *a, void *stream);

/* ---- state_scan ------------------------------------------------------------------- */

/* Forward. x [B,T,H,P], dt [B,T,H], b and c [B,T,G,N] of `type` with strides (H a multiple
 * of G: head h reads group h / (H/G)); A, D (may be NULL), dt_bias (may be NULL) float [H];
 * initial float [B,H,P,N] (may be NULL: zeros); y [B,T,H,P] of `type`, contiguous; final
 * float [B,H,P,N] (may be NULL). chunk_states (may be NULL) keeps the states between the
 * chunks of positions for the backward call, astra_state_scan_chunk_states() floats of it.
 * N <= ASTRA_SEQ_MAX_STATE. */
typedef struct astra_state_scan {
  const void *x, *dt, *b, *c;
  const float *A, *D, *dt_bias, *initial;
  const int32_t *lengths;
  void *y;
  float *final_state, *chunk_states;
  int64_t batch, length;
  int64_t x_stride_b, x_stride_t, x_stride_h, dt_stride_b, dt_stride_t, dt_stride_h;
  int64_t b_stride_b, b_stride_t, b_stride_g, c_stride_b, c_stride_t, c_stride_g;
  int32_t heads, dim, groups, state, type;
  void *workspace;
  size_t workspace_bytes;
} astra_state_scan;
int astra_state_scan_chunk_states(const astra_state_scan *a, size_t *floats);
int astra_state_scan_workspace_size(const astra_state_scan *a, size_t *bytes);
int astra_state_scan_forward(const astra_state_scan *a, void *stream);

/* Backward: `f` as in the forward call, with the chunk_states that it wrote (y,
 * final_state and f's workspace are not used). dy [B,T,H,P] contiguous, dfinal float
 * [B,H,P,N] (may be NULL); dx [B,T,H,P], ddt [B,T,H], db and dc [B,T,G,N], contiguous, of
 * `type`; dA, dD, ddt_bias float [H] and dinitial float [B,H,P,N] (these four may be NULL). */
typedef struct astra_state_scan_grad {
  astra_state_scan f;
  const void *dy;
  const float *dfinal;
  void *dx, *ddt, *db, *dc;
  float *dA, *dD, *ddt_bias, *dinitial;
  void *workspace;
  size_t workspace_bytes;
} astra_state_scan_grad;
int astra_state_scan_grad_workspace_size(const astra_state_scan *f, size_t *bytes);
int astra_state_scan_backward(const astra_state_scan_grad *a, void *stream);

/* One position: x and y [B,H,P], dt [B,H], b and c [B,G,N] with strides (y contiguous);
 * h float [B,H,P,N], contiguous, is moved on in place. */
typedef struct astra_state_scan_one {
  const void *x, *dt, *b, *c;
  const float *A, *D, *dt_bias;
  float *h;
  void *y;
  int64_t batch;
  int64_t x_stride_b, x_stride_h, dt_stride_b, dt_stride_h, b_stride_b, b_stride_g, c_stride_b, c_stride_g;
  int32_t heads, dim, groups, state, type;
} astra_state_scan_one;
int astra_state_scan_step(const astra_state_scan_one *a, void *stream);

/* ---- join_norm -------------------------------------------------------------------- */

/* Forward. residual and joined [R,D] of residual_type; block, gate and normed of `type`;
 * post, next and scale (may be NULL: 1) float [D], or scale float [1] (scale_width 1).
 * gate (may be NULL: 1) is [R,D] or [R,1] (gate_width D or 1) before its sigmoid. block may
 * be NULL (then joined is not written and normed = rms(residual) * next), next may be NULL
 * (then normed is not written). rstd float [R,2] (may be NULL) keeps the two inverse roots
 * for the backward call. Row strides in elements; outputs contiguous. */
typedef struct astra_join_norm {
  const void *residual, *block, *gate;
  const float *post, *next, *scale;
  void *joined, *normed;
  float *rstd;
  int64_t rows, residual_stride, block_stride, gate_stride;
  int32_t width, gate_width, scale_width, type, residual_type;
  float eps;
} astra_join_norm;
int astra_join_norm_forward(const astra_join_norm *a, void *stream);

/* Backward: `f` as in the forward call with the rstd that it wrote (joined and normed are
 * not used). djoined [R,D] of residual_type (may be NULL: zeros) and dnormed [R,D] of
 * `type` (may be NULL), contiguous; dresidual, dblock, dgate contiguous; dpost, dnext
 * float [D], dscale float [scale_width]; gradients of what is absent are NULL, and any may
 * be NULL if not wanted. The workspace holds the partial sums over rows. */
typedef struct astra_join_norm_grad {
  astra_join_norm f;
  const void *djoined, *dnormed;
  void *dresidual, *dblock, *dgate;
  float *dpost, *dnext, *dscale;
  void *workspace;
  size_t workspace_bytes;
} astra_join_norm_grad;
int astra_join_norm_workspace_size(const astra_join_norm *f, size_t *bytes);
int astra_join_norm_backward(const astra_join_norm_grad *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ASTRA_SEQUENCE_H */
