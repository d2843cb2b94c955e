/*
 * ttt_ops.h — C ABI of the operators at the model's tail: layer norm and the
 * softmax cross entropy of a linear head, each with its gradient and its
 * double backward (the gradient of the gradient).
 *
 * libttt_attn.so exports these entry points beside the attention's
 * (ttt_attn.h), under the same rules: raw device pointers, int64 sizes, a HIP
 * stream as `void*`, nothing allocated inside, all checks on the host before
 * anything is enqueued, a ttt_status returned and its message in
 * ttt_last_error().  Calls that may run at the same time need separate
 * workspaces.  There are no atomics: results repeat bitwise.
 *
 * A ttt_rows operand is a matrix whose columns are contiguous: a base pointer
 * and the row stride in elements (at least the column count).
 *
 * Layer norm, per row of D values (mu, r = 1/sqrt(var + eps) of the row,
 * xh = (x - mu) r, P(a) = a - mean(a) - xh mean(a xh)):
 *   y = xh w + b
 *   backward of dy, with g = dy w:
 *     dx = r P(g);  dw = sum_rows dy xh;  db = sum_rows dy
 *   double backward of cotangents a, cw, cb on (dx, dw, db):
 *     t   = cw dy - r (a mean(g xh) + g mean(a xh))
 *     gx  = r P(t) - r^2 xh mean(a P(g))
 *     gw  = sum_rows dy r P(a)
 *     gdy = w r P(a) + cw xh + cb
 *
 * Linear cross entropy of hidden rows X [N,d], head W [V,d] and targets t
 * (z = X W^T, never stored whole):
 *   l_i = log sum_j exp(z_ij) - z_{i,t_i}
 *   loss = w_i l_i (NONE), sum_i w_i l_i (SUM), or the SUM over
 *   max(sum_i w_i, 1) (MEAN).  w_i is the row weight (1 without one), 0 where
 *   t_i = ignore_index.  Rows of weight 0 give and get nothing, whatever their
 *   values are; a target outside [0, V) makes the loss and the gradients NaN.
 *   backward, with c_i = upstream w_i (over the MEAN's denominator), p the
 *   softmax of z and G = c (p - 1_t):  dX = G W;  dW = G^T X
 *   double backward of cotangents A, B on (dX, dW):
 *     U = A W^T + X B^T;  h_i = sum_j p_ij U_ij;  H = c p (U - h)
 *     gX = H W + G B;  gW = H^T X + G^T A;
 *     gupstream_i = (w_i / denominator) (h_i - U_{i,t_i})  (summed unless NONE)
 */
#ifndef TTT_OPS_H
#define TTT_OPS_H

#include <stdint.h>

#include "ttt_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ttt_rows {
  void* data;
  int64_t stride;
} ttt_rows;

typedef struct ttt_norm_problem {
  int32_t dtype;       /* of x, y, their gradients and cotangents (ttt_dtype)       */
  int32_t param_dtype; /* of weight, bias, theirs: dtype, or TTT_F32                */
  int64_t rows;        /* >= 1                                                      */
  int64_t cols;        /* 1 .. 32768 (16-bit types), 1 .. 16384 (TTT_F32)           */
  float eps;
} ttt_norm_problem;

/* Bytes of workspace that ttt_norm_bwd and ttt_norm_gg take (the larger of the two). */
int64_t ttt_norm_workspace_size(const ttt_norm_problem* problem);

/* y, and the rows' mean and rstd ([rows] fp32; both NULL when no gradient will
 * be asked for).  weight and bias ([cols]) may each be NULL (1 and 0). */
int ttt_norm_fwd(const ttt_norm_problem* problem, const ttt_rows* x, const void* weight, const void* bias,
                 const ttt_rows* y, float* mean, float* rstd, void* stream);

/* Any of dx, dweight, dbias may be NULL. */
int ttt_norm_bwd(const ttt_norm_problem* problem, const ttt_rows* x, const void* weight, const ttt_rows* dy,
                 const float* mean, const float* rstd, const ttt_rows* dx, void* dweight, void* dbias,
                 void* workspace, int64_t workspace_bytes, void* stream);

/* Any cotangent (a, cw, cb) may be NULL (zero), as may any output (gx, gw, gdy). */
int ttt_norm_gg(const ttt_norm_problem* problem, const ttt_rows* x, const void* weight, const ttt_rows* dy,
                const float* mean, const float* rstd, const ttt_rows* a, const void* cw, const void* cb,
                const ttt_rows* gx, void* gw, const ttt_rows* gdy, void* workspace, int64_t workspace_bytes,
                void* stream);

typedef enum ttt_reduction {
  TTT_REDUCE_NONE = 0,
  TTT_REDUCE_SUM = 1,
  TTT_REDUCE_MEAN = 2
} ttt_reduction;

typedef enum ttt_lce_entry {
  TTT_LCE_FWD = 0,
  TTT_LCE_BWD = 1,
  TTT_LCE_GG = 2
} ttt_lce_entry;

/* x, w and their gradients and cotangents have type `dtype`.  16-bit rows whose
 * column count is a multiple of 8 must be 16-byte aligned (base and stride);
 * other rows are taken as they are. */
typedef struct ttt_lce_problem {
  int32_t dtype;
  int32_t reduction;    /* ttt_reduction                                        */
  int64_t rows;         /* N: 1 .. 2^22                                         */
  int64_t cols;         /* d: 1 .. 2^16                                         */
  int64_t vocab;        /* V: 1 .. 2^22                                         */
  int64_t ignore_index;
} ttt_lce_problem;

/* Bytes of workspace of an entry point (ttt_lce_entry), -1 for a bad problem. */
int64_t ttt_lce_workspace_size(const ttt_lce_problem* problem, int32_t entry);

/* loss: [rows] (NONE) or one value, fp32.  row_stats: [2 * rows + 2] fp32, the
 * softmax statistics and the reduction's factors that the backward entries read. */
int ttt_lce_fwd(const ttt_lce_problem* problem, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
                const float* row_weight, float* loss, float* row_stats, void* workspace, int64_t workspace_bytes,
                void* stream);

/* grad_loss: fp32, of loss's shape.  dx or dw may be NULL.  dx32 ([rows, cols]
 * contiguous, or NULL): dx before its rounding, for ttt_lce_gg. */
int ttt_lce_bwd(const ttt_lce_problem* problem, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
                const float* row_weight, const float* row_stats, const float* grad_loss, const ttt_rows* dx,
                const ttt_rows* dw, float* dx32, void* workspace, int64_t workspace_bytes, void* stream);

/* a, b: cotangents of dx and dw; either may be NULL (zero), not both.  Any of
 * gx, gw and ggrad_loss (of loss's shape) may be NULL.  dx32: what ttt_lce_bwd
 * wrote, or NULL (h is then summed from tiles, a third more work). */
int ttt_lce_gg(const ttt_lce_problem* problem, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
               const float* row_weight, const float* row_stats, const float* grad_loss, const float* dx32,
               const ttt_rows* a, const ttt_rows* b, const ttt_rows* gx, const ttt_rows* gw, float* ggrad_loss,
               void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TTT_OPS_H */
