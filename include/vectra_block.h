/*
 * vectra_block.h: C ABI of the transformer-block operators that stand
 * around RBF attention (libvectra_rbf.so).
 *
 *  - vectra_linear_*:        y = act(x W^T + b) + r
 *  - vectra_gated_linear_*:  h = act(x Wg^T + bg) * (x Wu^T + bu)
 *  - vectra_qk_norm_rope_*:  the RMS norm of every query and key head vector
 *                            and the rotation of its position, in one pass
 *
 * each with its backward pass. Conventions are those of vectra_rbf.h: plain
 * pointers, sizes and element strides; the caller owns every buffer; calls
 * are asynchronous on the given stream; functions return VECTRA_OK or a
 * negative status, whose text vectra_block_strerror gives. Sums, norms and
 * activations are computed in 32 bits and each result is rounded once to
 * its type. With 16-bit tensors two inner values are rounded as well, which
 * the tensor cores take in 16 bits or the caller keeps: a gradient dz (of a
 * gated layer dg and du) before its products with the weight and with x, and
 * vectra_linear's pre. A gated layer's gradients are then off by 2.3e-3 of
 * their size in bfloat16, where one rounding alone is 1.7e-3.
 *
 * A wait that runs out inside a kernel ends it early with an unfinished
 * result; the call has returned VECTRA_OK by then.
 * vectra_rbf_check_device_errors (vectra_rbf.h) reports it, for these calls
 * as for the attention's.
 *
 * The backward calls and some forward calls need a workspace, sized by the
 * matching *_workspace_bytes (which may answer 0) for the same arguments
 * (the buffers' addresses and strides count: they decide which kernel runs).
 * It must be 256-byte aligned, holds nothing between calls and may be shared
 * by calls on one stream.
 */
#ifndef VECTRA_BLOCK_H_
#define VECTRA_BLOCK_H_

#include <stddef.h>
#include <stdint.h>

#include "vectra_rbf.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes beyond those of vectra_rbf.h. */
enum {
  VECTRA_ERR_LAYOUT = -12,   /* a result's or a table's strides */
  VECTRA_ERR_WORKSPACE = -13 /* workspace too small or misaligned */
};

/* Activations. GELU is x * Phi(x) (erf); GELU_TANH its tanh form; SILU is
 * x * sigmoid(x). */
typedef enum {
  VECTRA_ACT_NONE = 0,
  VECTRA_ACT_RELU = 1,
  VECTRA_ACT_GELU = 2,
  VECTRA_ACT_GELU_TANH = 3,
  VECTRA_ACT_SILU = 4
} vectra_activation;
/* Their float32 values keep a relative accuracy down the negative tail; for
 * 16-bit results GELU is good to 1.5e-7 absolute. An infinite argument gives
 * what the formula gives in floating point: NaN for GELU, GELU_TANH or SILU
 * of minus infinity. */

/* y = act(x W^T + b) + r.
 *  x [M,K], weight [N,K], bias [N] (data NULL: none), residual [M,N] (data
 *  NULL: none): one dtype of F32 / F16 / BF16, any strides.
 *  y [M,N]: unit stride along N, non-negative row stride of at least N.
 *  pre [M,N] (data NULL: not wanted): receives x W^T + b in the same dtype,
 *  for the backward pass; same layout rule as y. */
typedef struct {
  vectra_tensor x, weight, bias, residual, y, pre;
  int32_t activation; /* vectra_activation */
  void* workspace;
  size_t workspace_bytes;
} vectra_linear_args;

/* Gradients of the above for dy [M,N]: dz = dy * act'(pre), dx = dz W,
 * dweight = dz^T x, dbias = sum of dz over rows (the residual's gradient is
 * dy itself).
 *  dy [M,N], x [M,K], weight [N,K]: as in the forward, any strides.
 *  pre [M,N]: the forward's, unless activation is NONE (data NULL then).
 *  dx [M,K], dweight [N,K], dbias [N]: data NULL when not wanted; unit
 *  inner stride. */
typedef struct {
  vectra_tensor dy, x, weight, pre, dx, dweight, dbias;
  int32_t activation;
  void* workspace;
  size_t workspace_bytes;
} vectra_linear_grad_args;

/* h = act(x Wg^T + bg) * (x Wu^T + bu).
 *  x [M,K], w_gate and w_up [F,K], b_gate and b_up [F] (data NULL: none),
 *  any strides; h [M,F] unit inner stride.
 *  gate, up [M,F] F32 (both or neither): receive the two projections for
 *  the backward pass, in 32 bits: the backward multiplies by them, and
 *  16-bit copies would add a rounding to every gradient. */
typedef struct {
  vectra_tensor x, w_gate, w_up, b_gate, b_up, h, gate, up;
  int32_t activation;
  void* workspace;
  size_t workspace_bytes;
} vectra_gated_args;

/* With a reduction (K) up to this long, forming gate and up again in the
 * backward pass takes less time than writing and reading them (bf16 / f16;
 * forward and whole backward on a B200, us, saved against formed again, for
 * 66,560 x K -> 704, 16,384 x K -> 2816, 4,096 x K -> 5632: K = 768, 497 / 468,
 * 517 / 432, 247 / 234; K = 1536, 799 / 870, 742 / 787, 393 / 421; level
 * around 1024). The second limit holds when db_gate and db_up are wanted,
 * whose sums cost the recomputing kernel more (K = 512, 404 / 400, 396 / 381,
 * 222 / 211; K = 768, 499 / 523, 467 / 466, 251 / 252). */
#define VECTRA_GATED_RECOMPUTE_K 768
#define VECTRA_GATED_RECOMPUTE_K_SUMS 512

/* Gradients of the above for dh [M,F]: dg = dh * up * act'(gate), du = dh *
 * act(gate), with gate and up as the forward saved them, or formed again
 * from x, the weights and the biases when both are NULL; dx = dg Wg + du Wu;
 * dw_gate = dg^T x, dw_up = du^T x; db_gate and db_up the sums of dg and du
 * (before their rounding) over rows. Unwanted results: data NULL
 * (dw_gate and dw_up together, db_gate and db_up together). dw_up directly
 * behind dw_gate in memory saves a pass over x. */
typedef struct {
  vectra_tensor dh, x, w_gate, w_up, b_gate, b_up, gate, up;
  vectra_tensor dx, dw_gate, dw_up, db_gate, db_up;
  int32_t activation;
  void* workspace;
  size_t workspace_bytes;
} vectra_gated_grad_args;

/* For each head vector v of q [B,Hq,N,D] and k [B,Hk,N,D] (any strides):
 *   n = v / sqrt(mean(v^2) + eps),   y = n * weight,
 * then the pairs (a, b) of y's first 2 R2 components turn by the angle of
 * the vector's position p: (a cos - b sin, b cos + a sin), with cos and sin
 * from row p of the tables [P, R2] (F32, 2 R2 <= D, unit inner stride).
 * Pairs are (i, i + R2), or (2i, 2i + 1) when interleaved.
 *  q_weight, k_weight [D]: q's dtype or F32; data NULL: no weight.
 *  positions: [B,N] int32 or int64 with any strides, or NULL: the token's
 *  index. A position outside [0, P) makes its vectors NaN.
 *  q_out, k_out: unit inner stride. */
typedef struct {
  vectra_tensor q, k, q_weight, k_weight, cos, sin;
  const void* positions;
  int32_t position_bytes;      /* 4 or 8 */
  int32_t interleaved;
  int64_t position_stride[2];  /* over B and N */
  double eps;
  vectra_tensor q_out, k_out;
} vectra_qk_args;

/* Gradients for dq_out, dk_out (any strides): dq, dk as in `fwd` (whose
 * q_out and k_out are not read), unit inner stride; dq_weight, dk_weight
 * [D] in their weights' dtype, data NULL when not wanted. */
typedef struct {
  vectra_qk_args fwd;
  vectra_tensor dq_out, dk_out, dq, dk, dq_weight, dk_weight;
  void* workspace;
  size_t workspace_bytes;
} vectra_qk_grad_args;

VECTRA_API int vectra_linear_forward(const vectra_linear_args* args, void* stream);
VECTRA_API int vectra_linear_backward(const vectra_linear_grad_args* args, void* stream);
VECTRA_API int vectra_gated_linear_forward(const vectra_gated_args* args, void* stream);
VECTRA_API int vectra_gated_linear_backward(const vectra_gated_grad_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_forward(const vectra_qk_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_backward(const vectra_qk_grad_args* args, void* stream);

/* Workspace of the call with these arguments, in bytes; a negative status
 * for invalid ones. */
VECTRA_API int64_t vectra_linear_forward_workspace_bytes(const vectra_linear_args* args);
VECTRA_API int64_t vectra_linear_backward_workspace_bytes(const vectra_linear_grad_args* args);
VECTRA_API int64_t vectra_gated_linear_forward_workspace_bytes(const vectra_gated_args* args);
VECTRA_API int64_t vectra_gated_linear_backward_workspace_bytes(const vectra_gated_grad_args* args);
VECTRA_API int64_t vectra_qk_norm_rope_backward_workspace_bytes(const vectra_qk_grad_args* args);

/* Message for a status of these calls. */
VECTRA_API const char* vectra_block_strerror(int status);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* VECTRA_BLOCK_H_ */
