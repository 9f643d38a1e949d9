/*
 * vectra_block.h: C ABI of the transformer-block operators that stand
 * around RBF attention (libvectra_rbf.so).
 *
 *  - vectra_linear_*:        y = act(x W^T + b) + r
 *  - vectra_gated_linear_*:  h = act(x Wg^T + bg) * (x Wu^T + bu)
 *  - vectra_qk_norm_rope_*:  the RMS norm of every query and key head vector
 *                            and the rotation of its position, in one pass
 *                            (vectra_qk_norm_rope_axes_*: of its positions
 *                            on several axes)
 *  - vectra_dropout:         zeros a share of a tensor by a mask that is a
 *                            function of an element's index
 *  - vectra_residual_norm_*: x_out = a x + gate dropout(norm(branch)) and the
 *                            next sublayer's norm of x_out, in one pass
 *  - vectra_cross_attention_*: RBF attention to an encoder's states, of
 *                            another length, with shared key heads
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

/* qk_norm_rope with positions on up to VECTRA_MAX_AXES axes: positions[axis]
 * starts `stride` elements behind positions[axis - 1], and the R2 pairs
 * belong to the axes in order, section[axis] of them to each: pair i turns by
 * entry i of the table row that its axis' position names. A position outside
 * [0, P) on any axis makes its vectors NaN. */
#define VECTRA_MAX_AXES 4
typedef struct {
  int32_t count;                       /* 1 to VECTRA_MAX_AXES */
  int32_t section[VECTRA_MAX_AXES];    /* not negative, sum R2 */
  int64_t stride;
} vectra_qk_axes;
typedef struct {
  vectra_qk_args qk; /* positions must not be NULL */
  vectra_qk_axes axes;
} vectra_qk_axes_args;
typedef struct {
  vectra_qk_grad_args qk;
  vectra_qk_axes axes;
} vectra_qk_axes_grad_args;

/* Dropout. Element e of a tensor, counted in row-major order of its sizes
 * (whatever its strides), is kept when its 16-bit random number is at least
 * cut = round(65536 p), and then scaled by 65536 / (65536 - cut); the others
 * become 0, whatever they hold. The random numbers are those of Philox4x32-10
 * (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) with
 * the key rng[0] (its low, then its high half) and the counter
 * (e / 8 low half, e / 8 high half, rng[1] low half, stream): number e % 8 is
 * the low (even) or high half of output word (e % 8) / 2. */
typedef struct {
  double p;             /* 0 to 1 */
  const int64_t* rng;   /* device memory: seed, step. NULL: p is 0 */
  uint32_t stream;      /* keeps the masks of one step apart */
} vectra_drop;

/* y = dropout(x), which is also its own gradient.
 *  x [M,C], one of F32 / F16 / BF16, any strides; y [M,C] contiguous. */
typedef struct {
  vectra_tensor x, y;
  vectra_drop drop;
} vectra_dropout_args;

/* u = norm(branch) * branch_weight  (branch_weight's data NULL: u = branch)
 * x_out = residual_scale x + gate * dropout(u)
 * y = norm(x_out) * weight + bias
 * with norm(v) = v / sqrt(mean(v^2) + eps) over C, of v - mean(v) first when
 * `kind` is VECTRA_NORM_LAYER.
 *  x, branch [M,C]: one dtype of F32 / F16 / BF16, any strides. branch's data
 *  NULL: x_out is x itself and not written; residual_scale must be 1 and p 0
 *  then, gate and branch_weight NULL.
 *  weight, bias, branch_weight [C] (data NULL: none), gate [G,C] (NULL: 1)
 *  with M a multiple of G: row r takes gate row r / (M / G).
 *  x_out, y [M,C]: contiguous. y's data NULL: no second norm (weight and bias
 *  NULL then). The norm is of x_out before its rounding.
 *  stats [M,4] F32, contiguous, on a 16-byte boundary: mean and factor of the
 *  second norm, mean and factor of the first, for the backward pass; data NULL:
 *  not wanted.
 * C is at most 16384. */
typedef enum { VECTRA_NORM_RMS = 0, VECTRA_NORM_LAYER = 1 } vectra_norm_kind;
typedef struct {
  vectra_tensor x, branch, weight, bias, branch_weight, gate;
  vectra_tensor x_out, y, stats;
  vectra_drop drop;
  double residual_scale, eps;
  int32_t kind; /* vectra_norm_kind */
} vectra_residual_norm_args;

/* The same for a backward pass to come. rest [M,C], of 16-bit tensors with a
 * branch and y only, contiguous, their type: what x_out's rounding left, itself
 * rounded (of F16 2^11 times that, which stays in its range). The second norm's
 * gradient takes x_out less its mean, and a mean of many deviations would
 * multiply that rounding. Data NULL: not wanted. */
typedef struct {
  vectra_residual_norm_args fwd;
  vectra_tensor rest;
} vectra_residual_norm_train_args;

/* Gradients of the above for dx_out and dy [M,C] (any strides; dx_out's data
 * NULL: zero; dy's: y had none, its norm is left out). Of fwd, x_out and
 * stats are read as the forward wrote them (x_out is x, strides and all, where
 * there was no branch), branch, weight, branch_weight and gate as it read
 * them. x, y and bias are not read, x_out only with dy, stats only with dy or
 * branch_weight, branch only with branch_weight or dgate.
 *  dx, dbranch [M,C], dgate [G,C], dweight, dbias, dbranch_weight [C]:
 *  contiguous; data NULL when not wanted. */
typedef struct {
  vectra_residual_norm_args fwd;
  vectra_tensor dx_out, dy;
  vectra_tensor dx, dbranch, dweight, dbias, dbranch_weight, dgate;
  void* workspace;
  size_t workspace_bytes;
} vectra_residual_norm_grad_args;

/* The same with the forward's rest (data NULL where it wrote none, or without
 * dy); vectra_residual_norm_backward takes x_out as it was rounded. */
typedef struct {
  vectra_residual_norm_grad_args grad;
  vectra_tensor rest;
} vectra_residual_norm_train_grad_args;

/* out[b,h,i] = sum over j < len_b of softmax_j(-scale |q_i - k_j|^2) v_j, with
 * q of head h and k, v of head h / (H / Hk).
 *  q [B,H,Nq,D], k [B,Hk,Nk,D], v [B,Hk,Nk,Dv]: one dtype of F32 / F16 / BF16,
 *  any strides; H a multiple of Hk; D and Dv at most 256.
 *  scale [B|1,H|1,1,1]: any float type; zero and negative values are legal.
 *  key_lengths [B]: int32 or int64, or NULL: Nk. Values outside [0, Nk] count
 *  as the nearer end. Keys and values at or past a length are never used; a
 *  sequence of length 0 has zero results (and gradients).
 *  out [B,H,Nq,Dv]: unit inner stride.
 * For the backward pass (data NULL: not wanted):
 *  lse [B,H,Nq] F32, contiguous: log2 of the sum of each row's weights before
 *  division (in 16-bit types without their common factor exp(-scale |q|^2)),
 *  infinity for a sequence of length 0.
 *  rest [B,H,Nq,Dv], of 16-bit tensors only, contiguous, their type: what out's
 *  rounding left, itself rounded (of F16 2^11 times that). The backward pass
 *  subtracts numbers that are nearly equal where a row has one large weight,
 *  and out alone would decide their difference. */
typedef struct {
  vectra_tensor q, k, v, scale;
  const void* key_lengths;
  int32_t length_bytes;  /* 4 or 8 */
  int64_t length_stride;
  vectra_tensor out, lse, rest;
  void* workspace;
  size_t workspace_bytes;
} vectra_cross_args;

/* Gradients for dout [B,H,Nq,Dv] (any strides), with out, lse and rest as the
 * forward wrote them:
 *  dq, dk, dv: as q, k and v, unit inner stride; rows of dk and dv at or past
 *  the length are zero. dscale [B,H] F32, contiguous. data NULL when not
 *  wanted (dk and dv together). */
typedef struct {
  vectra_cross_args fwd;
  vectra_tensor dout, dq, dk, dv, dscale;
  void* workspace;
  size_t workspace_bytes;
} vectra_cross_grad_args;

VECTRA_API int vectra_linear_forward(const vectra_linear_args* args, void* stream);
VECTRA_API int vectra_linear_backward(const vectra_linear_grad_args* args, void* stream);
VECTRA_API int vectra_gated_linear_forward(const vectra_gated_args* args, void* stream);
VECTRA_API int vectra_gated_linear_backward(const vectra_gated_grad_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_forward(const vectra_qk_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_backward(const vectra_qk_grad_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_axes_forward(const vectra_qk_axes_args* args, void* stream);
VECTRA_API int vectra_qk_norm_rope_axes_backward(const vectra_qk_axes_grad_args* args, void* stream);
VECTRA_API int vectra_dropout(const vectra_dropout_args* args, void* stream);
VECTRA_API int vectra_residual_norm_forward(const vectra_residual_norm_args* args, void* stream);
VECTRA_API int vectra_residual_norm_forward_train(const vectra_residual_norm_train_args* args, void* stream);
VECTRA_API int vectra_residual_norm_backward(const vectra_residual_norm_grad_args* args, void* stream);
VECTRA_API int vectra_residual_norm_backward_train(const vectra_residual_norm_train_grad_args* args, void* stream);
VECTRA_API int vectra_cross_attention_forward(const vectra_cross_args* args, void* stream);
VECTRA_API int vectra_cross_attention_backward(const vectra_cross_grad_args* args, void* stream);

/* Workspace of the call with these arguments, in bytes; a negative status
 * for invalid ones. */
VECTRA_API int64_t vectra_linear_forward_workspace_bytes(const vectra_linear_args* args);
VECTRA_API int64_t vectra_linear_backward_workspace_bytes(const vectra_linear_grad_args* args);
VECTRA_API int64_t vectra_gated_linear_forward_workspace_bytes(const vectra_gated_args* args);
VECTRA_API int64_t vectra_gated_linear_backward_workspace_bytes(const vectra_gated_grad_args* args);
VECTRA_API int64_t vectra_qk_norm_rope_backward_workspace_bytes(const vectra_qk_grad_args* args);
VECTRA_API int64_t vectra_qk_norm_rope_axes_backward_workspace_bytes(const vectra_qk_axes_grad_args* args);
VECTRA_API int64_t vectra_residual_norm_backward_workspace_bytes(const vectra_residual_norm_grad_args* args);
VECTRA_API int64_t vectra_residual_norm_backward_train_workspace_bytes(const vectra_residual_norm_train_grad_args* args);
VECTRA_API int64_t vectra_cross_attention_forward_workspace_bytes(const vectra_cross_args* args);
VECTRA_API int64_t vectra_cross_attention_backward_workspace_bytes(const vectra_cross_grad_args* args);

/* Message for a status of these calls. */
VECTRA_API const char* vectra_block_strerror(int status);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* VECTRA_BLOCK_H_ */
