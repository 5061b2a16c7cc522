/*
 * kat_qk_norm_rope.h — C ABI of the per-head norm of queries and keys with the position
 * rotation, in one pass, in libkat_rational.so (sm_100a).
 *
 * Every head's vector x [D] of a token becomes
 *
 *     n = x r w,   r = 1 / sqrt(mean(x^2) + eps)
 *     y = R n      on the first rot_dim values, pair by pair
 *                  (y_a, y_b) = (n_a cos - n_b sin, n_a sin + n_b cos);  the others are n
 *
 * with pairs (i, i + rot_dim / 2), or (2i, 2i + 1) where `interleaved`.  cos and sin are fp32
 * tables [table_rows, rot_dim / 2]; token t of batch b takes row positions[b, t], or row t where
 * positions is NULL.  A position outside the table gives NaN in that token's outputs (forward)
 * and input gradients (backward) and adds NaN to the weights' gradients; no table row is read.
 * w may be NULL (no scaling).
 *
 * The backward recomputes r from x:  dn = R^T dy,  dw = sum over tokens and heads of dn x r,
 * dx = r (dn w - x r^2 mean(dn w x)).  Sums are fp32 within a thread and a block and fp64 over
 * the blocks, in a fixed order: the same bits from run to run.
 *
 * Tensors are [batch, tokens, heads, D] with the given strides (in elements); the D values of a
 * head are consecutive.  Queries and keys are two `kat_head_stream`s of one call and may have
 * different head counts.  The same rules as in kat_rational.h: nothing is allocated, work is
 * enqueued on `stream` of the current device, argument errors are reported before anything is
 * enqueued.  1 <= D <= 1024; rot_dim even, 0 <= rot_dim <= D; fewer than 2^31 heads in all tokens
 * of a stream.  Any alignment and strides are accepted; 16-byte aligned heads with D and rot_dim
 * multiples of 16, D <= 256, take the vector kernels.
 */
#ifndef KAT_QK_NORM_ROPE_H_
#define KAT_QK_NORM_ROPE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KAT_MAX_HEAD_STREAMS 3

typedef struct {
  const void* x;         /* input (NULL in the backward: dx is a copy of dy) */
  const void* dy;        /* backward: gradient of the output */
  void* out;             /* forward: y; backward: dx */
  const void* weight;    /* [D] of type weight_dtype, or NULL */
  float* dweight;        /* backward: [D], or NULL (not wanted) */
  int64_t x_stride[3];   /* batch, token, head */
  int64_t dy_stride[3];
  int64_t out_stride[3];
  int32_t heads;
} kat_head_stream;

typedef struct {
  int64_t batch, tokens;
  int32_t head_dim, rot_dim;
  int32_t interleaved;
  int32_t dtype;         /* of x, dy and out: KAT_DTYPE_* */
  int32_t weight_dtype;
  float eps;
  const float* cos_table;
  const float* sin_table;
  int64_t table_rows;
  const int64_t* positions;     /* [batch, tokens] or NULL */
  int64_t position_stride[2];
} kat_head_problem;

/* y of `count` streams (1 .. KAT_MAX_HEAD_STREAMS). */
int kat_qk_norm_rope_fwd(const kat_head_problem* problem, const kat_head_stream* streams,
                         int32_t count, void* stream);

/* Workspace bytes of the backward on `device` (partial sums of the weights' gradients). */
size_t kat_qk_norm_rope_bwd_workspace_bytes(int32_t head_dim, int32_t count, int device);

/* dx and dweight of `count` streams.  A stream without x copies dy to out: values that pass the
 * operator by, into the gradient they share with it. */
int kat_qk_norm_rope_bwd(const kat_head_problem* problem, const kat_head_stream* streams,
                         int32_t count, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KAT_QK_NORM_ROPE_H_ */
