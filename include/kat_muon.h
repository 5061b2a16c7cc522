/*
 * kat_muon.h — C ABI of the orthogonalised matrix updates in libkat_rational.so (sm_100a:
 * tcgen05 MMA on pairs of fp16 planes with fp32 accumulators in tensor memory).
 *
 * An update u [r, c] is replaced by its Newton-Schulz polar factor.  With X = u / |u|_F on the
 * side with fewer rows (X = u^T where r > c), `steps` times
 *
 *     A = X X^T,   X <- a X + (b A + c A^2) X,   (a, b, c) = (3.4445, -4.7750, 2.0315)
 *
 * which takes every singular value into about 0.7 .. 1.2 (after five steps, from 1/500 of the
 * norm on).  A zero update stays zero; an update with a NaN or an infinity becomes NaN.
 *
 *   kat_orthogonalize:  out = X, in the input's type
 *   kat_muon_step:      m <- mu m + g;  u = g + mu m (nesterov) or m;
 *                       w <- (1 - lr wd) w - lr scale X(u)
 *
 * Small singular values grow by a^steps, and with them the rounding of the operands.  Every
 * matrix is therefore held as two fp16 planes (value x 2^14 = hi + lo, 22 bits), and a product
 * is hi hi + hi lo + lo hi in an fp32 accumulator; sums of more than 1024 terms are added up from
 * parts.  After five steps the result's relative error is about 1e-5 and at most 1e-4, for any type
 * and size (2e-6 and 7e-6 with fp32 products, whose sums are rounded where the tensor cores' are cut;
 * 2e-3 with single fp16 or bf16 operands).
 *
 * Conventions as in kat_rational.h: the caller owns every buffer, nothing is allocated, work is
 * enqueued on `stream` of the current device, argument errors are reported before anything is
 * enqueued.  The matrices of one call have one shape and are contiguous, r, c in [1, 65536]; the
 * pointer arrays are host memory and are read before the call returns.  Results are the same from
 * run to run and do not depend on what the other matrices hold; how many there are chooses the
 * tiles, and with them the order of some sums, within the error above.
 */
#ifndef KAT_MUON_H_
#define KAT_MUON_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Matrices one call takes at most. */
#define KAT_MUON_MAX_MATRICES 64

/* Workspace bytes for `count` matrices [rows, cols] (0 for arguments out of range). */
size_t kat_muon_workspace_bytes(int32_t count, int64_t rows, int64_t cols);

/* out[i] = the orthogonalised x[i], i < count; both of type `dtype` (KAT_DTYPE_*).  out[i] may
 * be x[i]. */
int kat_orthogonalize(const void* const* x, void* const* out, int32_t count, int64_t rows,
                      int64_t cols, int32_t dtype, int32_t steps, void* workspace,
                      size_t workspace_bytes, void* stream);

/* One optimizer step of `count` matrices: weights and gradients of type `dtype`, momenta fp32,
 * weights and momenta updated in place.  Where lr_device is not NULL the step size is read from
 * that fp32 device word when the kernels run, and `lr` is not used. */
int kat_muon_step(void* const* weights, const void* const* grads, float* const* momenta,
                  int32_t count, int64_t rows, int64_t cols, int32_t dtype, float lr,
                  const float* lr_device, float momentum, int32_t nesterov, float weight_decay,
                  float scale, int32_t steps, void* workspace, size_t workspace_bytes,
                  void* stream);

/* Sticky device status of these kernels (0 = no pipeline wait ran out), optionally reset to 0.
 * Synchronous. */
int kat_muon_device_status(int device, int reset, int* status);

#ifdef __cplusplus
}
#endif

#endif /* KAT_MUON_H_ */
