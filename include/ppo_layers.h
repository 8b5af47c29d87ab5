/*
 * ppo_layers.h — C ABI of `libppo_layers.so`: the feed-forward layers of a
 * policy network on MI355X (gfx950), beside the PPO update of ppo_amd.h.
 *
 * Conventions are those of ppo_amd.h: device pointers owned by the caller,
 * every call only enqueues work on `stream` of the current device, dense
 * row-major layouts, PPO_OK or a PPO_ERR_* code (ppo_amd_strerror renders
 * it).  `workspace` is scratch of at least the matching *_workspace_bytes(),
 * 16-byte aligned, whose contents on entry do not matter and mean nothing
 * afterwards; calls that share one must be ordered.  No call keeps state, so
 * calls on different streams need no ordering as long as their outputs and
 * workspaces differ.
 *
 * Matrices are `dtype` (fp32, bf16 or fp16) with rows of any width and any
 * alignment; sums, activations and scales are held in fp32 and rounded once, to
 * nearest even.  The products take up to 2^26 rows of x and of each weight,
 * rows (of x and the weights, and of 2 F elements in the backward pass) below
 * 4 MiB, and up to 2^34 elements in a result: PPO_ERR_TOO_LARGE otherwise.
 */
#ifndef PPO_LAYERS_H
#define PPO_LAYERS_H

#include <stddef.h>
#include <stdint.h>

#include "ppo_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#define PPO_DTYPE_F32 0
#define PPO_DTYPE_BF16 1
#define PPO_DTYPE_F16 2

/*
 * Workspaces hold copies of operands whose rows do not start at multiples of 16
 * bytes.  Added to `dtype` (to `quantize` of the 8-bit product's
 * *_workspace_bytes), this says that x, xq and the weights themselves do, so
 * that no room for copies is needed unless the rows' length asks for it (x of
 * ppo_layer_int8_linear may start anywhere).  A call that adds it to operands
 * that start elsewhere gets PPO_ERR_INVALID_ARG.  Size function and call go
 * together: without it the workspace is that of operands at any address.
 */
#define PPO_LAYER_ALIGNED 0x100

/* The networks' activations (PPO_ACT_RELU, PPO_ACT_TANH) and two more. */
#define PPO_LAYER_RELU 0
#define PPO_LAYER_TANH 1
#define PPO_LAYER_SILU 2 /* g * sigmoid(g)                       */
#define PPO_LAYER_GELU 3 /* g * Phi(g), Phi the normal CDF       */

/*
 * Dropout from a counter-based generator.  Element (r, c) is kept where
 *   Philox4x32-7(key = seed, counter = (c / 4, id mod 2^32, id / 2^32, 0))[c % 4]
 *     < round((1 - p) * 2^32),      id = row_ids[r], or r without row_ids
 * and is then x / (1 - p); other elements are 0 (also where x is infinite or
 * NaN).  The mask is never stored: the gradient of y is this call on dy with
 * the same arguments.  `seed_at`, when not NULL, is a device pointer to the
 * seed (read when the kernel runs, so a replayed graph sees its current
 * value) and `seed` is ignored.  0 <= p <= 1.  y may be x itself.
 */
typedef struct ppo_dropout {
  double p;
  uint64_t seed;
  const uint64_t* seed_at;
  const int64_t* row_ids;
} ppo_dropout;

int ppo_layer_dropout(const void* x, void* y, int dtype, int64_t rows, int64_t cols,
                      const ppo_dropout* drop, void* stream);

/*
 * 8-bit rows: scale[r] = max_c |x[r,c]| times 1/127, both in fp32, and
 * q[r,c] = x[r,c] / scale[r] (in fp32) to the nearest integer, ties to even,
 * within [-127, 127].  A row of zeros has scale 0 and q = 0; a row that holds
 * an infinity or a NaN has scale NaN and q = 0, so that products with it are
 * NaN.
 */
int ppo_layer_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int8_t* q,
                            float* scale, void* stream);

/*
 * out[m,n] = (sum_k xq[m,k] * wq[n,k]) * xs[m] * ws[n] + bias[n], the sum
 * exact in int32 (K <= 2^17, else PPO_ERR_TOO_LARGE; at K = 2^17 a sum of
 * nothing but (-128)^2, which ppo_layer_quantize_rows never makes, would wrap),
 * scales and bias in fp32.  With x != NULL the rows of x (dtype) are quantised
 * first, as ppo_layer_quantize_rows does, and xq and xs are not read; out and
 * bias are of `dtype`.  bias may be NULL.
 */
size_t ppo_layer_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int quantize);
int ppo_layer_int8_linear(const void* x, const int8_t* xq, const float* xs, const int8_t* wq,
                          const float* ws, const void* bias, int dtype, int64_t M, int64_t N,
                          int64_t K, void* out, void* workspace, size_t workspace_bytes,
                          void* stream);

/*
 * The gated feed-forward block
 *   g = x wg^T + bg,  u = x wu^T + bu,  h = dropout(act(g) * u)
 * for x [M,D], wg and wu [F,D] (nn.Linear's layout), bg and bu [F] (both or
 * neither NULL), h [M,F].  drop may be NULL.  `saved`, when not NULL, is
 * fp32 [2][M][F4] with F4 = F rounded up to 4, 16-byte aligned, and receives
 * g and u for ppo_layer_gated_backward.
 */
size_t ppo_layer_gated_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t F);
int ppo_layer_gated_forward(const void* x, const void* wg, const void* wu, const void* bg,
                            const void* bu, int dtype, int64_t M, int64_t D, int64_t F,
                            int activation, const ppo_dropout* drop, void* h, float* saved,
                            void* workspace, size_t workspace_bytes, void* stream);

/*
 * Its backward pass: from dh [M,F] and the forward's `saved`,
 *   dh' = dropout(dh),  du = dh' * act(g),  dg = dh' * u * act'(g)
 *   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x,  dbg, dbu = column sums
 * Outputs that are NULL are not computed (dwg and dwu, and dbg and dbu, go
 * together).  M > 0 (over no rows the weights' gradients are the caller's
 * zeros).  dg and du are rounded to `dtype`, the matrix cores' operand
 * type, before the products: a 16-bit gradient is then off by about 1.4 times
 * what its own rounding makes (in short passes the products take what that
 * rounding left as well), and an fp16 dg or du past 65504 is infinite.  Sums
 * are split and joined in a fixed order: the same call gives the same bits (one
 * that asks for other outputs may cut the sums elsewhere).
 */
size_t ppo_layer_gated_backward_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t F);
int ppo_layer_gated_backward(const void* dh, const void* x, const void* wg, const void* wu,
                             const float* saved, int dtype, int64_t M, int64_t D, int64_t F,
                             int activation, const ppo_dropout* drop, void* dx, void* dwg,
                             void* dwu, void* dbg, void* dbu, void* workspace,
                             size_t workspace_bytes, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* PPO_LAYERS_H */
