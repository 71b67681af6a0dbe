/*
 * naiwa_linear.h -- products of rows with 16-bit weights: one matrix for all rows (a dense
 * projection, a shared expert), or an expert's matrix for each segment of rows sorted by
 * expert (naiwa_tokens.h), with bias, activation, gate and residual in the same pass; and
 * their gradients.
 *
 * With W [experts, n, k], rows m of expert e (all rows without offsets):
 *   p = x[m] W_e' + b_e                                      (k products summed in f32)
 *   out[m] = act(p) + residual[m]                            or, with a second matrix U:
 *   out[m] = act(p) q + residual[m],   q = x[m] U_e' + c_e   (act(gate) * up)
 * The input gradient of the same matrices is dy W_e (+ dy_up U_e); where x came out of a
 * product with an activation, the activation's gradient is taken in the same pass.  The
 * weights' gradient is sum_m dy[m]' x[m] over an expert's rows.
 *
 * Values are bf16 or f16 (x, the weights and the gradients the same), bias f32, out f32 or
 * the values' type.  Products are exact, sums f32 on the matrix cores, everything behind
 * them f32, each result rounded once.  A NaN or an infinity stays in the results that its
 * row and its weights have a part in.  Results do not depend on the run.  SiLU(v) is right to
 * (1.3 |v| + 6) 2^-24 of itself, GELU(v), with u = 1.6 (v + 0.045 v^3), to (8.3 |u| + 6) 2^-24 of itself:
 * as far as a few half steps of v move them; values below 2^-119 may be 0.
 *
 * offsets u32 [experts + 1] (device; NULL: one expert, all rows): rows offsets[e] ..
 * offsets[e + 1] - 1 are expert e's, at most `rows`; entries past `rows` count as `rows`.
 * Rows that are no expert's are left as they were and not read.  Row lengths are in values,
 * 0: tightly packed.  Sizes of any kind: rows, n and k need not be multiples of anything;
 * rows, weights and row lengths that are multiples of 16 bytes are faster.  Outputs may not overlap
 * inputs or each other, unless stated (NAIWA_E_INVALID); columns side by side in rows of one length in bytes (the
 * halves of a gate-and-up buffer) do not.  rows = 0 returns at once (naiwa_linear_weight_grad: with zeros
 * written).  rows <= 2^31 - 1 and row lengths (n and k with them) <= 2^21 (NAIWA_E_UNSUPPORTED),
 * experts <= 4096; and the tiles of a call have to fit one launch's 2^32 threads (NAIWA_E_UNSUPPORTED otherwise):
 * those of 2^29 rows of n <= 128 do, or 512 experts' weight gradients of n <= 128 and k <= 2^20.
 *
 * All three products leave parts of long sums in scratch where a call has few tiles: a buffer of the
 * stream's own, which only grows (to 64 MB; the first call that needs more allocates, with a device
 * sync), so that calls on different streams need no order.  Captured calls have another, which is kept
 * until the process ends and which all graphs captured on the stream (or on one made after its
 * destruction) share: their replays have to be ordered.  A stream is destroyed behind its calls.
 *
 * No counterpart in the reference, whose expert weights are quantised.
 */
#ifndef NAIWA_LINEAR_H
#define NAIWA_LINEAR_H

#include "naiwa_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NAIWA_ACT_NONE (-1) /* beside NAIWA_ACT_SILU and NAIWA_ACT_GELU_PYTORCH_TANH */

typedef struct naiwa_weights {
    const void* w;     /* weight (e, n, k) at w[e * stride + n * ld + k]; device       */
    const float* bias; /* f32 [experts, n], device, or NULL                              */
    int64_t ld;        /* values between rows (0: k)                                     */
    int64_t stride;    /* values between experts (0: n * ld)                              */
    int32_t experts;
    int32_t n;         /* output features                                                */
    int32_t k;         /* input features                                                 */
    int32_t dtype;     /* NAIWA_BF16 or NAIWA_F16                                         */
} naiwa_weights;

/* out [rows, n] as above.  up: U and c (the sizes and type of w), or NULL.  residual [rows, n]
 * of out's type or NULL; it may be out (with rows as far apart).  pre, pre_up [rows, n] of
 * the values' type (rows pre_ld apart): p and q rounded, what the gradient takes; either may be
 * NULL.  act: NAIWA_ACT_*. */
int naiwa_linear(const naiwa_weights* w, const naiwa_weights* up, const void* x, int64_t x_ld, const uint32_t* offsets,
                 int64_t rows, int act, const void* residual, int64_t residual_ld, void* out, int out_dtype,
                 int64_t out_ld, void* pre, void* pre_up, int64_t pre_ld, int64_t stream);

/* g = dy W_e (+ dy_up U_e), dy and dy_up [rows, n] (rows dy_ld apart); up and dy_up both or
 * neither.  Without pre: dx [rows, k] = g.  With pre [rows, k], what x was the activation of
 * (act; rows pre_ld apart): dx = g act'(pre); with pre_up too (x = act(pre) * pre_up): dx =
 * g pre_up act'(pre), the gradient of pre, and dx_up = g act(pre), that of pre_up.  dx and dx_up
 * (rows dx_ld apart) are f32 or the values' type (dx_dtype).  flags
 * NAIWA_LINEAR_ACCUMULATE (without pre): dx += g, in f32, rounded once. */
#define NAIWA_LINEAR_ACCUMULATE 1
int naiwa_linear_input_grad(const naiwa_weights* w, const naiwa_weights* up, const void* dy, const void* dy_up,
                            int64_t dy_ld, const uint32_t* offsets, int64_t rows, int act, const void* pre,
                            const void* pre_up, int64_t pre_ld, void* dx, void* dx_up, int dx_dtype, int64_t dx_ld,
                            int flags, int64_t stream);

/* dw [experts, n, k] (f32 or dtype: dw_dtype; ld and stride as in naiwa_weights) and dbias
 * f32 [experts, n] (NULL: not wanted) from dy [rows, n] and x [rows, k] of dtype.  Experts
 * without rows get zeros.  flags NAIWA_LINEAR_ACCUMULATE: dw += and dbias +=, in f32,
 * rounded once. */
int naiwa_linear_weight_grad(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype,
                             const uint32_t* offsets, int experts, int64_t rows, int n, int k, void* dw, int dw_dtype,
                             int64_t ld, int64_t stride, float* dbias, int flags, int64_t stream);

/* The activation's gradient alone: dpre = dout act'(pre), or with pre_up dpre = dout pre_up
 * act'(pre) and dpre_up = dout act(pre); all [rows, n] of dtype (f32, bf16 or f16), rows ld apart.
 * dpre may be dout or pre, dpre_up may be pre_up. */
int naiwa_act_backward(const void* dout, const void* pre, const void* pre_up, int dtype, int64_t rows, int n, int64_t ld,
                       int act, void* dpre, void* dpre_up, int64_t stream);

#ifdef __cplusplus
}
#endif
#endif
