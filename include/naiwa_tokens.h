/*
 * naiwa_tokens.h -- a batch's tokens sorted by expert and back, the weights applied, and
 * the gradients: of the rows, of the routed weights and of the router's logits.
 *
 * A batch of T tokens with k experts each has T * k pairs (t, j); pair p = t k + j.
 * naiwa_expert_sort puts the pairs in the order of their experts (a stable sort: flat
 * order within an expert).  Row r of the sorted rows belongs to pair perm[r]; rows
 * offsets[e] .. offsets[e + 1] - 1 are expert e's; inv[p] is pair p's row.  Pairs of
 * masked tokens (mask[t] == 0) and pairs with an id >= E are in no segment: their inv is
 * NAIWA_NO_ROW, they read and write no sorted row and add nothing.
 *   to the experts    rows[inv[t,j]] = x[t]
 *   from the experts  out[t] = sum_j w[t,j] y[inv[t,j]]    (j ascending, in f32)
 *   its gradient      dy[inv[t,j]] = w[t,j] dout[t],  dw[t,j] = <dout[t], y[inv[t,j]]>
 * The gradient of "to the experts" is "from the experts" without weights.  Rows behind
 * offsets[E] are left as they were.  No counterpart in the reference, which groups pairs
 * inside its expert stages (src/moe/stages/gpu.rs:100-133) and does not train.
 *
 * Row values are f32, bf16 or f16; products and sums are f32, each result rounded once.
 * Results do not depend on the run.  Row lengths (ld) are in values, 0: tightly packed.
 * T * k <= 2^31 - 1, H <= 2^24, row lengths <= 2^28.  Inputs and outputs may not overlap
 * unless stated (NAIWA_E_INVALID); columns side by side in rows of one length in bytes do
 * not.  Calls of no tokens return at once (naiwa_expert_sort then sets its offsets to 0).
 * Sizes and pointers are checked (NAIWA_E_INVALID; NAIWA_E_UNSUPPORTED past a limit or for
 * another type); entries of inv and offsets that lie outside the T * k rows count as
 * NAIWA_NO_ROW.
 */
#ifndef NAIWA_TOKENS_H
#define NAIWA_TOKENS_H

#include "naiwa_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NAIWA_NO_ROW 0xffffffffu

/* ids u32 [T, k] (rows ids_ld entries apart, 0: k), mask u8 [T] or NULL ->
 * perm u32 [T * k] (the first offsets[E] entries are written), inv u32 [T, k], offsets
 * u32 [E + 1].  *bad (NULL: not reported) = ids >= E among the valid tokens.  E <= 4096,
 * T * k <= 2^31 - 1.  Calls of more than 4096 pairs use a scratch buffer of the stream's
 * own, which only grows; captured ones have another, which all graphs captured on the
 * stream (or on one made after its destruction) share: their replays have to be ordered.
 * A stream is destroyed behind its calls. */
int naiwa_expert_sort(const uint32_t* ids, int ids_ld, int64_t T, int k, int E, const uint8_t* mask, uint32_t* perm,
                      uint32_t* inv, uint32_t* offsets, uint32_t* bad, int64_t stream);

/* rows[inv[t,j]] = x[t]: x [T, H] and rows [T * k, H] of dtype. */
int naiwa_tokens_to_experts(const void* x, int dtype, int64_t ld, const uint32_t* inv, int64_t T, int k, int H,
                            void* rows, int64_t rows_ld, int64_t stream);

/* out[t] = sum_j w[t,j] y[inv[t,j]]: y [T * k, H] of dtype, w f32 [T, k] (rows w_ld
 * apart) or NULL (all 1), out [T, H] f32 or dtype (out_dtype).  A token without rows gets
 * zeros.  flags NAIWA_TOKENS_ACCUMULATE: the sum starts from out's value (tokens
 * without rows keep theirs). */
#define NAIWA_TOKENS_ACCUMULATE 1
int naiwa_tokens_from_experts(const void* y, int dtype, int64_t ld, const uint32_t* inv, const float* w, int w_ld,
                              int64_t T, int k, int H, void* out, int out_dtype, int64_t out_ld, int flags,
                              int64_t stream);

/* The gradient of naiwa_tokens_from_experts from dout [T, H] (f32 or dtype): dy [T * k, H]
 * of dtype and dw f32 [T, k] (0 where a pair has no row); either may be NULL, and y may be
 * when dw is.  dy may be y (with rows as far apart). */
int naiwa_tokens_from_experts_backward(const void* dout, int dout_dtype, int64_t dout_ld, const void* y, int dtype,
                                       int64_t ld, const uint32_t* inv, const float* w, int w_ld, int64_t T, int k,
                                       int H, void* dy, int64_t dy_ld, float* dw, int dw_ld, int64_t stream);

/* The gradient of naiwa_router_topk*'s weights with respect to the logits that it returned:
 * from dw f32 [T, k] (rows dw_ld apart), the chosen ids and the weights' mode, with p the
 * softmax over the chosen (NAIWA_ROUTE_SOFTMAX_TOPK_RENORM, NAIWA_ROUTE_TOPK_SOFTMAX) or
 * over all E (NAIWA_ROUTE_SOFTMAX_TOPK):
 *   dlogits[t, e] = p_e (sum_{j: ids[t,j] = e} dw[t,j] - sum_j p_{ids[t,j]} dw[t,j])
 * and 0 for the unchosen of the first two modes.  logits f32 or bf16 [T, E] (rows ld
 * apart), dlogits of the same type (rows dld apart; may be logits, with rows as far apart).
 * flags NAIWA_TOKENS_ACCUMULATE adds to dlogits (in f32, rounded once), beside
 * naiwa_router_balance_backward's share; masked rows are then left, else set to 0.
 * Ids >= E add nothing.  E <= 1024, k <= 32. */
int naiwa_router_topk_backward(const void* logits, int dtype, int ld, const uint32_t* ids, int ids_ld, const float* dw,
                               int dw_ld, int64_t T, int E, int k, int mode, const uint8_t* mask, void* dlogits,
                               int dld, int flags, int64_t stream);

#ifdef __cplusplus
}
#endif
#endif
