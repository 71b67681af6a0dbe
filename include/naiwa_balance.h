/*
 * naiwa_balance.h -- how evenly a router spreads its tokens: per-expert counts, the
 * balance loss of a batch, and the loss's gradient with respect to the router's logits.
 *
 * With V the valid tokens (mask[t] != 0; all without a mask), N their number, c_e the
 * times expert e was chosen among them, p_t = softmax(logits_t) over all E experts and
 * P_e = 1/N sum_{t in V} p_te:
 *   loss = E / (k N) sum_e c_e P_e            (1 for an even spread; 0 when N = 0)
 *   dloss/dlogits_tj = E / (k N^2) p_tj (c_j - sum_e c_e p_te) for t in V, else 0
 * (the counts are constants of the gradient).  The logits and ids are what
 * naiwa_router_topk* return.  The counts are also what naiwa_cache_seed_hits takes to
 * seed an expert cache from a prompt.  No counterpart in the reference, which serves
 * models and does not train them.
 *
 * Sums are deterministic: counts are integers, and P is added up in f32 over 64 rows
 * at most and beyond that in f64, in an order that depends on the sizes alone (and on
 * whether logits lie so that 4 can be read at once).  The entry points share one
 * grow-only scratch buffer per device: calls on different streams have to be ordered, and
 * a graph's replays and other calls.  Captured calls keep the buffer that they were given.
 */
#ifndef NAIWA_BALANCE_H
#define NAIWA_BALANCE_H

#include "naiwa_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* counts[e] = entries of ids [T, k] (rows ids_ld entries apart, 0: k) equal to e among
 * the valid tokens; mask u8 [T] or NULL.  Ids >= E are counted in *bad (NULL: not
 * reported) and nowhere else.  E <= 1024, T * k <= 2^31 - 1. */
int naiwa_expert_counts(const uint32_t* ids, int ids_ld, int64_t T, int k, int E, const uint8_t* mask,
                        uint32_t* counts, uint32_t* bad, int64_t stream);

/* counts [E], *valid = N, probs [E] = P and *loss of a batch: logits [T, E] f32 or
 * bf16 (dtype), rows ld values apart (0: E); ids as above (ids >= E add to no count).
 * T = 0 gives zeros.  A valid token's row with a NaN or +inf gives NaN in P and the
 * loss, and so does one of nothing but -inf; other -inf logits have probability 0.  What
 * masked rows hold does not matter.  E <= 1024. */
int naiwa_router_balance(const void* logits, int dtype, int ld, const uint32_t* ids, int ids_ld, int64_t T, int E,
                         int k, const uint8_t* mask, uint32_t* counts, uint32_t* valid, float* probs, float* loss,
                         int64_t stream);

/* dlogits [T, E] (the logits' dtype, rows dld values apart, 0: E) = *grad_loss (device
 * f32) times dloss/dlogits, from the forward's counts and valid.  flags
 * NAIWA_BALANCE_ACCUMULATE adds to dlogits (in f32, rounded once) instead of
 * overwriting; masked rows are then left as they are, otherwise set to 0.  dlogits may
 * be logits, with rows as far apart (NAIWA_E_INVALID otherwise). */
#define NAIWA_BALANCE_ACCUMULATE 1
int naiwa_router_balance_backward(const void* logits, int dtype, int ld, const uint32_t* counts,
                                  const uint32_t* valid, int64_t T, int E, int k, const uint8_t* mask,
                                  const float* grad_loss, void* dlogits, int dld, int flags, int64_t stream);

#ifdef __cplusplus
}
#endif
#endif
