"""Tokens sorted by expert and back, products over 16-bit weights, and their gradients.

- ``expert_sort``, ``tokens_to_experts``, ``tokens_from_experts`` and its backward,
  ``router_topk_backward`` (include/naiwa_tokens.h);
- ``Weights``, ``linear``, ``linear_input_grad``, ``linear_weight_grad``, ``act_backward``
  (include/naiwa_linear.h).

Arguments that name memory are device pointers or ``DeviceBuffer``s.  Calls on different streams need no order (long sorts and
products with parts of sums have scratch of the stream's own), replays of graphs that were captured on one stream do.  A training step of a
MoE layer over them: router_topk, expert_sort, tokens_to_experts, linear (gate and up),
linear (down), tokens_from_experts; then the backwards in the opposite order.
"""
from __future__ import annotations

import ctypes as C

from ._lib import ACT_NONE, F32, ROUTE_SOFTMAX_TOPK_RENORM, LinearWeights, check, lib
from .ops import _dev, _opt


class Weights:
    """16-bit weights [experts, n, k] on the device (rows ld values apart, experts stride apart; 0: packed),
    with an f32 bias [experts, n] or none."""

    def __init__(self, w, dtype: int, experts: int, n: int, k: int, bias=None, ld: int = 0, stride: int = 0):
        self.w, self.bias = w, bias          # kept while the descriptor is in use
        self.dtype, self.experts, self.n, self.k = dtype, experts, n, k
        self.desc = LinearWeights(_dev(w), _opt(bias), ld, stride, experts, n, k, dtype)


def _ref(w: Weights | None):
    return None if w is None else C.byref(w.desc)


def expert_sort(ids, T: int, k: int, E: int, perm, inv, offsets, mask=None, bad=None, ids_ld: int = 0,
                stream: int = 0) -> None:
    """The T * k pairs in the order of their experts: perm[row] = pair, inv[pair] = row (NO_ROW: masked or an id >= E),
    rows offsets[e] .. offsets[e + 1] - 1 are expert e's; all u32."""
    check(lib().naiwa_expert_sort(_dev(ids), ids_ld, T, k, E, _opt(mask), _dev(perm), _dev(inv), _dev(offsets), _opt(bad),
                                  stream), "naiwa_expert_sort")


def tokens_to_experts(x, dtype: int, inv, T: int, k: int, H: int, rows, ld: int = 0, rows_ld: int = 0,
                      stream: int = 0) -> None:
    """rows[inv[t, j]] = x[t]."""
    check(lib().naiwa_tokens_to_experts(_dev(x), dtype, ld, _dev(inv), T, k, H, _dev(rows), rows_ld, stream),
          "naiwa_tokens_to_experts")


def tokens_from_experts(y, dtype: int, inv, T: int, k: int, H: int, out, w=None, out_dtype: int | None = None,
                        accumulate: bool = False, ld: int = 0, w_ld: int = 0, out_ld: int = 0, stream: int = 0) -> None:
    """out[t] (+)= sum_j w[t, j] y[inv[t, j]] (w f32, None: 1); also the gradient of tokens_to_experts."""
    check(lib().naiwa_tokens_from_experts(_dev(y), dtype, ld, _dev(inv), _opt(w), w_ld, T, k, H, _dev(out),
                                          dtype if out_dtype is None else out_dtype, out_ld, 1 if accumulate else 0, stream),
          "naiwa_tokens_from_experts")


def tokens_from_experts_backward(dout, dout_dtype: int, y, dtype: int, inv, T: int, k: int, H: int, dy=None, dw=None, w=None,
                                 dout_ld: int = 0, ld: int = 0, w_ld: int = 0, dy_ld: int = 0, dw_ld: int = 0,
                                 stream: int = 0) -> None:
    """dy[inv[t, j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], y[inv[t, j]]> (f32)."""
    check(lib().naiwa_tokens_from_experts_backward(_dev(dout), dout_dtype, dout_ld, _opt(y), dtype, ld, _dev(inv), _opt(w),
                                                   w_ld, T, k, H, _opt(dy), dy_ld, _opt(dw), dw_ld, stream),
          "naiwa_tokens_from_experts_backward")


def router_topk_backward(logits, dtype: int, ids, dw, T: int, E: int, k: int, dlogits, mode: int = ROUTE_SOFTMAX_TOPK_RENORM,
                         mask=None, accumulate: bool = False, ld: int = 0, ids_ld: int = 0, dw_ld: int = 0, dld: int = 0,
                         stream: int = 0) -> None:
    """dlogits [T, E] (+)= the gradient of router_topk's weights, from theirs (dw f32 [T, k])."""
    check(lib().naiwa_router_topk_backward(_dev(logits), dtype, ld, _dev(ids), ids_ld, _dev(dw), dw_ld, T, E, k, mode,
                                           _opt(mask), _dev(dlogits), dld, 1 if accumulate else 0, stream),
          "naiwa_router_topk_backward")


def linear(w: Weights, x, rows: int, out, up: Weights | None = None, offsets=None, act: int = ACT_NONE, residual=None,
           out_dtype: int | None = None, pre=None, pre_up=None, x_ld: int = 0, residual_ld: int = 0, out_ld: int = 0,
           pre_ld: int = 0, stream: int = 0) -> None:
    """out [rows, n] = act(x W' + b) (* (x U' + c), up) + residual; pre and pre_up keep x W' + b and x U' + c."""
    check(lib().naiwa_linear(_ref(w), _ref(up), _dev(x), x_ld, _opt(offsets), rows, act, _opt(residual), residual_ld, _dev(out),
                             w.dtype if out_dtype is None else out_dtype, out_ld, _opt(pre), _opt(pre_up), pre_ld, stream),
          "naiwa_linear")


def linear_input_grad(w: Weights, dy, rows: int, dx, up: Weights | None = None, dy_up=None, offsets=None, act: int = ACT_NONE,
                      pre=None, pre_up=None, dx_up=None, dx_dtype: int | None = None, accumulate: bool = False,
                      dy_ld: int = 0, pre_ld: int = 0, dx_ld: int = 0, stream: int = 0) -> None:
    """dx [rows, k] (+)= dy W (+ dy_up U); with pre (and pre_up) the gradients of pre in dx (and of pre_up in dx_up), where
    x = act(pre) (* pre_up)."""
    check(lib().naiwa_linear_input_grad(_ref(w), _ref(up), _dev(dy), _opt(dy_up), dy_ld, _opt(offsets), rows, act, _opt(pre),
                                        _opt(pre_up), pre_ld, _dev(dx), _opt(dx_up), w.dtype if dx_dtype is None else dx_dtype,
                                        dx_ld, 1 if accumulate else 0, stream), "naiwa_linear_input_grad")


def linear_weight_grad(dy, x, dtype: int, rows: int, n: int, k: int, dw, experts: int = 1, offsets=None, dw_dtype: int = F32,
                       dbias=None, accumulate: bool = False, dy_ld: int = 0, x_ld: int = 0, ld: int = 0, stride: int = 0,
                       stream: int = 0) -> None:
    """dw [experts, n, k] (+)= dy' x and dbias f32 [experts, n] (+)= sum dy over every expert's rows."""
    check(lib().naiwa_linear_weight_grad(_opt(dy), dy_ld, _opt(x), x_ld, dtype, _opt(offsets), experts, rows, n, k, _dev(dw),
                                         dw_dtype, ld, stride, _opt(dbias), 1 if accumulate else 0, stream),
          "naiwa_linear_weight_grad")


def act_backward(dout, pre, dtype: int, rows: int, n: int, act: int, dpre, pre_up=None, dpre_up=None, ld: int = 0,
                 stream: int = 0) -> None:
    """dpre = dout act'(pre) (* pre_up) and dpre_up = dout act(pre)."""
    check(lib().naiwa_act_backward(_dev(dout), _dev(pre), _opt(pre_up), dtype, rows, n, ld, act, _dev(dpre), _opt(dpre_up),
                                   stream), "naiwa_act_backward")


__all__ = ["Weights", "expert_sort", "tokens_to_experts", "tokens_from_experts", "tokens_from_experts_backward",
           "router_topk_backward", "linear", "linear_input_grad", "linear_weight_grad", "act_backward"]
