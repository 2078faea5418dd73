"""Mixture of experts on NVFP4 weights: the router, the experts' products, the way back.

    r = route(logits, top_k, scoring="sigmoid", bias=balance, groups=8, top_groups=4)
    h = expert_gemm(quantize_routed(x, r), r, w_up, w_up_sf, activation="swiglu", nvfp4_out=True)
    y = expert_gemm(h, r, w_down, w_down_sf)
    out = combine(y, r.rows, r.weights, residual=x)

or all of it in one call, :func:`expert_layer`.  Between the router and the combination there is one row per pair
(token, choice), in expert order: by expert, within an expert by token.  ``w`` [N, K/2, E] and ``w_sf``
[32, 4, N/128, 4, K/64, E] are laid out like ``b`` and ``sfb_permuted`` of :func:`submission.custom_kernel` with one batch entry per
expert.  Everything is enqueued on torch's current stream of the tensors' device and not waited for; nothing is kept
between calls.  All compute is in the CUDA library behind the C ABI; there is no PyTorch or CPU path, and no gradient.  The reference has one
dense product and no counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_SCORING = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}
_GROUP_SCORE = {"max": 1, "top2": 2}
_ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU, "swiglu": _lib.ACT_SWIGLU}


class Routing(NamedTuple):
    """Who goes where: ``experts`` and ``weights`` [T, k], ``rows`` [T, k] (row of each pair in expert order, -1 for none),
    ``offsets`` [E + 1] (first row of each expert, then the number of rows), and the plan of the grouped product."""
    experts: torch.Tensor
    weights: Optional[torch.Tensor]
    rows: torch.Tensor
    offsets: torch.Tensor
    plan: torch.Tensor
    num_experts: int


class RoutedRows(NamedTuple):
    """NVFP4 rows in expert order: packed e2m1 [T * k, K/2] and their scales, in the atoms of the routing's tiles."""
    packed: torch.Tensor
    sf: torch.Tensor


def _checked(result):
    if type(result) is int:
        _lib.check(result)
    return result


def _choice(table: dict, value, name: str) -> int:
    if value not in table:
        raise ValueError(f"{name} must be one of {', '.join(map(repr, table))} (got {value!r})")
    return table[value]


def route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1,
          group_score: str = "max", renormalize: bool = True, scale: float = 1.0) -> Routing:
    """The ``top_k`` experts of every token by router logits [T, E] (fp16, bf16 or fp32), and the plan of their products.

    Scores are the softmax over the experts or the sigmoid; experts are chosen by score + ``bias`` (fp32 [E]), largest first,
    ties to the lowest index.  With ``groups`` > 1 only experts of the ``top_groups`` best of that many equal ranges can be
    chosen; a range is judged by its largest choice (``group_score="max"``) or the sum of its two largest (``"top2"``).  Weights are the
    scores without bias, divided by their sum if ``renormalize`` (0 where that is 0), times ``scale``.
    An expert whose logit or bias is -inf or NaN cannot be chosen (+inf counts as the largest number); a token with fewer than
    ``top_k`` others gets expert -1, row -1 and weight 0 for the rest, so a padded token is one whose logits are all -inf.

    Choices are made in 64 bits.  Without ``bias``, and with groups judged by their largest choice if there are any, the logits
    themselves are compared, whose order both scores keep; so experts are told apart there whose scores 64 bits hold as one
    number (sigmoids from about 37 on, all 1; softmax scores more than 745 below the largest, all 0).  In every other case these
    are a tie, which the lowest index takes: a ``bias`` of zeros takes the lowest of them, no ``bias`` the one of the largest logit.
    Weights are made in 32 bits: that of a logit x is within ``(60 + 2 * abs(x - largest logit)) * 2**-24`` of its value by softmax,
    within ``20 * 2**-24`` by sigmoid, as long as it and the score that it is made of are normal numbers of 32 bits."""
    result = _lib.native().route(logits, top_k, _SCORING.get(scoring) or _choice(_SCORING, scoring, "scoring"), bias, groups, top_groups,
                                 _GROUP_SCORE.get(group_score) or _choice(_GROUP_SCORE, group_score, "group_score"), bool(renormalize), scale)
    if type(result) is int:
        _lib.check(result)
    return tuple.__new__(Routing, result)


def plan(experts: torch.Tensor, num_experts: int) -> Routing:
    """The routing for choices made elsewhere: int32 [T, k], each token's experts; what is not in [0, num_experts) counts as none.
    ``weights`` is None."""
    rows, offsets, plan_ = _checked(_lib.native().plan(experts, num_experts))
    return Routing(experts, None, rows, offsets, plan_, num_experts)


def quantize_routed(x: torch.Tensor, routing: Routing) -> RoutedRows:
    """Token rows [T, K] (fp16 or bf16) -> NVFP4 rows in expert order, by the rule of ``nvfp4_quantize``.

    Rows are quantised as they are: beyond 6 * 448 = 2688 values saturate without notice, and where a block of 16 has its maximum below
    6 * 2**-6 (0.094) its e4m3 scale is subnormal and loses bits.  Rows outside that range are the caller's to scale ahead of the call, and
    to undo in the product's ``alpha``."""
    return RoutedRows(*_checked(_lib.native().quantize_routed(x, routing.rows, routing.plan, routing.num_experts)))


def expert_gemm(rows: RoutedRows, routing: Routing, w: torch.Tensor, w_sf: torch.Tensor, *, alpha: Optional[torch.Tensor] = None,
                bias: Optional[torch.Tensor] = None, activation: str = "none", out_scale: float = 1.0, nvfp4_out: bool = False,
                out: Optional[torch.Tensor] = None):
    """Each expert's rows times its weights: ``out_scale * act(alpha[e] * rows @ w[e].T + bias[e])``, ``alpha`` fp32 [E], ``bias`` fp16 [E, N].

    ``activation``: "none", "relu", "silu", or "swiglu" for silu(gate) * up with N/2 columns, gate and up rows of ``w`` alternating in
    groups of eight (:func:`interleave_gate_up`).  Returns fp16 [T * k, columns] in expert order (``out``, if given), or with
    ``nvfp4_out`` the :class:`RoutedRows` of the following product, quantised from the fp16-rounded values (``out_scale`` brings
    small values into the scales' range; undo it in the following ``alpha``).  Rows of pairs that are none are left as they were.
    Results are fp16 whatever the type of the tokens, infinite beyond 65504; the NVFP4 form saturates at 2688.  "relu" keeps a NaN."""
    result = _checked(_lib.native().expert_gemm(rows[0], rows[1], routing.rows, routing.plan, routing.num_experts, w, w_sf, alpha, bias,
                                                _choice(_ACTIVATIONS, activation, "activation"), out_scale, bool(nvfp4_out), out))
    return RoutedRows(*result) if nvfp4_out else result[0]


def combine(y: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``residual[t] + sum_j weights[t, j] * y[rows[t, j]]``, summed in fp32 in the order of j and rounded once to ``dtype`` (fp16 or bf16;
    default: the type of ``out``, else of ``residual``, else fp16).  A row outside ``y`` adds nothing; ``out`` may be ``residual``, and is
    otherwise apart from what is read."""
    if dtype is None:
        dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.float16
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("combine writes fp16 or bf16")
    return _checked(_lib.native().combine(y, rows, weights, residual, out, dtype == torch.bfloat16))[0]


def expert_layer(x: torch.Tensor, logits: torch.Tensor, up, down, top_k: int, *, up_alpha=None, up_bias=None, down_alpha=None, down_bias=None,
                 activation: str = "swiglu", hidden_scale: float = 1.0, residual: Optional[torch.Tensor] = None, **router) -> torch.Tensor:
    """The feed-forward of a layer: route, quantise, up product (re-quantised), down product, combine, in x's type.

    ``up`` and ``down`` are (w, w_sf); ``router`` are the keywords of :func:`route`.  ``hidden_scale`` multiplies the hidden values
    before they are quantised; it is the caller's to undo in ``down_alpha``.  ``residual`` (usually the layer's input) is added.

    Ranges are those of the steps, also where x is bf16: x is quantised as it is (:func:`quantize_routed`), and the experts' rows between
    the down product and the combination are fp16, so what is beyond 65504 there is infinite in the result.  A smaller ``down_alpha``
    and a larger ``scale`` of the router bring such rows into range."""
    r = route(logits, top_k, **router)
    hidden = expert_gemm(quantize_routed(x, r), r, up[0], up[1], alpha=up_alpha, bias=up_bias, activation=activation, out_scale=hidden_scale,
                         nvfp4_out=True)
    y = expert_gemm(hidden, r, down[0], down[1], alpha=down_alpha, bias=down_bias)
    return combine(y, r.rows, r.weights, residual=residual, dtype=x.dtype)


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[F, ...] and [F, ...] -> [2 F, ...] with the rows of the two alternating in groups of eight: the order of rows that
    ``activation="swiglu"`` expects, before the weights (or their codes, plain scales or bias) are laid out.  F a multiple of 64."""
    if gate.shape != up.shape or gate.shape[0] % 64:
        raise ValueError("gate and up must have the same shape with a multiple of 64 rows")
    f = gate.shape[0]
    return torch.stack([gate.view(f // 8, 8, *gate.shape[1:]), up.view(f // 8, 8, *up.shape[1:])], 1).reshape(2 * f, *gate.shape[1:])


__all__ = ["Routing", "RoutedRows", "route", "plan", "quantize_routed", "expert_gemm", "combine", "expert_layer", "interleave_gate_up"]
