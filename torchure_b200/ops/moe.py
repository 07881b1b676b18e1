"""Operators of a mixture-of-experts feed-forward: router, rows by expert and back, products grouped by expert.

``route``           top-k choice (by logits, or by scores with a bias and groups of experts), weights, the order of rows by expert, the
                    load-balancing term;   ``balance_bias_``  the bias of the next step
``dispatch``        token rows in expert order;   ``combine``  their weighted sums back in token order
``grouped_linear``  rows grouped by expert times each expert's matrix
``expert_mlp``      all of it: router, gate / up product, SwiGLU, down product, weighted sum, in one native call per direction

Rows of expert e are offsets[e] .. offsets[e + 1] - 1, in the order of (token, choice); ``offsets`` stays on the GPU, no call waits
for it.  Group sizes are free: an expert may have no rows, all of them, or any number between.  bf16 operands, fp32 sums; gradients
of bf16 matrices are bf16, of fp32 ones (rounded to bf16 for the products) fp32.

On tensors that are not on a GPU the plain statements of ``ops/oracle.py`` run, in the precision of the rows and at any width.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from torchure_b200 import ops
from torchure_b200.ops import debug, oracle
from torchure_b200.ops.kernels import _C

BF16 = torch.bfloat16


class Routing(NamedTuple):
    """What ``route`` found, T tokens and k choices each."""

    weights: torch.Tensor     # fp32 [T, k], sum 1 over the choices made (`normalize`; times `scale`); differentiable
    aux_loss: torch.Tensor    # fp32, 0-dim; differentiable
    experts: torch.Tensor     # int32 [T, k], falling logits (or biased scores)
    slots: torch.Tensor       # int32 [T, k]: row of the choice in expert order; -1: not made, or beyond the capacity
    offsets: torch.Tensor     # int32 [E + 1]: first row of each expert
    rows: torch.Tensor        # int32 [T k]: t k + j of each row; -1 behind offsets[E]
    counts: torch.Tensor      # int32 [E]: choices made for each expert, before the capacity


def _plain(*tensors: torch.Tensor) -> bool:
    """Whether the plain statements run: off the GPU, or with the kernels switched off."""
    if not ops.available():
        return True
    for t in tensors:
        if not t.is_cuda:
            return True
    return False


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


class Scoring(NamedTuple):
    """How ``route`` scores experts, where the softmax over the chosen logits is not what is wanted."""

    score: str = "softmax"            # or "sigmoid"
    bias: torch.Tensor | None = None  # fp32 [E], added to the scores for the choice only; no gradient
    groups: int = 1                   # experts in so many equal, consecutive groups
    top_groups: int = 1               # groups that stay open to a token
    normalize: bool = True            # weights over their sum
    scale: float = 1.0                # ... times this
    group_scores: int = 2             # a group counts by its so many largest scores, 1 or 2


def scoring(experts: int, top_k: int, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1, top_groups: int = 0,
            normalize: bool = True, scale: float = 1.0, group_scores: int = 2) -> Scoring | None:
    """The ``Scoring`` of these arguments for a router of so many experts, or None where they ask for the plain choice by logits."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f'route: scores are "softmax" or "sigmoid", not {score!r}')
    if groups < 1 or experts % groups:
        raise ValueError(f"route: {experts} experts in {groups} equal groups")
    if groups == 1 and top_groups in (0, 1):
        top_groups = 1
    elif not 1 <= top_groups <= groups:
        raise ValueError(f"route: {top_groups} of {groups} groups")
    if top_k > top_groups * (experts // groups):
        raise ValueError(f"route: top_k of {top_k} among {top_groups} groups of {experts // groups} experts")
    if not 0 < scale < float("inf"):
        raise ValueError(f"route: scale {scale}")
    if group_scores not in (1, 2):
        raise ValueError(f"route: the largest {group_scores} scores of a group (1 or 2 expected)")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (experts,)):
        raise ValueError(f"route: a bias of {experts} fp32 elements expected, got {bias.dtype} {tuple(bias.shape)}")
    if score == "softmax" and bias is None and groups == 1 and normalize and scale == 1.0:
        return None
    return Scoring(score, bias, groups, top_groups, bool(normalize), float(scale), int(group_scores))


_checked = scoring      # (where an argument has its name)


def _native(how: Scoring | None):
    return None if how is None else (how.score == "sigmoid", how.bias, how.groups, how.top_groups, how.normalize, how.scale, how.group_scores)


def route(logits: torch.Tensor, top_k: int, capacity: int = 0, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int = 0, normalize: bool = True, scale: float = 1.0, group_scores: int = 2) -> Routing:
    """The ``top_k`` experts of every token by its logits [T, E] (fp32 or bf16, others in fp32; at most 384 experts, 16 choices).

    Ties go to the lowest index.  A weight is the softmax over the token's choices (the probabilities renormalised over them).  An
    expert whose logit is -inf is closed to the token: such a choice is not made (weight 0, no row), so a padding token can be kept
    out of every expert.  ``capacity``: rows an expert takes at most, the first in token order; 0: no limit.  ``aux_loss`` is
    E * sum_e (share of the choices, before the capacity, that went to e) * (mean probability of e).

    ``score`` "sigmoid": an expert's score s is the sigmoid of its logit, not its softmax.  ``bias`` (fp32 [E]) is added to the scores for
    the choice alone, see ``balance_bias_``.  ``groups``: the experts lie in so many equal groups, at most 32, of which the ``top_groups``
    whose two largest (biased) scores have the largest sum are open to a token; with ``group_scores`` 1 those whose largest score is largest, the
    usual rule of routers without a bias.  With a bias or groups the choice goes by biased scores (each score
    rounded to fp32 once from 64 bits: a CPU and a GPU differ in about one of 2^22, by one unit), else by the logits.  ``normalize`` False: weights are the scores
    themselves, not divided by their sum over the choices; ``scale`` multiplies them.  The load-balancing term's probabilities are the
    scores over their sum.  A bias of -inf closes its expert to the choice."""
    how = None
    if not (score == "softmax" and bias is None and groups == 1 and top_groups == 0 and normalize and scale == 1.0
            and group_scores == 2) and logits.dim() == 2:
        how = scoring(logits.shape[1], top_k, score, bias, groups, top_groups, normalize, scale, group_scores)
    if not _plain(logits):
        return Routing(*_C().moe_route(logits, top_k, capacity, _native(how), debug.enabled()))
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route: logits [tokens, experts] expected, got {logits.dtype} {tuple(logits.shape)}")
    if not 1 <= top_k <= logits.shape[1]:
        raise ValueError(f"route: top_k of {top_k} among {logits.shape[1]} experts")
    if capacity < 0:
        raise ValueError(f"route: capacity {capacity}")
    found = oracle.route(logits, top_k, capacity) if how is None else oracle.route_scored(logits, top_k, capacity, *how)
    weights, experts, slots, offsets, rows, counts, aux = found
    return Routing(weights, aux, experts, slots, offsets, rows, counts)


def balance_bias_(bias: torch.Tensor, counts: torch.Tensor, rate: float) -> torch.Tensor:
    """``bias`` (fp32 [E], in place) for the next step: ``rate`` more for an expert with fewer choices than the mean of ``counts`` (int32 [E],
    ``Routing.counts``, of several ranks or micro-batches their sum), ``rate`` less for one with more."""
    if not _plain(bias, counts):
        return _C().moe_balance_bias(bias, counts, rate)
    if bias.dim() != 1 or bias.shape != counts.shape or counts.dtype != torch.int32 or bias.dtype != torch.float32:
        raise ValueError(f"balance_bias_: fp32 [E] and int32 [E] expected, got {bias.dtype} {tuple(bias.shape)} and {counts.dtype} "
                         f"{tuple(counts.shape)}")
    return bias.copy_(oracle.balance_bias(bias, counts, rate))


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The rows of x [T, D] (bf16 or fp32) in expert order, bf16 [T k, D]; zeros in rows of no choice."""
    if x.dim() != 2 or x.shape[0] != routing.slots.shape[0]:
        raise ValueError(f"dispatch: {routing.slots.shape[0]} tokens were routed, got {tuple(x.shape)}")
    if _plain(x, routing.rows):
        return oracle.dispatch(x, routing.rows, routing.slots.shape[1])
    return _C().moe_dispatch(x, routing.slots, routing.rows, debug.enabled())


def combine(y: torch.Tensor, routing: Routing, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Weighted sums of the rows y [T k, D] (bf16, expert order) for every token, [T, D] in bf16 or fp32 (None: y's type)."""
    if y.dim() != 2 or y.shape[0] != routing.slots.numel():
        raise ValueError(f"combine: {routing.slots.numel()} rows expected, got {tuple(y.shape)}")
    if _plain(y, routing.slots):
        wide = y.dtype if out_dtype is None else torch.promote_types(y.dtype, out_dtype)
        out = oracle.combine(y.to(wide), routing.weights.to(wide), routing.slots)
        return out if out_dtype is None else out.to(out_dtype)
    if out_dtype not in (None, BF16, torch.float32):
        raise TypeError(f"combine: sums in bf16 or fp32, not {out_dtype}")
    return _C().moe_combine(y, routing.weights, routing.slots, routing.offsets, out_dtype == torch.float32, debug.enabled())


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] @ w[e]^T for the rows offsets[e] <= r < offsets[e + 1] of x [R, K]; w [E, N, K]; [R, N].

    ``offsets`` int32 [E + 1], from 0 and not falling, on the same GPU; rows from offsets[E] on get zeros and no gradient.  x bf16
    of any strides; w bf16 or fp32; at most 384 experts."""
    if not _plain(x, w):
        return _C().grouped_linear(x, w, offsets, debug.enabled())
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"grouped_linear: rows {tuple(x.shape)} and matrices {tuple(w.shape)} do not fit")
    if offsets.shape != (w.shape[0] + 1,):
        raise ValueError(f"grouped_linear: {w.shape[0] + 1} offsets expected, got {tuple(offsets.shape)}")
    return oracle.grouped_linear(x, w, offsets)


def expert_mlp(x: torch.Tensor, logits: torch.Tensor, w_gate_up, w_down: torch.Tensor, top_k: int, capacity: int = 0,
               act_bits: int = 16, scoring: Scoring | None = None, counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out [T, D], aux_loss): every token through its ``top_k`` experts' SwiGLU feed-forwards, weighted by the router.

    x [T, D] bf16 or fp32 (the output's type), logits [T, E] as ``route`` takes them, ``w_gate_up`` [E, 2F, D] or the pair
    (w_gate, w_up) of [E, F, D], ``w_down`` [E, D, F]; matrices bf16 or fp32 (then rounded for the products, with fp32 gradients);
    D and F multiples of 8.  ``act_bits`` 8: gate and up are kept in 8 bits (``act8``) for the backward pass instead of bf16, which
    takes from them the gradients of gate and up and the activation, and with it the gradients of ``w_down`` and of the weights.
    ``scoring``: the further arguments of ``route``.  ``counts`` (int32 [E]): the choices made for each expert are added to it.

    On a GPU sums, weights and the weighted sum are fp32; what a product reads and writes between is bf16: the rows of x, the
    activation and, with more than 64 rows per expert on average, the down product's rows; in the backward pass the rows of the
    output's gradient and of dx, dout W_down, d(gate) | d(up) and the weighted activation.  Up to four tokens without gradients are
    rounded only at the end.  A pair, and fp32 matrices, are packed into one bf16 stack by every call, all experts of it, and the
    stack is held for the backward pass; bf16 matrices as [E, 2F, D] are read where they lie."""
    first, second = w_gate_up if isinstance(w_gate_up, (tuple, list)) else (w_gate_up, None)
    if scoring is not None and logits.dim() == 2:
        scoring = _checked(logits.shape[1], top_k, *scoring)
    if not _plain(x, logits, first, w_down):
        if x.dim() != 2 or logits.dim() != 2:
            raise ValueError(f"expert_mlp: x [T, D] and logits [T, E] expected, got {tuple(x.shape)} and {tuple(logits.shape)}")
        out, aux = _C().expert_mlp(_rows(x), _rows(logits), first, second, w_down, top_k, capacity, _native(scoring),
                                   counts, act_bits, debug.enabled())
        return out, aux
    if x.dim() != 2 or logits.dim() != 2 or first.dim() != 3 or w_down.dim() != 3:
        raise ValueError("expert_mlp: x [T, D], logits [T, E], w_gate_up [E, 2F, D] and w_down [E, D, F] expected")
    if act_bits not in (8, 16):
        raise ValueError(f"expert_mlp: activations are kept in 8 or 16 bits, not {act_bits}")
    if not 1 <= top_k <= logits.shape[1] or capacity < 0:
        raise ValueError(f"expert_mlp: top_k of {top_k} among {logits.shape[1]} experts, capacity {capacity}")
    if second is not None and (first.shape != second.shape or first.dtype != second.dtype):
        raise ValueError("expert_mlp: w_gate and w_up differ")
    E, D, f = w_down.shape
    if first.shape != (E, 2 * f if second is None else f, D) or x.shape[1] != D or logits.shape != (x.shape[0], E):
        raise ValueError(f"expert_mlp: x {tuple(x.shape)}, logits {tuple(logits.shape)}, w_gate_up {tuple(first.shape)}, w_down "
                         f"{tuple(w_down.shape)} do not fit")
    if counts is not None and (counts.shape != (E,) or counts.dtype != torch.int32):
        raise ValueError(f"expert_mlp: counts int32 [{E}] expected, got {counts.dtype} {tuple(counts.shape)}")
    wgu = first if second is None else torch.cat([first, second], dim=1)
    return oracle.expert_mlp(x, logits, wgu, w_down, top_k, capacity, act_bits, scoring, counts)
