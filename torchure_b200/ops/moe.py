"""Operators of a mixture-of-experts feed-forward: router, rows by expert and back, products grouped by expert.

``route``           top-k choice, weights, the order of rows by expert, the load-balancing term
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

    weights: torch.Tensor     # fp32 [T, k], sum 1 over the choices made; differentiable
    aux_loss: torch.Tensor    # fp32, 0-dim; differentiable
    experts: torch.Tensor     # int32 [T, k], falling logits
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


def route(logits: torch.Tensor, top_k: int, capacity: int = 0) -> Routing:
    """The ``top_k`` experts of every token by its logits [T, E] (fp32 or bf16, others in fp32; at most 384 experts, 16 choices).

    Ties go to the lowest index.  A weight is the softmax over the token's choices (the probabilities renormalised over them).  An
    expert whose logit is -inf is closed to the token: such a choice is not made (weight 0, no row), so a padding token can be kept
    out of every expert.  ``capacity``: rows an expert takes at most, the first in token order; 0: no limit.  ``aux_loss`` is
    E * sum_e (share of the choices, before the capacity, that went to e) * (mean probability of e)."""
    if not _plain(logits):
        return Routing(*_C().moe_route(logits, top_k, capacity, debug.enabled()))
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route: logits [tokens, experts] expected, got {logits.dtype} {tuple(logits.shape)}")
    if not 1 <= top_k <= logits.shape[1]:
        raise ValueError(f"route: top_k of {top_k} among {logits.shape[1]} experts")
    if capacity < 0:
        raise ValueError(f"route: capacity {capacity}")
    weights, experts, slots, offsets, rows, counts, aux = oracle.route(logits, top_k, capacity)
    return Routing(weights, aux, experts, slots, offsets, rows, counts)


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
               act_bits: int = 16) -> tuple[torch.Tensor, torch.Tensor]:
    """(out [T, D], aux_loss): every token through its ``top_k`` experts' SwiGLU feed-forwards, weighted by the router.

    x [T, D] bf16 or fp32 (the output's type), logits [T, E] as ``route`` takes them, ``w_gate_up`` [E, 2F, D] or the pair
    (w_gate, w_up) of [E, F, D], ``w_down`` [E, D, F]; matrices bf16 or fp32 (then rounded for the products, with fp32 gradients);
    D and F multiples of 8.  ``act_bits`` 8: gate and up are kept in 8 bits (``act8``) for the backward pass instead of bf16, which
    takes from them the gradients of gate and up and the activation, and with it the gradients of ``w_down`` and of the weights.

    On a GPU sums, weights and the weighted sum are fp32; what a product reads and writes between is bf16: the rows of x, the
    activation and, with more than 64 rows per expert on average, the down product's rows; in the backward pass the rows of the
    output's gradient and of dx, dout W_down, d(gate) | d(up) and the weighted activation.  Up to four tokens without gradients are
    rounded only at the end.  A pair, and fp32 matrices, are packed into one bf16 stack by every call, all experts of it, and the
    stack is held for the backward pass; bf16 matrices as [E, 2F, D] are read where they lie."""
    first, second = w_gate_up if isinstance(w_gate_up, (tuple, list)) else (w_gate_up, None)
    if not _plain(x, logits, first, w_down):
        if x.dim() != 2 or logits.dim() != 2:
            raise ValueError(f"expert_mlp: x [T, D] and logits [T, E] expected, got {tuple(x.shape)} and {tuple(logits.shape)}")
        out, aux = _C().expert_mlp(_rows(x), _rows(logits), first, second, w_down, top_k, capacity, act_bits, debug.enabled())
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
    wgu = first if second is None else torch.cat([first, second], dim=1)
    return oracle.expert_mlp(x, logits, wgu, w_down, top_k, capacity, act_bits)
