"""Operators of a mixture-of-experts feed-forward: router, rows by expert and back, products grouped by expert.

``route``           top-k choice, weights, the order of rows by expert, the load-balancing term
``dispatch``        token rows in expert order;   ``combine``  their weighted sums back in token order
``grouped_linear``  rows grouped by expert times each expert's matrix
``expert_mlp``      all of it: router, gate / up product, SwiGLU, down product, weighted sum, in one native call per direction

Rows of expert e are offsets[e] .. offsets[e + 1] - 1, in the order of (token, choice); ``offsets`` stays on the GPU, no call waits
for it.  Group sizes are free: an expert may have no rows, all of them, or any number between.  bf16 operands, fp32 sums; gradients
of bf16 matrices are bf16, of fp32 ones (rounded to bf16 for the products) fp32.

On tensors that are not on a GPU the plain statements of ``ops/oracle.py`` run, in the operands' precision.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F

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


def _kernels(*tensors: torch.Tensor) -> bool:
    return ops.available() and all(t.is_cuda for t in tensors)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, capacity):
        out = _C().moe_route(logits, k, capacity, debug.tracker())
        ops.count_launch()
        weights, _, experts, slots, offsets, rows, counts = out
        ctx.save_for_backward(logits, weights, experts, counts)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(experts, slots, offsets, rows, counts)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, daux, *_):
        logits, weights, experts, counts = ctx.saved_tensors
        if dweights is None and daux is None:
            return None, None, None
        dl = _C().moe_route_bwd(logits, weights, experts, counts, None if dweights is None else dweights.float().contiguous(),
                                None if daux is None else daux.float(), debug.tracker())
        ops.count_launch()
        return dl, None, None


def route(logits: torch.Tensor, top_k: int, capacity: int = 0) -> Routing:
    """The ``top_k`` experts of every token by its logits [T, E] (fp32 or bf16; at most 384 experts, 16 choices).

    Ties go to the lowest index.  A weight is the softmax over the token's choices (the probabilities renormalised over them).  An
    expert whose logit is -inf is closed to the token: such a choice is not made (weight 0, no row), so a padding token can be kept
    out of every expert.  ``capacity``: rows an expert takes at most, the first in token order; 0: no limit.  ``aux_loss`` is
    E * sum_e (share of the choices, before the capacity, that went to e) * (mean probability of e)."""
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route: logits [tokens, experts] expected, got {logits.dtype} {tuple(logits.shape)}")
    if not 1 <= top_k <= logits.shape[1]:
        raise ValueError(f"route: top_k of {top_k} among {logits.shape[1]} experts")
    if capacity < 0:
        raise ValueError(f"route: capacity {capacity}")
    if not _kernels(logits):
        weights, experts, slots, offsets, rows, counts, aux = oracle.route(logits, top_k, capacity)
        return Routing(weights, aux, experts, slots, offsets, rows, counts)
    if logits.dtype not in (BF16, torch.float32):
        logits = logits.float()
    return Routing(*_Route.apply(_rows(logits), top_k, capacity))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, rows):
        ctx.save_for_backward(slots)
        ctx.f32 = x.dtype == torch.float32
        out = _C().moe_gather(x, rows, slots.shape[1], debug.tracker())
        ops.count_launch()
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxg):
        slots, = ctx.saved_tensors
        dx = _C().moe_combine(dxg.contiguous(), None, slots, ctx.f32, debug.tracker())
        ops.count_launch()
        return dx, None, None


def _check_tokens(x: torch.Tensor, routing: Routing, what: str) -> None:
    if x.dim() != 2 or x.shape[0] != routing.slots.shape[0]:
        raise ValueError(f"{what}: {routing.slots.shape[0]} tokens were routed, got {tuple(x.shape)}")


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The rows of x [T, D] (bf16 or fp32) in expert order, bf16 [T k, D]; zeros in rows of no choice."""
    _check_tokens(x, routing, "dispatch")
    if not _kernels(x, routing.rows):
        return oracle.dispatch(x, routing.rows, routing.slots.shape[1])
    if x.dtype not in (BF16, torch.float32):
        raise TypeError(f"dispatch: bf16 or fp32 expected, got {x.dtype}")
    return _Dispatch.apply(_rows(x), routing.slots, routing.rows)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots, offsets, f32):
        ctx.save_for_backward(y, weights, slots, offsets)
        out = _C().moe_combine(y, weights, slots, f32, debug.tracker())
        ops.count_launch()
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights, slots, offsets = ctx.saved_tensors
        dy, dw = _C().moe_combine_bwd(_rows(dout), y, weights, slots, offsets, debug.tracker())
        ops.count_launch()
        return dy, dw, None, None, None


def combine(y: torch.Tensor, routing: Routing, out_dtype: torch.dtype = BF16) -> torch.Tensor:
    """Weighted sums of the rows y [T k, D] (bf16, expert order) for every token, [T, D] in bf16 or fp32."""
    T, k = routing.slots.shape
    if y.dim() != 2 or y.shape[0] != T * k:
        raise ValueError(f"combine: {T * k} rows expected, got {tuple(y.shape)}")
    if not _kernels(y, routing.slots):
        return oracle.combine(y, routing.weights.to(y.dtype), routing.slots)
    if y.dtype != BF16 or out_dtype not in (BF16, torch.float32):
        raise TypeError(f"combine: bf16 rows to bf16 or fp32 sums expected, got {y.dtype} to {out_dtype}")
    return _Combine.apply(y.contiguous(), routing.weights.contiguous(), routing.slots, routing.offsets, out_dtype == torch.float32)


def _operand(x: torch.Tensor) -> torch.Tensor:
    """x [R, K] as the products read it: rows contiguous, a row stride and a base on 16 bytes, columns in eights."""
    if x.shape[1] % 8 == 0 and x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1] and x.data_ptr() % 16 == 0:
        return x
    return F.pad(x, (0, -x.shape[1] % 8)).contiguous() if x.shape[1] % 8 else x.clone(memory_format=torch.contiguous_format)


def _matrices(w: torch.Tensor) -> torch.Tensor:
    """w [E, N, K] in bf16 as the products read it: both widths in eights (zeros behind)."""
    w = w if w.dtype == BF16 else w.to(BF16)
    n, k = -w.shape[1] % 8, -w.shape[2] % 8
    w = F.pad(w, (0, k, 0, n)) if n or k else w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        wb, xb = _matrices(w), _operand(x)
        y = _C().grouped_gemm(xb, wb, offsets, False, debug.tracker())
        ops.count_launch()
        ctx.save_for_backward(xb, wb, offsets)
        ctx.shape, ctx.f32 = tuple(w.shape), w.dtype == torch.float32
        return y[:, :w.shape[1]]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xb, wb, offsets = ctx.saved_tensors
        _, n, k = ctx.shape
        dyb = _operand(dy)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = _C().grouped_gemm(dyb, wb, offsets, True, debug.tracker())[:, :k]
            ops.count_launch()
        if ctx.needs_input_grad[1]:
            dw = _C().grouped_wgrad(dyb, xb, offsets, ctx.f32, debug.tracker())[:, :n, :k]
            ops.count_launch()
        return dx, dw, None


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] @ w[e]^T for the rows offsets[e] <= r < offsets[e + 1] of x [R, K]; w [E, N, K]; [R, N].

    ``offsets`` int32 [E + 1], from 0 and not falling, on the same GPU; rows from offsets[E] on get zeros and no gradient.  x bf16
    of any strides; w bf16 or fp32."""
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"grouped_linear: rows {tuple(x.shape)} and matrices {tuple(w.shape)} do not fit")
    if offsets.shape != (w.shape[0] + 1,):
        raise ValueError(f"grouped_linear: {w.shape[0] + 1} offsets expected, got {tuple(offsets.shape)}")
    if not _kernels(x, w):
        return oracle.grouped_linear(x, w, offsets)
    if x.dtype != BF16 or w.dtype not in (BF16, torch.float32):
        raise TypeError(f"grouped_linear: bf16 rows and bf16 or fp32 matrices expected, got {x.dtype} and {w.dtype}")
    if offsets.dtype != torch.int32 or offsets.device != x.device or w.device != x.device:
        raise ValueError("grouped_linear: int32 offsets and matrices on the GPU of the rows expected")
    return _GroupedLinear.apply(x, w, offsets.contiguous())


class _ExpertMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, logits, w_gate_up, w_up, w_down, k, capacity, bits):
        f32 = w_down.dtype == torch.float32
        if w_up is None:
            wgu = w_gate_up.to(BF16).contiguous()
        else:
            e, f, d = w_up.shape
            wgu = torch.empty(e, 2 * f, d, dtype=BF16, device=w_up.device)
            wgu[:, :f].copy_(w_gate_up)
            wgu[:, f:].copy_(w_up)
        wd = w_down.to(BF16).contiguous()
        keep = any(ctx.needs_input_grad)
        (out, aux, weights, experts, slots, offsets, rows, counts, gu, q, scales), n = _C().expert_mlp_fwd(
            x, logits, wgu, wd, k, capacity, bits, keep, debug.tracker())
        ops.count_launch(n)
        if keep:
            ctx.save_for_backward(x, logits, wgu, wd, weights, experts, slots, offsets, rows, counts, gu, q, scales)
            ctx.f32, ctx.pair = f32, w_up is not None
            ctx.set_materialize_grads(False)
        return out, aux

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, daux):
        x, logits, wgu, wd, weights, experts, slots, offsets, rows, counts, gu, q, scales = ctx.saved_tensors
        if dout is None:
            if daux is None:
                return (None,) * 8
            dl = _C().moe_route_bwd(logits, weights, experts, counts, None, daux.float(), debug.tracker())
            ops.count_launch()
            return (None, dl) + (None,) * 6
        (dx, dl, dwgu, dwd), n = _C().expert_mlp_bwd(_rows(dout), None if daux is None else daux.float(), x, logits, wgu, wd, weights,
                                                     experts, slots, offsets, rows, counts, gu, q, scales, ctx.f32, debug.tracker())
        ops.count_launch(n)
        f = wd.shape[2]
        first, second = (dwgu[:, :f], dwgu[:, f:]) if ctx.pair else (dwgu, None)
        return dx, dl, first, second, dwd, None, None, None


def expert_mlp(x: torch.Tensor, logits: torch.Tensor, w_gate_up, w_down: torch.Tensor, top_k: int, capacity: int = 0,
               act_bits: int = 16) -> tuple[torch.Tensor, torch.Tensor]:
    """(out [T, D], aux_loss): every token through its ``top_k`` experts' SwiGLU feed-forwards, weighted by the router.

    x [T, D] bf16 or fp32 (the output's type), logits [T, E] as ``route`` takes them, ``w_gate_up`` [E, 2F, D] or the pair
    (w_gate, w_up) of [E, F, D], ``w_down`` [E, D, F]; matrices bf16 or fp32 (then rounded for the products, with fp32 gradients);
    D and F multiples of 8.  ``act_bits`` 8: gate and up are kept in 8 bits (``act8``) for the backward pass instead of bf16."""
    pair = isinstance(w_gate_up, (tuple, list))
    first, second = w_gate_up if pair else (w_gate_up, None)
    if x.dim() != 2 or logits.dim() != 2 or first.dim() != 3 or w_down.dim() != 3:
        raise ValueError("expert_mlp: x [T, D], logits [T, E], w_gate_up [E, 2F, D] and w_down [E, D, F] expected")
    if act_bits not in (8, 16):
        raise ValueError(f"expert_mlp: activations are kept in 8 or 16 bits, not {act_bits}")
    if not 1 <= top_k <= logits.shape[1] or capacity < 0:
        raise ValueError(f"expert_mlp: top_k of {top_k} among {logits.shape[1]} experts, capacity {capacity}")
    if pair and (first.shape != second.shape or first.dtype != second.dtype):
        raise ValueError("expert_mlp: w_gate and w_up differ")
    E, D, f = w_down.shape
    if first.shape != (E, f if pair else 2 * f, D) or x.shape[1] != D or logits.shape != (x.shape[0], E):
        raise ValueError(f"expert_mlp: x {tuple(x.shape)}, logits {tuple(logits.shape)}, w_gate_up {tuple(first.shape)}, w_down "
                         f"{tuple(w_down.shape)} do not fit")
    if not _kernels(x, logits, first, w_down):
        wgu = torch.cat([first, second], dim=1) if pair else first
        return oracle.expert_mlp(x, logits, wgu, w_down, top_k, capacity, act_bits)
    if any(t.dtype not in (BF16, torch.float32) for t in (x, logits, first, w_down)) or first.dtype != w_down.dtype:
        raise TypeError("expert_mlp: bf16 or fp32 tensors expected, the matrices of one type")
    if D % 8 or f % 8:
        raise ValueError(f"expert_mlp: widths in multiples of 8 expected, got D {D} and F {f}")
    return _ExpertMlp.apply(_rows(x), _rows(logits), first, second, w_down, top_k, capacity, act_bits)
