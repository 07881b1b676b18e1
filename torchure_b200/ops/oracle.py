"""Plain PyTorch (fp32) statements of every hand-written op: the references the GPU tests compare against."""

from __future__ import annotations

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x: (..., S, hd) float; cos/sin: (S, hd)."""
    half = x.shape[-1] // 2
    rot = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * cos + rot * sin


def qknorm_rope(qkv, qw, kw, cos, sin, B, S, Hq, Hkv, hd, eps, use_norm=True):
    """qkv (B*S, (Hq+2Hkv)*hd) -> (B*S, (Hq+Hkv)*hd) fp32: per-head norm then RoPE on q and k."""
    x = qkv.float().view(B, S, Hq + 2 * Hkv, hd)
    q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv]
    if use_norm:
        q, k = rmsnorm(q, qw, eps), rmsnorm(k, kw, eps)
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    q = q * c + torch.cat((-q[..., hd // 2:], q[..., :hd // 2]), -1) * s
    k = k * c + torch.cat((-k[..., hd // 2:], k[..., :hd // 2]), -1) * s
    return torch.cat([q, k], dim=2).reshape(B * S, (Hq + Hkv) * hd)


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    g, u = gu.float().chunk(2, dim=-1)
    return F.silu(g) * u


def attention(q, k, v, causal=True):
    """q (B,S,Hq,hd), k/v (B,S,Hkv,hd) float -> (B,S,Hq,hd), lse (B,Hq,S) natural log."""
    B, S, Hq, hd = q.shape
    Hkv = k.shape[2]
    rep = Hq // Hkv
    qf, kf, vf = q.float().transpose(1, 2), k.float().transpose(1, 2), v.float().transpose(1, 2)
    kf, vf = kf.repeat_interleave(rep, 1), vf.repeat_interleave(rep, 1)
    s = qf @ kf.transpose(-1, -2) / hd ** 0.5
    if causal:
        s = s.masked_fill(~torch.ones(S, S, dtype=torch.bool, device=q.device).tril(), float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    o = torch.softmax(s, dim=-1) @ vf
    return o.transpose(1, 2), lse


def adamw(p, g, m, v, lr, b1, b2, eps, wd, step):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - (lr / (1 - b1 ** step)) * m / (v.sqrt() / (1 - b2 ** step) ** 0.5 + eps)
    return p, m, v


# ---- mixture of experts -----------------------------------------------------------------------------
def route(logits, k, capacity=0):
    """(weights, experts, slots, offsets, rows, counts, aux), weights and aux differentiable; ties go to the lowest index, a choice
    whose logit is -inf is not made, the choices of an expert beyond ``capacity`` (0: none) have no row."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    T, E = x.shape
    experts = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    top = x.gather(1, experts)
    made = top.detach() != float("-inf")
    closed = ~made.any(1, keepdim=True)              # no expert at all: zeros instead of 0 / 0
    weights = torch.softmax(torch.where(closed, torch.zeros_like(top), top), -1) * made
    p = torch.softmax(torch.where(closed, torch.zeros_like(x), x), -1) * ~closed
    of = torch.where(made, experts, E).reshape(-1)
    counts = torch.bincount(of, minlength=E + 1)[:E]
    kept = counts.clamp_max(capacity) if capacity else counts
    offsets = torch.cat([kept.new_zeros(1), kept.cumsum(0)])
    slots = torch.full((T * k,), -1, dtype=torch.int64, device=x.device)
    rows = torch.full((T * k,), -1, dtype=torch.int64, device=x.device)
    for e in range(E):
        mine = (of == e).nonzero()[:, 0][:int(kept[e])]
        slots[mine] = offsets[e] + torch.arange(mine.numel(), device=x.device)
        rows[offsets[e]:offsets[e + 1]] = mine
    aux = E * (counts.to(p.dtype) / max(1, T * k) * p.sum(0) / max(1, T)).sum()
    return weights, experts.int(), slots.view(T, k).int(), offsets.int(), rows.int(), counts.int(), aux


def grouped_linear(x, w, offsets):
    """Row r of x [R, K] times w[e]^T, w [E, N, K] in the type of x, for offsets[e] <= r < offsets[e + 1]; zeros behind offsets[E].
    Offsets count from 0, do not fall and stay within the rows; others are brought there."""
    edge = [0]
    for v in offsets[1:].tolist():
        edge.append(max(edge[-1], min(v, x.shape[0])))
    parts = [x[a:b] @ w[e].t().to(x.dtype) for e, (a, b) in enumerate(zip(edge[:-1], edge[1:]))]
    return torch.cat(parts + [x.new_zeros(x.shape[0] - edge[-1], w.shape[1])])


def dispatch(x, rows, k):
    return torch.where((rows >= 0)[:, None], x[rows.clamp_min(0).long() // k], torch.zeros((), dtype=x.dtype, device=x.device))


def combine(y, weights, slots):
    got = y[slots.clamp_min(0).long()] if y.shape[0] else y.new_zeros(*slots.shape, y.shape[1])
    got = torch.where((slots >= 0)[..., None], got, torch.zeros((), dtype=y.dtype, device=y.device))
    return (weights[..., None] * got).sum(1)


def expert_mlp(x, logits, w_gate_up, w_down, k, capacity=0, act_bits=16):
    """(out, aux) in the operands' precision."""
    weights, _, slots, offsets, rows, _, aux = route(logits, k, capacity)
    gu = grouped_linear(dispatch(x, rows, k), w_gate_up, offsets)
    act = swiglu_8bit(gu) if act_bits == 8 else swiglu_plain(gu)
    return combine(grouped_linear(act, w_down, offsets), weights.to(x.dtype), slots), aux


def swiglu_plain(gu):
    g, u = gu.chunk(2, dim=-1)
    return F.silu(g) * u


# ---- 8-bit activation checkpoints -------------------------------------------------------------------
ACT8_BLOCK = 64


def quantize8(x):
    """(int8 values, fp32 scales) of a matrix: blocks of 64 columns, halves away from zero."""
    rows, cols = x.shape
    n = -(-cols // ACT8_BLOCK)
    b = F.pad(x.float(), (0, n * ACT8_BLOCK - cols)).view(rows, n, ACT8_BLOCK)
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    some = finite & (top >= 2.0 ** -120)
    safe = torch.where(some, top, torch.ones_like(top))[..., None]
    q = torch.where(some[..., None], torch.floor(b.abs() * 127.0 / safe + 0.5) * b.sign(), torch.zeros_like(b))
    scales = torch.where(some, top / 127.0, torch.where(finite, torch.zeros_like(top), torch.full_like(top, float("nan"))))
    return q.view(rows, -1)[:, :cols].to(torch.int8).contiguous(), scales


def dequantize8(values, scales):
    rows, cols = values.shape
    return values.float() * scales.repeat_interleave(ACT8_BLOCK, dim=1)[:, :cols].reshape(rows, cols)


class _KeptIn8(torch.autograd.Function):
    """SwiGLU whose gradient is taken at gate and up as 8 bits stand for them."""

    @staticmethod
    def forward(ctx, gu):
        g, u = gu.chunk(2, dim=-1)
        ctx.kept = (*quantize8(g), *quantize8(u))
        return F.silu(g) * u

    @staticmethod
    def backward(ctx, dact):
        g, u = (dequantize8(*ctx.kept[i:i + 2]).to(dact.dtype) for i in (0, 2))
        s = torch.sigmoid(g)
        return torch.cat([dact * u * s * (1 + g * (1 - s)), dact * g * s], dim=-1)


def swiglu_8bit(gu):
    return _KeptIn8.apply(gu)
