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


class _Embedding(torch.autograd.Function):
    """Rows in fp32 (or the table's wider type), scaled and rounded once; a row's gradient likewise."""

    @staticmethod
    def forward(ctx, ids, table, scale, padding, dtype):
        if ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < table.shape[0]):
            raise IndexError(f"embedding: ids from {int(ids.min())} to {int(ids.max())} in a table of {table.shape[0]} rows")
        ctx.save_for_backward(ids)
        ctx.how = table.shape, table.dtype, scale, padding
        wide = torch.promote_types(table.dtype, torch.float32)
        return (table[ids.long()].to(wide) * scale).to(dtype)

    @staticmethod
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        shape, dtype, scale, padding = ctx.how
        wide = torch.promote_types(dtype, torch.float32)
        d = torch.zeros(shape, dtype=wide, device=dout.device)
        d.index_add_(0, ids.reshape(-1).long(), dout.reshape(ids.numel(), shape[1]).to(wide))
        d = d * scale
        if padding is not None:
            d[padding] = 0
        return None, d.to(dtype), None, None, None


def embedding(ids, table, scale=1.0, padding=None, dtype=None):
    return _Embedding.apply(ids, table, scale, padding, table.dtype if dtype is None else dtype)


# ---- moments in 8 bits --------------------------------------------------------------------------------
# A block of 128 values shares the scale a / TOP, a its largest magnitude.  y = |x| TOP / a + FIRST is held as its fp32 pattern cut to 3 bits
# of mantissa, counted from FIRST's.  First moment: 7 bits and a sign; second moment: 8 bits.  A value goes to one of its two neighbours
# by 16 random bits, so that the mean is its own; a second moment above zero keeps at least the first step.  fp32, one rounding for each
# operation: the kernel's results have the same bits.
STATE8_BLOCK = 128
_S8 = {True: (2.0 ** -15, 896, 127, 1.875 - 2.0 ** -15), False: (2.0 ** -31, 768, 255, 1.875)}      # FIRST, its pattern >> 20, last code, TOP
_LOW32 = 0xFFFFFFFF


def _mix32(x):
    x = (x ^ (x >> 16)) * 0x7FEB352D & _LOW32
    x = (x ^ (x >> 15)) * 0x846CA68B & _LOW32
    return x ^ (x >> 16)


def state8_key(seed: int, step: int) -> int:
    return _mix32((seed + 0x9E3779B9 * step) & _LOW32)


def state8_bits(n: int, key: int, index: int, device) -> torch.Tensor:
    """32 random bits (int64) for each of the n values of tensor number `index`: the lower 16 for the first moment."""
    i = torch.arange(n, device=device)
    if n <= 1 << 32:
        return _mix32((i & _LOW32) ^ _mix32((key + 0x85EBCA6B * index) & _LOW32))
    return _mix32((i & _LOW32) ^ _mix32((key + 0x85EBCA6B * index + 0xC2B2AE35 * (i >> 32)) & _LOW32))


def _blocks128(x):
    x = x.reshape(-1)
    return F.pad(x, (0, -x.numel() % STATE8_BLOCK)).view(-1, STATE8_BLOCK)


def state8_encode(x, bits, signed):
    """(uint8 codes of x's shape, fp32 scales) of x in fp32; `bits`: 0 to 65535 for each value (32768: nearly to the nearest)."""
    first, base, last, most = _S8[signed]
    b = _blocks128(x)
    top = b.abs().amax(-1, keepdim=True) if x.numel() else b.new_zeros(b.shape[0], 1)
    y = b.abs() * (top.reciprocal() * most) + first
    code = ((y.view(torch.int32) + (_blocks128(bits) << 4).int()) >> 20) - base
    code = code.clamp_max(last)
    code = torch.where(torch.signbit(b), code + 128, code) if signed else torch.where(b > 0, code.clamp_min(1), code)
    tiny = top < 2.0 ** -100
    fine = (top < float("inf")) & ~tiny
    code = torch.where(fine, code, torch.zeros_like(code))
    scale = torch.where(fine, top * torch.tensor(1.0 / most, dtype=torch.float32, device=x.device),
                        torch.where(tiny, torch.zeros_like(top), torch.full_like(top, float("nan"))))
    return code.view(-1)[:x.numel()].view(x.shape).to(torch.uint8), scale.view(-1)


def state8_decode(codes, scales, signed):
    first, base, _, _ = _S8[signed]
    c = _blocks128(codes).int()
    y = ((((c & 127) if signed else c) + base << 20).view(torch.float32) - first) * scales[:, None]
    if signed:
        y = torch.where(c >= 128, -y, y)
    return y.view(-1)[:codes.numel()].view(codes.shape)


def adamw8(params, grads, ms, m_scales, vs, v_scales, shadows, lr, b1, b2, eps, wd, step, grad_scale=None, maximize=False, seed=0, numbers=None):
    """AdamW in place with moments in 8 bits."""
    numbers = range(len(params)) if numbers is None else numbers
    size, root, key = lr / (1.0 - b1 ** step), (1.0 - b2 ** step) ** -0.5, state8_key(seed, step)
    for i, p, g, mc, msc, vc, vsc, sh in zip(numbers, params, grads, ms, m_scales, vs, v_scales, shadows, strict=True):
        g = g.float()
        if grad_scale is not None:
            g = g * grad_scale.float()
        if maximize:
            g = -g
        m = state8_decode(mc, msc, True) * b1 + g * (1.0 - b1)
        v = state8_decode(vc, vsc, False) * b2 + (g * (1.0 - b2)) * g
        # correctly rounded (a CPU's fp32 root need not be), and not of zero: no 0 / 0 with eps 0
        r = torch.sqrt(v.clamp_min(2.0 ** -126).double()).float()
        p.copy_(p * (1.0 - lr * wd) - (m / (r * root + eps)) * size)
        if sh is not None:
            sh.copy_(p)
        bits = state8_bits(p.numel(), key, i, p.device).view(p.shape)
        for x, r, codes, scales, signed in ((m, bits & 0xFFFF, mc, msc, True), (v, bits >> 16, vc, vsc, False)):
            c, s = state8_encode(x, r, signed)
            codes.copy_(c)
            scales.copy_(s)


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
    slots, offsets, rows, counts = _plan_rows(experts, made, E, capacity)
    aux = E * (counts.to(p.dtype) / max(1, T * k) * p.sum(0) / max(1, T)).sum()
    return weights, experts.int(), slots, offsets, rows, counts.int(), aux


def _plan_rows(experts, made, E, capacity):
    """(slots, offsets, rows, counts) of choices [T, k]: rows in the order of (expert, token, choice)."""
    T, k = experts.shape
    of = torch.where(made, experts, E).reshape(-1)
    counts = torch.bincount(of, minlength=E + 1)[:E]
    kept = counts.clamp_max(capacity) if capacity else counts
    offsets = torch.cat([kept.new_zeros(1), kept.cumsum(0)])
    slots = torch.full((T * k,), -1, dtype=torch.int64, device=of.device)
    rows = torch.full((T * k,), -1, dtype=torch.int64, device=of.device)
    for e in range(E):
        mine = (of == e).nonzero()[:, 0][:int(kept[e])]
        slots[mine] = offsets[e] + torch.arange(mine.numel(), device=of.device)
        rows[offsets[e]:offsets[e + 1]] = mine
    return slots.view(T, k).int(), offsets.int(), rows.int(), counts


def route_scored(logits, k, capacity=0, score="softmax", bias=None, groups=1, top_groups=1, normalize=True, scale=1.0, group_scores=2):
    """``route`` by scores: s = sigmoid or softmax of the logits, rounded to fp32 from 64 bits for the choice; with a bias or groups the choice goes
    by s + bias inside the ``top_groups`` groups whose two largest have the largest sums (``group_scores`` 1: whose largest is largest), else by the
    logits."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    T, E = x.shape
    lowest = torch.full((), float("-inf"), device=x.device)
    low = x.detach()
    is_open = low != lowest
    closed = ~is_open.any(1, keepdim=True)             # no expert at all: zeros instead of 0 / 0
    safe = torch.where(closed, torch.zeros_like(x), x)
    if bias is None and groups == 1:
        key = low
    else:
        wide = safe.detach().double()
        s = (torch.sigmoid(wide) if score == "sigmoid" else torch.softmax(wide, -1)).float()
        key = torch.where(is_open, s if bias is None else s + bias.detach(), lowest)
    if groups > 1:
        two = key.view(T, groups, E // groups).sort(-1, descending=True).values[..., :2]
        one = group_scores == 1 or two.shape[-1] == 1
        total = two[..., 0] if one else torch.where(two[..., 1] == lowest, two[..., 0], two.sum(-1))
        best = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :top_groups]
        stays = torch.zeros(T, groups, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        key = torch.where(stays.repeat_interleave(E // groups, 1), key, lowest)
    experts = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    made = key.gather(1, experts) != lowest
    # logarithms of the scores: they may all be tiny
    log_s = F.logsigmoid(safe) if score == "sigmoid" else torch.log_softmax(safe, -1)
    top = log_s.gather(1, experts)
    none = ~made.any(1, keepdim=True)
    if normalize:
        weights = torch.softmax(torch.where(none, torch.zeros_like(top), torch.where(made, top, lowest)), -1) * made
    else:
        weights = torch.where(made, torch.exp(top), torch.zeros_like(top))
    p = torch.softmax(log_s, -1) * ~closed
    slots, offsets, rows, counts = _plan_rows(experts, made, E, capacity)
    aux = E * (counts.to(p.dtype) / max(1, T * k) * p.sum(0) / max(1, T)).sum()
    return scale * weights, experts.int(), slots, offsets, rows, counts.int(), aux


def balance_bias(bias, counts, rate):
    n = counts.long()
    return bias + rate * torch.sign(n.sum() - n * n.numel()).to(bias.dtype)


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


def expert_mlp(x, logits, w_gate_up, w_down, k, capacity=0, act_bits=16, scoring=None, counts=None):
    """(out, aux) in the operands' precision.  scoring: the further arguments of ``route_scored``."""
    weights, _, slots, offsets, rows, made, aux = route(logits, k, capacity) if scoring is None else route_scored(logits, k, capacity, *scoring)
    if counts is not None:
        counts += made
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
