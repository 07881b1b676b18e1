"""The operators of the mixture-of-experts feed-forward and of 8-bit activation checkpoints, as measured cases.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``exact`` the same from the definitions in 64 bits and ``work`` what a pass cannot do without.  With
``own`` false ``run`` is made of plain tensor operations in 32 bits, with ``own`` true of this package's entry points.

Kinds:

``route``    top-k choice of experts with its plan (row order, offsets, slots), the load-balancing term and the gradient of both.
``grouped``  rows grouped by expert times each expert's matrix; with ``train`` the gradients of rows and matrices as well.
``experts``  the whole feed-forward: routing, gather, gate / up product, SwiGLU, down product, weighted sum; with ``train`` the
             gradients of tokens, logits and both stacks of matrices.
``swiglu8``  SwiGLU whose backward pass reads gate and up from 8 bits: activation and gradient.
``store8``   an activation written as 8 bits and read back.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 64            # values that share a scale


def listed():
    return [
        # one token of a served mixture, 8 experts
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 8, "k": 2, "factor": 0.0, "half": False, "masked": False},
        # many small experts, odd token count, mixed precision logits, some experts closed to some tokens
        {"name": "route_many", "kind": "route", "tokens": 16389, "experts": 128, "k": 8, "factor": 1.5, "half": True, "masked": True},
        # serving a handful of tokens: a few rows for each expert, bound by the matrices
        {"name": "grouped_few", "kind": "grouped", "rows": 16, "experts": 8, "inner": 1024, "outer": 1536, "empty": 0, "train": False},
        # odd sizes all round, a quarter of the experts without rows
        {"name": "grouped_odd", "kind": "grouped", "rows": 1003, "experts": 16, "inner": 520, "outer": 776, "empty": 4, "train": True},
        # a micro-batch's rows through a bank of many experts, forward and both gradients
        {"name": "grouped_batch", "kind": "grouped", "rows": 32768, "experts": 32, "inner": 1024, "outer": 1536, "empty": 1, "train": True},
        # one token through the shipped mixture's feed-forward
        {"name": "experts_token", "kind": "experts", "tokens": 1, "experts": 8, "k": 2, "width": 1024, "units": 1536, "factor": 0.0, "train": False},
        # the tokens of a small served batch
        {"name": "experts_few", "kind": "experts", "tokens": 61, "experts": 16, "k": 4, "width": 1024, "units": 768, "factor": 0.0, "train": False},
        # the shipped mixture's layer in a training step
        {"name": "experts_batch", "kind": "experts", "tokens": 8192, "experts": 8, "k": 2, "width": 1024, "units": 1536, "factor": 1.25, "train": True},
        # gate and up of that layer's rows, kept in 8 bits for the backward pass
        {"name": "swiglu8_batch", "kind": "swiglu8", "rows": 16384, "units": 1536},
        # odd: rows and units that fill no block
        {"name": "swiglu8_odd", "kind": "swiglu8", "rows": 333, "units": 1000},
        # a layer input's checkpoint
        {"name": "store8_batch", "kind": "store8", "rows": 16384, "cols": 2560},
        # a short, odd one
        {"name": "store8_odd", "kind": "store8", "rows": 77, "cols": 519},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["route", "grouped", "experts", "swiglu8", "store8"])
    if kind == "route":
        experts = _log(rng, 2, 256)
        return {"kind": kind, "tokens": _log(rng, 1, max(1, min(32768, 2097152 // experts))), "experts": experts,
                "k": rng.randint(1, min(8, experts)), "factor": rng.choice([0.0, 1.0, 1.25, 2.0]), "half": rng.random() < 0.5,
                "masked": rng.random() < 0.4}
    if kind == "grouped":
        rows, experts = _log(rng, 1, 16384), _log(rng, 2, 64)
        return {"kind": kind, "rows": rows, "experts": experts, "inner": 8 * _log(rng, 16, 160), "outer": 8 * _log(rng, 16, 192),
                "empty": rng.randint(0, experts // 4), "train": rows > 64 and rng.random() < 0.6}
    if kind == "experts":
        tokens, experts = _log(rng, 1, 4096), _log(rng, 4, 64)
        return {"kind": kind, "tokens": tokens, "experts": experts, "k": rng.randint(1, 4), "width": 8 * _log(rng, 32, 128),
                "units": 8 * _log(rng, 32, 128), "factor": rng.choice([1.0, 1.25]) if tokens > 256 else 0.0,
                "train": tokens > 64 and rng.random() < 0.6}
    if kind == "swiglu8":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "units": _log(rng, 64, 1536)}
    return {"kind": kind, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 2560)}


def _capacity(case):
    """Rows that an expert takes at most; 0: as many as there are."""
    if not case["factor"]:
        return 0
    return max(1, int(case["factor"] * case["tokens"] * case["k"] / case["experts"] + 0.999))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    def router_logits(tokens, experts, dtype):
        # a learned router prefers some experts: a bias of its own for each
        bias = torch.randn(experts, device="cuda", generator=g) * 0.3
        return (torch.randn(tokens, experts, device="cuda", generator=g) + bias).to(dtype)

    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "route":
        logits = router_logits(case["tokens"], case["experts"], torch.bfloat16 if case["half"] else torch.float32)
        if case["masked"]:
            closed = torch.rand(case["tokens"], case["experts"], device="cuda", generator=g) < 0.2
            closed |= torch.rand(case["tokens"], 1, device="cuda", generator=g) < 0.02       # padding: no expert at all
            logits = logits.masked_fill(closed, float("-inf"))
        s["logits"] = logits.requires_grad_()
        s["capacity"] = _capacity(case)
        s["dweights"] = normal(case["tokens"], case["k"], dtype=torch.float32)
        s["daux"] = torch.tensor(0.01, device="cuda")
    elif kind == "grouped":
        rows, experts, empty = case["rows"], case["experts"], case["empty"]
        share = torch.rand(experts, device="cuda", generator=g) + 0.25
        share[torch.randperm(experts, device="cuda", generator=g)[:empty]] = 0.0
        edge = (share.cumsum(0) / share.sum() * rows).round().to(torch.int32)
        edge[-1] = rows
        s["offsets"] = torch.cat([edge.new_zeros(1), edge])
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())       # rows of the largest group, known where they were grouped
        s["x"] = normal(rows, case["inner"]).requires_grad_(case["train"])
        s["w"] = normal(experts, case["outer"], case["inner"], std=0.02).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = normal(rows, case["outer"])
    elif kind == "experts":
        tokens, experts, width, units = (case[n] for n in ("tokens", "experts", "width", "units"))
        train = case["train"]
        s["x"] = normal(tokens, width).requires_grad_(train)
        s["logits"] = router_logits(tokens, experts, torch.bfloat16).requires_grad_(train)
        s["w_gate_up"] = normal(experts, 2 * units, width, std=width ** -0.5).requires_grad_(train)
        s["w_down"] = normal(experts, width, units, std=units ** -0.5).requires_grad_(train)
        s["capacity"] = _capacity(case)
        if train:
            s["dout"] = normal(tokens, width)
            s["daux"] = torch.tensor(0.01, device="cuda")
    elif kind == "swiglu8":
        s["gu"] = normal(case["rows"], 2 * case["units"]).requires_grad_()
        s["dact"] = normal(case["rows"], case["units"])
    else:
        s["x"] = normal(case["rows"], case["cols"])
    return s


# ---- with this package ---------------------------------------------------------------------------
def _run_own(s):
    from torchure_b200.ops import act8, moe

    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        r = moe.route(s["logits"], case["k"], s["capacity"])
        dlogits, = torch.autograd.grad((r.weights, r.aux_loss), (s["logits"],), (s["dweights"], s["daux"]))
        return {"weights": r.weights.detach(), "experts": r.experts, "slots": r.slots, "offsets": r.offsets, "rows": r.rows,
                "aux": r.aux_loss.detach(), "dlogits": dlogits}
    if kind == "grouped":
        y = moe.grouped_linear(s["x"], s["w"], s["offsets"])
        if not case["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if kind == "experts":
        out, aux = moe.expert_mlp(s["x"], s["logits"], s["w_gate_up"], s["w_down"], case["k"], s["capacity"])
        if not case["train"]:
            return {"out": out, "aux": aux}
        wrt = (s["x"], s["logits"], s["w_gate_up"], s["w_down"])
        dx, dlogits, dgu, dd = torch.autograd.grad((out, aux), wrt, (s["dout"], s["daux"]))
        return {"out": out.detach(), "aux": aux.detach(), "dx": dx, "dlogits": dlogits, "dw_gate_up": dgu, "dw_down": dd}
    if kind == "swiglu8":
        act = act8.swiglu_8bit(s["gu"])
        dgu, = torch.autograd.grad(act, (s["gu"],), s["dact"])
        return {"act": act.detach(), "dgu": dgu}
    return {"x": act8.dequantize8(act8.quantize8(s["x"]))}


# ---- plain, 32 bits -------------------------------------------------------------------------------
def _plain_route(logits, k, capacity):
    tokens, experts = logits.shape
    top, chosen = (t[:, :k] for t in torch.sort(logits, dim=-1, descending=True, stable=True))
    made = top > float("-inf")
    e = torch.where(made, torch.exp(top - top[:, :1].clamp_min(-3e38)), torch.zeros_like(top))
    weights = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    of = torch.where(made, chosen, experts).reshape(-1)                     # the expert of each choice, `experts`: none
    counts = torch.zeros(experts + 1, device=logits.device, dtype=torch.int64).scatter_add_(0, of, torch.ones_like(of))
    order = torch.sort(of, stable=True).indices
    start = counts.cumsum(0) - counts
    place = torch.empty_like(of).scatter_(0, order, torch.arange(of.numel(), device=of.device)) - start[of]
    kept = counts[:experts].clamp_max(capacity if capacity else of.numel())
    offsets = torch.cat([kept.new_zeros(1), kept.cumsum(0)])
    live = (of < experts) & (place < torch.cat([kept, kept.new_zeros(1)])[of])
    slots = torch.where(live, offsets[of.clamp_max(experts - 1)] + place, -1)
    rows = torch.full((of.numel() + 1,), -1, device=of.device).scatter_(
        0, torch.where(live, slots, of.numel()), torch.where(live, torch.arange(of.numel(), device=of.device), -1))[:-1]
    p = torch.exp(logits - logits.max(-1, keepdim=True).values.clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    share = counts[:experts].float() / (tokens * k)
    aux = experts * (share * p.mean(0)).sum()
    return {"weights": weights, "chosen": chosen, "slots": slots.view(tokens, k), "offsets": offsets, "rows": rows, "p": p, "share": share,
            "aux": aux, "made": made}


def _plain_route_grad(r, dweights, daux):
    w, p, share = r["weights"], r["p"], r["share"]
    at = torch.where(r["made"], w * (dweights - (w * dweights).sum(-1, keepdim=True)), torch.zeros_like(w))
    dl = daux * (p.shape[1] / p.shape[0]) * p * (share - (p * share).sum(-1, keepdim=True))
    return dl.scatter_add(1, r["chosen"], at)


def _padded(x, offsets, most):
    """Rows by group, [groups, most, columns], zeros behind; and where each row went."""
    n = torch.arange(x.shape[0], device=x.device)
    group = torch.searchsorted(offsets[1:].contiguous(), n.to(offsets.dtype), right=True)
    at = group * most + n - offsets[group.clamp_max(offsets.numel() - 1)]
    return x.new_zeros((offsets.numel() - 1) * most, x.shape[1]).index_copy(0, at, x).view(-1, most, x.shape[1]), at


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        logits = s["logits"].detach()
        r = _plain_route(logits.float(), case["k"], s["capacity"])
        dlogits = _plain_route_grad(r, s["dweights"], s["daux"])
        return {"weights": r["weights"], "experts": r["chosen"].int(), "slots": r["slots"].int(), "offsets": r["offsets"].int(),
                "rows": r["rows"].int(), "aux": r["aux"], "dlogits": dlogits.to(logits.dtype)}
    if kind == "grouped":
        x, w = s["x"].detach(), s["w"].detach()
        xp, at = _padded(x.float(), s["offsets"].long(), s["most"])
        wf = w.float()
        y = torch.bmm(xp, wf.transpose(1, 2)).flatten(0, 1)[at].to(x.dtype)
        if not case["train"]:
            return {"y": y}
        dyp, _ = _padded(s["dy"].float(), s["offsets"].long(), s["most"])
        return {"y": y, "dx": torch.bmm(dyp, wf).flatten(0, 1)[at].to(x.dtype), "dw": torch.bmm(dyp.transpose(1, 2), xp).to(w.dtype)}
    if kind == "experts":
        x, logits = s["x"].detach(), s["logits"].detach()
        wgu, wd = s["w_gate_up"].detach().float(), s["w_down"].detach().float()
        tokens, width = x.shape
        k, experts = case["k"], case["experts"]
        most = s["capacity"] or tokens
        r = _plain_route(logits.float(), k, s["capacity"])
        # rows in buffers of `most` for each expert, one more row for what was dropped
        slots = r["slots"].reshape(-1)
        chosen = r["chosen"].reshape(-1)
        at = torch.where(slots >= 0, chosen * most + slots - r["offsets"][chosen], experts * most)
        token = torch.arange(tokens, device=x.device).repeat_interleave(k)

        def spread(t):
            return t.new_zeros(experts * most + 1, t.shape[1]).index_copy(0, at, t[token])[:-1].view(experts, most, -1)

        def back(t):
            return torch.cat([t.reshape(experts * most, -1), t.new_zeros(1, t.shape[-1])])[at].view(tokens, k, -1)

        xp = spread(x.float())
        gu = torch.bmm(xp, wgu.transpose(1, 2))
        gate, up = gu.chunk(2, dim=-1)
        sig = 1.0 / (1.0 + torch.exp(-gate))
        act = gate * sig * up
        y = back(torch.bmm(act, wd.transpose(1, 2)))
        out = (r["weights"][:, :, None] * y).sum(1).to(x.dtype)
        if not case["train"]:
            return {"out": out, "aux": r["aux"]}
        dout = s["dout"].float()
        dweights = torch.where(r["slots"] >= 0, (y * dout[:, None]).sum(-1), torch.zeros_like(r["weights"]))
        wp = torch.zeros(experts * most + 1, device=x.device).index_copy(0, at, r["weights"].reshape(-1))[:-1].view(experts, most, 1)
        dyp = spread(dout) * wp
        dact = torch.bmm(dyp, wd)
        dg = dact * up * sig * (1.0 + gate * (1.0 - sig))
        du = dact * gate * sig
        dgu = torch.cat([dg, du], dim=-1)
        return {"out": out, "aux": r["aux"], "dx": back(torch.bmm(dgu, wgu)).sum(1).to(x.dtype),
                "dlogits": _plain_route_grad(r, dweights, s["daux"]).to(logits.dtype),
                "dw_gate_up": torch.bmm(dgu.transpose(1, 2), xp).to(x.dtype), "dw_down": torch.bmm(dyp.transpose(1, 2), act).to(x.dtype)}
    if kind == "swiglu8":
        gu = s["gu"].detach()
        gate, up = gu.float().chunk(2, dim=-1)
        act = gate / (1.0 + torch.exp(-gate)) * up
        gate, up = _plain_8bit(gate), _plain_8bit(up)
        sig = 1.0 / (1.0 + torch.exp(-gate))
        dact = s["dact"].float()
        dgu = torch.cat([dact * up * sig * (1.0 + gate * (1.0 - sig)), dact * gate * sig], dim=-1)
        return {"act": act.to(gu.dtype), "dgu": dgu.to(gu.dtype)}
    return {"x": _plain_8bit(s["x"].float()).to(s["x"].dtype)}


def _plain_8bit(x):
    """x as 8 bits stand for it: whole multiples of the block's largest magnitude / 127, halves away from zero."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.floor(b.abs() * 127.0 / top + 0.5), torch.zeros_like(b)) * b.sign()
    return (q * (top / 127.0)).view(rows, -1)[:, :cols]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions, 64 bits ---------------------------------------------------------------------
def _exact_route(logits, k, capacity):
    l = logits.detach().double().cpu()
    T, E = l.shape
    chosen = torch.empty(T, k, dtype=torch.int64)
    left = l.clone()
    barred = torch.zeros(T, E, dtype=torch.bool)
    index = torch.arange(E).expand(T, E)
    for j in range(k):                                    # the lowest index among the largest that are left
        best = left.masked_fill(barred, float("-inf")).amax(1, keepdim=True)
        is_best = (left == best) & ~barred
        chosen[:, j] = torch.where(is_best, index, E).amin(1)
        barred.scatter_(1, chosen[:, j:j + 1], True)
    top = l.gather(1, chosen)
    made = top != float("-inf")
    weights = torch.where(made, torch.nan_to_num(torch.softmax(top, 1)), torch.zeros_like(top))
    p = torch.nan_to_num(torch.softmax(l, 1))
    slots = torch.full((T * k,), -1, dtype=torch.int64)
    rows = torch.full((T * k,), -1, dtype=torch.int64)
    offsets, counts = [0], []
    flat = torch.where(made, chosen, -1).reshape(-1)
    for e in range(E):
        mine = (flat == e).nonzero()[:, 0]
        counts.append(mine.numel())
        mine = mine[:capacity] if capacity else mine
        slots[mine] = offsets[-1] + torch.arange(mine.numel())
        rows[offsets[-1]:offsets[-1] + mine.numel()] = mine
        offsets.append(offsets[-1] + mine.numel())
    share = torch.tensor(counts, dtype=torch.float64) / (T * k)
    aux = E * (share * p.mean(0)).sum()
    return weights, chosen, slots, offsets, rows, p, share, aux


def _exact_route_grad(weights, chosen, p, share, dweights, daux):
    T, E = p.shape
    dl = torch.zeros(T, E, dtype=torch.float64)
    inner = (weights * dweights).sum(1)
    for j in range(chosen.shape[1]):
        dl.scatter_add_(1, chosen[:, j:j + 1], (weights[:, j] * (dweights[:, j] - inner))[:, None])
    return dl + daux * E / T * (p * share - p * (p @ share)[:, None])


def _exact_8bit(x):
    out = torch.empty_like(x)
    for lo in range(0, x.shape[1], BLOCK):
        b = x[:, lo:lo + BLOCK]
        top = b.abs().max(1, keepdim=True).values
        q = torch.sign(b) * torch.floor(b.abs() * 127 / torch.where(top > 0, top, torch.ones_like(top)) + 0.5)
        out[:, lo:lo + BLOCK] = q * top / 127
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        w, chosen, slots, offsets, rows, p, share, aux = _exact_route(s["logits"], case["k"], s["capacity"])
        dl = _exact_route_grad(w, chosen, p, share, s["dweights"].double().cpu(), float(s["daux"]))
        return {"weights": w, "experts": chosen.int(), "slots": slots.view(-1, case["k"]).int(),
                "offsets": torch.tensor(offsets, dtype=torch.int32), "rows": rows.int(), "aux": aux, "dlogits": dl}
    if kind == "grouped":
        edges = s["offsets"].tolist()
        x, w = s["x"].detach().double(), s["w"].detach().double()
        spans = list(zip(edges[:-1], edges[1:]))
        y = torch.cat([x[a:b] @ w[e].t() for e, (a, b) in enumerate(spans)])
        if not case["train"]:
            return {"y": y}
        dy = s["dy"].double()
        return {"y": y, "dx": torch.cat([dy[a:b] @ w[e] for e, (a, b) in enumerate(spans)]),
                "dw": torch.stack([dy[a:b].t() @ x[a:b] for a, b in spans])}
    if kind == "experts":
        k = case["k"]
        w, chosen, _, offsets, rows, p, share, aux = _exact_route(s["logits"], k, s["capacity"])
        x, wgu, wd = (s[n].detach().double() for n in ("x", "w_gate_up", "w_down"))
        F = case["units"]
        dev = x.device
        out = torch.zeros_like(x)
        if case["train"]:
            dout = s["dout"].double()
            dx, dwgu, dwd = torch.zeros_like(x), torch.zeros_like(wgu), torch.zeros_like(wd)
            dweights = torch.zeros(w.numel(), dtype=torch.float64, device=dev)
        wflat = w.reshape(-1).to(dev)
        for e in range(case["experts"]):
            mine = rows[offsets[e]:offsets[e + 1]].to(dev)
            t = mine // k
            g, u = x[t] @ wgu[e, :F].t(), x[t] @ wgu[e, F:].t()
            sg = torch.sigmoid(g)
            a = g * sg * u
            y = a @ wd[e].t()
            out.index_add_(0, t, wflat[mine, None] * y)
            if case["train"]:
                dweights[mine] = (y * dout[t]).sum(1)
                dy = wflat[mine, None] * dout[t]
                da = dy @ wd[e]
                dwd[e] = dy.t() @ a
                dg, du = da * u * (sg + g * sg * (1 - sg)), da * g * sg
                dwgu[e, :F], dwgu[e, F:] = dg.t() @ x[t], du.t() @ x[t]
                dx.index_add_(0, t, dg @ wgu[e, :F] + du @ wgu[e, F:])
        if not case["train"]:
            return {"out": out, "aux": aux}
        dl = _exact_route_grad(w, chosen, p, share, dweights.cpu().view_as(w), float(s["daux"]))
        return {"out": out, "aux": aux, "dx": dx, "dlogits": dl, "dw_gate_up": dwgu, "dw_down": dwd}
    if kind == "swiglu8":
        gu, dact, F = s["gu"].detach().double(), s["dact"].double(), case["units"]
        act = gu[:, :F] * torch.sigmoid(gu[:, :F]) * gu[:, F:]
        g, u = _exact_8bit(gu[:, :F]), _exact_8bit(gu[:, F:])
        sg = torch.sigmoid(g)
        return {"act": act, "dgu": torch.cat([dact * u * (sg + g * sg * (1 - sg)), dact * g * sg], 1)}
    return {"x": _exact_8bit(s["x"].double())}


def work(case):
    kind = case["kind"]
    if kind == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        size = 2 if case["half"] else 4
        # logits in, gradient out; weights, experts, slots and rows of each choice out, the weights' gradient in
        return {"bytes": 2 * T * E * size + T * k * 20 + 4 * (E + 1), "flops": 12 * T * E}
    if kind == "grouped":
        R, E, K, N = case["rows"], case["experts"], case["inner"], case["outer"]
        used = min(R, E - case["empty"])
        if not case["train"]:
            return {"bytes": 2 * (R * (K + N) + used * N * K), "flops": 2 * R * N * K}
        return {"bytes": 2 * (2 * R * (K + N) + used * N * K + E * N * K), "flops": 6 * R * N * K}
    if kind == "experts":
        T, E, k, D, F = (case[n] for n in ("tokens", "experts", "k", "width", "units"))
        used = min(E, T * k)
        once = 2 * (2 * T * D + T * E + used * 3 * D * F)
        if not case["train"]:
            return {"bytes": once, "flops": 6 * T * k * D * F}
        return {"bytes": once + 2 * (2 * T * D + T * E + E * 3 * D * F), "flops": 18 * T * k * D * F}
    if kind == "swiglu8":
        return {"bytes": case["rows"] * case["units"] * 2 * (2 + 1 + 1 + 2), "flops": 30 * case["rows"] * case["units"]}
    return {"bytes": 4 * case["rows"] * case["cols"], "flops": 6 * case["rows"] * case["cols"]}
