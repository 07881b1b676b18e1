"""The operators at both ends and in the routers of a mixture-of-experts training step, as measured cases.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``exact`` the same from the definitions in 64 bits and ``work`` what a pass cannot do without.  With
``own`` false ``run`` is made of plain tensor operations in 32 bits, with ``own`` true of this package's entry points.

Kinds:

``scored``     routing by sigmoid or softmax scores with a bias for balance and groups of experts: choices, weights, row order,
               load-balancing term; with ``train`` the gradient of both and the bias of the next step.
``adamw8``     an AdamW step over many tensors whose two moments are held in 8 bits, and the moments that it leaves, read back
               in bf16.
``embedding``  token rows looked up and scaled; with ``train`` the gradient of the table.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 128                                      # values of a moment that share a scale
KEY = {"m": 896, "v": 768}                       # code + KEY, shifted by 20 bits, is the value's pattern, FIRST[..] too large
FIRST = {"m": 2.0 ** -15, "v": 2.0 ** -31}
LAST = {"m": 127, "v": 255}
TOP = {"m": 1.875 - 2.0 ** -15, "v": 1.875}      # what the largest magnitude of a block is brought to
LOW = 0xFFFFFFFF


def listed():
    return [
        # one token of a served mixture of many experts in groups
        {"name": "scored_token", "kind": "scored", "tokens": 1, "experts": 64, "k": 6, "score": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "normalize": True, "scale": 2.5, "factor": 0.0, "half": False, "masked": False, "train": False},
        # a micro-batch's router: 256 experts in 8 groups, fp32 logits
        {"name": "scored_groups", "kind": "scored", "tokens": 8192, "experts": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "normalize": True, "scale": 2.5, "factor": 0.0, "half": False, "masked": False, "train": True},
        # groups of 20, probabilities as weights, experts closed to some tokens, a capacity, an odd token count
        {"name": "scored_odd", "kind": "scored", "tokens": 4099, "experts": 160, "k": 6, "score": "softmax", "bias": False, "groups": 8,
         "top_groups": 3, "normalize": False, "scale": 16.0, "factor": 1.25, "half": True, "masked": True, "train": True},
        # a long batch, no groups, mixed precision logits
        {"name": "scored_long", "kind": "scored", "tokens": 32768, "experts": 128, "k": 8, "score": "sigmoid", "bias": True, "groups": 1,
         "top_groups": 0, "normalize": True, "scale": 1.0, "factor": 0.0, "half": True, "masked": False, "train": True},
        # a tiny model's parameters: a few calls' latency
        {"name": "adamw8_tiny", "kind": "adamw8", "vocab": 1024, "emb": 256, "ffn": 512, "experts": 1, "blocks": 2, "half": False,
         "shadow": True, "clip": True, "step": 3},
        # odd widths, gradients in bf16, no shadow weights
        {"name": "adamw8_odd", "kind": "adamw8", "vocab": 32001, "emb": 519, "ffn": 1003, "experts": 3, "blocks": 2, "half": True,
         "shadow": False, "clip": False, "step": 1000},
        # the shipped mixture's table and a part of its blocks, gradients in fp32
        {"name": "adamw8_mixture", "kind": "adamw8", "vocab": 151936, "emb": 1024, "ffn": 1536, "experts": 8, "blocks": 3, "half": False,
         "shadow": True, "clip": True, "step": 100},
        # one token while a model answers
        {"name": "embedding_token", "kind": "embedding", "tokens": 1, "vocab": 151936, "width": 1024, "scale": 1.0, "padding": 0.0,
         "table_half": True, "out_half": True, "train": False},
        # a short sequence through a small table
        {"name": "embedding_short", "kind": "embedding", "tokens": 509, "vocab": 8192, "width": 512, "scale": 1.0, "padding": 0.0,
         "table_half": False, "out_half": False, "train": True},
        # the shipped mixture's micro-batch
        {"name": "embedding_batch", "kind": "embedding", "tokens": 8192, "vocab": 151936, "width": 1024, "scale": 1.0, "padding": 0.0,
         "table_half": False, "out_half": False, "train": True},
        # padded rows of an odd width, table and activations in bf16, rows scaled by the root of the width
        {"name": "embedding_padded", "kind": "embedding", "tokens": 65521, "vocab": 50257, "width": 1003, "scale": 31.67, "padding": 0.3,
         "table_half": True, "out_half": True, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["scored", "adamw8", "embedding"])
    if kind == "scored":
        groups = rng.choice([1, 1, 2, 4, 8])
        each = _log(rng, 2, 256 // groups)
        top_groups = rng.randint(1, groups) if groups > 1 else 0
        experts = groups * each
        return {"kind": kind, "tokens": _log(rng, 1, max(1, min(32768, 2097152 // experts))), "experts": experts,
                "k": rng.randint(1, min(8, max(1, top_groups) * each)), "score": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.7, "groups": groups, "top_groups": top_groups, "normalize": rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5]), "factor": rng.choice([0.0, 0.0, 1.25]), "half": rng.random() < 0.5,
                "masked": rng.random() < 0.3, "train": rng.random() < 0.7}
    if kind == "adamw8":
        return {"kind": kind, "vocab": _log(rng, 100, 65536), "emb": _log(rng, 64, 1024), "ffn": _log(rng, 64, 1536),
                "experts": rng.choice([1, 1, 2, 4]), "blocks": rng.randint(1, 3), "half": rng.random() < 0.3,
                "shadow": rng.random() < 0.6, "clip": rng.random() < 0.6, "step": _log(rng, 1, 100000)}
    tokens, vocab = _log(rng, 1, 65536), _log(rng, 1000, 151936)
    return {"kind": kind, "tokens": tokens, "vocab": vocab, "width": min(_log(rng, 64, 2560), 155582464 // vocab, 65716563 // tokens),
            "scale": rng.choice([1.0, 1.0, 22.6]), "padding": rng.choice([0.0, 0.0, 0.2, 0.6]), "table_half": rng.random() < 0.4,
            "out_half": rng.random() < 0.5, "train": rng.random() < 0.75}


def _capacity(case):
    """Rows that an expert takes at most; 0: as many as there are."""
    if not case["factor"]:
        return 0
    return max(1, int(case["factor"] * case["tokens"] * case["k"] / case["experts"] + 0.999))


def _shapes(case):
    D, F, E = case["emb"], case["ffn"], case["experts"]
    block = [(D,), (2 * D, D), (E, D), (E, 2 * F, D), (E, D, F)]
    return [(case["vocab"], D)] + block * case["blocks"] + [(D,)]


HYPER = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "scored":
        tokens, experts = case["tokens"], case["experts"]
        # a learned router prefers some experts; the bias that balances them takes some of that back
        liking = normal(experts, std=0.5)
        logits = (normal(tokens, experts) + liking).to(torch.bfloat16 if case["half"] else torch.float32)
        if case["masked"]:
            closed = torch.rand(tokens, experts, device="cuda", generator=g) < 0.2
            closed |= torch.rand(tokens, 1, device="cuda", generator=g) < 0.02       # padding: no expert at all
            logits = logits.masked_fill(closed, float("-inf"))
        s["logits"] = logits.requires_grad_(case["train"])
        s["bias"] = (normal(experts, std=0.02) - 0.1 * liking * (1.0 if case["score"] == "sigmoid" else 0.01)) if case["bias"] else None
        s["capacity"] = _capacity(case)
        if case["train"]:
            s["dweights"] = normal(tokens, case["k"])
            s["daux"] = torch.tensor(0.01, device="cuda")
    elif kind == "adamw8":
        s["params"], s["grads"], s["shadows"] = [], [], []
        kept = {"m": [], "v": []}
        for i, shape in enumerate(_shapes(case)):
            p = normal(*shape, std=0.02) if len(shape) > 1 else torch.ones(shape, device="cuda")
            # rows (tokens, units) differ in how strong their gradients are
            strength = torch.exp(normal(*shape[:-1], 1)) * 1e-3
            grad = normal(*shape) * strength
            m, v = normal(*shape) * strength * 0.3, (normal(*shape).abs() * 0.3 + 0.1) * strength * strength
            s["params"].append(p)
            s["grads"].append(grad.to(torch.bfloat16) if case["half"] and len(shape) > 1 else grad)
            s["shadows"].append(p.to(torch.bfloat16) if case["shadow"] and len(shape) > 1 else None)
            kept["m"].append(_pack(m, "m", seed * 1000 + i))
            kept["v"].append(_pack(v, "v", seed * 1000 + i))
        for n in "mv":
            s[n + "_codes"], s[n + "_scales"] = ([k[j] for k in kept[n]] for j in (0, 1))
        s["clip"] = torch.tensor(0.73, device="cuda") if case["clip"] else None
        s["seed"] = seed & 0xFFFF
    else:
        tokens, vocab, width = case["tokens"], case["vocab"], case["width"]
        # the n-th most frequent token has a share of about 1 / n
        ids = (float(vocab) ** torch.rand(tokens, device="cuda", generator=g, dtype=torch.float64)).long() - 1
        s["pad"] = vocab - 1 if case["padding"] else None
        ids = ids.clamp_(0, vocab - 1)
        if case["padding"]:
            row = max(1, min(1024, tokens // 4))            # the last part of every sequence
            ids[torch.arange(tokens, device="cuda") % row >= row * (1 - case["padding"])] = vocab - 1
        s["ids"] = ids
        s["table"] = normal(vocab, width, std=0.02, dtype=torch.bfloat16 if case["table_half"] else torch.float32).requires_grad_(case["train"])
        s["out_type"] = torch.bfloat16 if case["out_half"] else torch.float32
        if case["train"]:
            s["dout"] = normal(tokens, width, std=1e-3, dtype=s["out_type"])
    return s


# ---- with this package ---------------------------------------------------------------------------
def _run_own(s):
    from torchure_b200.ops import moe, multi_tensor
    from torchure_b200.ops.embedding import embedding

    case = s["case"]
    kind = case["kind"]
    if kind == "scored":
        r = moe.route(s["logits"], case["k"], s["capacity"], score=case["score"], bias=s["bias"], groups=case["groups"],
                      top_groups=case["top_groups"], normalize=case["normalize"], scale=case["scale"])
        out = {"weights": r.weights.detach(), "experts": r.experts, "slots": r.slots, "offsets": r.offsets, "rows": r.rows,
               "aux": r.aux_loss.detach()}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad((r.weights, r.aux_loss), (s["logits"],), (s["dweights"], s["daux"]))
            if s["bias"] is not None:
                out["bias"] = moe.balance_bias_(s["bias"].clone(), r.counts, 1e-3)
        return out
    if kind == "adamw8":
        multi_tensor.adamw8_step(s["params"], s["grads"], s["m_codes"], s["m_scales"], s["v_codes"], s["v_scales"], s["shadows"],
                                 step=case["step"], grad_scale=s["clip"], seed=s["seed"], **HYPER)
        return {"params": s["params"], "shadows": [t for t in s["shadows"] if t is not None],
                "m": multi_tensor.state8_values(s["m_codes"], s["m_scales"], signed=True, dtype=torch.bfloat16),
                "v": multi_tensor.state8_values(s["v_codes"], s["v_scales"], signed=False, dtype=torch.bfloat16)}
    out = embedding(s["ids"], s["table"], case["scale"], s["pad"], s["out_type"])
    if not case["train"]:
        return {"out": out}
    dtable, = torch.autograd.grad(out, (s["table"],), s["dout"])
    return {"out": out.detach(), "dtable": dtable}


# ---- plain: routing ---------------------------------------------------------------------------------
def _plain_scored(logits, bias, case, capacity):
    tokens, experts = logits.shape
    k, groups = case["k"], case["groups"]
    l = logits.double()                                    # the choice goes by scores rounded to fp32 once: neighbours may be that close
    lowest = torch.tensor(float("-inf"), device=l.device)
    is_open = l > lowest
    if case["score"] == "sigmoid":
        s = (1.0 / (1.0 + torch.exp(-l))).float()
        p = s / s.sum(-1, keepdim=True).clamp_min(1e-30)
    else:
        e = torch.exp(l - l.amax(-1, keepdim=True).clamp_min(-3e38))
        s = p = (e / e.sum(-1, keepdim=True).clamp_min(1e-30)).float()
    key = logits.float() if bias is None and groups == 1 else s if bias is None else s + bias
    key = torch.where(is_open, key, lowest)
    if groups > 1:
        best = torch.sort(key.view(tokens, groups, -1), dim=-1, descending=True).values[..., :2]
        of_group = torch.where(best[..., 0] > lowest, torch.where(best > lowest, best, 0.0).sum(-1), lowest)
        order = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        stays = torch.zeros(tokens, groups, dtype=torch.bool, device=l.device).scatter_(1, order, True)
        key = torch.where(stays.repeat_interleave(experts // groups, dim=1), key, lowest)
    top, chosen = (t[:, :k] for t in torch.sort(key, dim=-1, descending=True, stable=True))
    made = top > lowest
    got = torch.where(made, s.gather(1, chosen), 0.0)
    whole = got.sum(-1, keepdim=True).clamp_min(1e-30) if case["normalize"] else torch.ones_like(got[:, :1])
    weights = case["scale"] * (got / whole)
    of = torch.where(made, chosen, experts).reshape(-1)                     # the expert of each choice, `experts`: none
    counts = torch.zeros(experts + 1, device=l.device, dtype=torch.int64).scatter_add_(0, of, torch.ones_like(of))
    order = torch.sort(of, stable=True).indices
    start = counts.cumsum(0) - counts
    place = torch.empty_like(of).scatter_(0, order, torch.arange(of.numel(), device=of.device)) - start[of]
    kept = counts[:experts].clamp_max(capacity if capacity else of.numel())
    offsets = torch.cat([kept.new_zeros(1), kept.cumsum(0)])
    live = (of < experts) & (place < torch.cat([kept, kept.new_zeros(1)])[of])
    slots = torch.where(live, offsets[of.clamp_max(experts - 1)] + place, -1)
    rows = torch.full((of.numel() + 1,), -1, device=of.device).scatter_(
        0, torch.where(live, slots, of.numel()), torch.where(live, torch.arange(of.numel(), device=of.device), -1))[:-1]
    share = counts[:experts].float() / (tokens * k)
    aux = experts * (share * p.mean(0)).sum()
    return {"weights": weights, "chosen": chosen, "slots": slots.view(tokens, k), "offsets": offsets, "rows": rows, "p": p, "s": s,
            "share": share, "aux": aux, "counts": counts[:experts], "whole": whole}


def _plain_scored_grad(r, case, dweights, daux):
    p, share, w = r["p"], r["share"], r["weights"] / case["scale"]
    sigmoid = case["score"] == "sigmoid"
    dw = case["scale"] * dweights
    steep = 1.0 - r["s"] if sigmoid else torch.ones_like(p)                 # what is left of a score's own slope, over the score
    dl = daux * (p.shape[1] / p.shape[0]) * p * (share - (p * share).sum(-1, keepdim=True)) * steep
    inner = (w * dw).sum(-1, keepdim=True)
    if case["normalize"]:
        at = w * (dw - inner) * steep.gather(1, r["chosen"])
    else:
        at = w * dw * steep.gather(1, r["chosen"])
        if not sigmoid:
            dl = dl - p * inner
    return dl.scatter_add(1, r["chosen"], at)


# ---- plain: moments in 8 bits -----------------------------------------------------------------------
# A block of 128 values shares the scale (its largest magnitude) / TOP.  A magnitude y, brought to TOP by the block's largest, is held as
# the pattern of y + FIRST in 3 bits of mantissa, counted from FIRST's: even steps next to zero, steps of an eighth further up.  Which of
# its two neighbours a value goes to is decided by 16 random bits, so that the mean over many steps is the value's own; a second moment
# that is not zero keeps at least the first step.
def _mix(x):
    x = (x ^ (x >> 16)) * 0x7FEB352D & LOW
    x = (x ^ (x >> 15)) * 0x846CA68B & LOW
    return x ^ (x >> 16)


def _mix_int(x):
    x = (x ^ (x >> 16)) * 0x7FEB352D & LOW
    x = (x ^ (x >> 15)) * 0x846CA68B & LOW
    return x ^ (x >> 16)


def _random_bits(n, seed, step, index, device):
    """32 bits for each of a tensor's n values (the `index`-th tensor's): 16 for each moment."""
    key = _mix_int((seed + 0x9E3779B9 * step) & LOW)
    key = _mix_int((key + 0x85EBCA6B * index) & LOW)
    return _mix(torch.arange(n, device=device) ^ key)


def _blocks(x):
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _encode(x, which, bits):
    """(codes, scales) of x (fp32) with 16 random bits for each value."""
    shape, n = x.shape, x.numel()
    b = _blocks(x)
    top = b.abs().amax(-1, keepdim=True)
    inverse = TOP[which] / top
    y = b.abs() * inverse + FIRST[which]
    code = ((y.view(torch.int32) + (_blocks(bits) << 4).int()) >> 20) - KEY[which]
    code = code.clamp_max(LAST[which])
    if which == "v":
        code = torch.where(b > 0, code.clamp_min(1), code)
    else:
        code = torch.where(b < 0, code + 128, code)
    fine = (top >= 2.0 ** -100) & (top < float("inf"))
    code = torch.where(fine, code, 0)
    scale = torch.where(fine, top / TOP[which], torch.where(top < 2.0 ** -100, 0.0, float("nan")))
    return code.view(-1)[:n].view(shape).to(torch.uint8), scale.view(-1)


def _decode(codes, scales, which):
    n = codes.numel()
    c = _blocks(codes).int()
    size = c & 127 if which == "m" else c
    y = (((size + KEY[which]) << 20).view(torch.float32) - FIRST[which]) * scales[:, None]
    if which == "m":
        y = torch.where(c >= 128, -y, y)
    return y.view(-1)[:n].view(codes.shape)


def _pack(x, which, seed):
    g = torch.Generator(device=x.device).manual_seed(seed)
    return _encode(x, which, torch.randint(0, 65536, (x.numel(),), device=x.device, generator=g))


def _plain_adamw8(s, i):
    case = s["case"]
    b1, b2, lr = HYPER["beta1"], HYPER["beta2"], HYPER["lr"]
    step_size = lr / (1.0 - b1 ** case["step"])
    root = (1.0 - b2 ** case["step"]) ** -0.5
    p, g = s["params"][i], s["grads"][i].float()
    if s["clip"] is not None:
        g = g * s["clip"]
    m = _decode(s["m_codes"][i], s["m_scales"][i], "m") * b1 + g * (1.0 - b1)
    v = _decode(s["v_codes"][i], s["v_scales"][i], "v") * b2 + (g * (1.0 - b2)) * g
    p.copy_(p * (1.0 - lr * HYPER["weight_decay"]) - (m / (torch.sqrt(v) * root + HYPER["eps"])) * step_size)
    if s["shadows"][i] is not None:
        s["shadows"][i].copy_(p)
    bits = _random_bits(p.numel(), s["seed"], case["step"], i, p.device)
    for which, x, r in (("m", m, bits & 0xFFFF), ("v", v, bits >> 16)):
        codes, scales = _encode(x, which, r)
        s[which + "_codes"][i].copy_(codes)
        s[which + "_scales"][i].copy_(scales)
    m, v = (_decode(s[n + "_codes"][i], s[n + "_scales"][i], n).to(torch.bfloat16) for n in "mv")
    return p, s["shadows"][i], m, v


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "scored":
        logits = s["logits"].detach()
        r = _plain_scored(logits, s["bias"], case, s["capacity"])
        out = {"weights": r["weights"], "experts": r["chosen"].int(), "slots": r["slots"].int(), "offsets": r["offsets"].int(),
               "rows": r["rows"].int(), "aux": r["aux"]}
        if case["train"]:
            out["dlogits"] = _plain_scored_grad(r, case, s["dweights"], s["daux"]).to(logits.dtype)
            if s["bias"] is not None:
                n = r["counts"]
                out["bias"] = s["bias"] + 1e-3 * torch.sign(n.sum() - n * n.numel()).float()
        return out
    if kind == "adamw8":
        p, shadows, m, v = zip(*[_plain_adamw8(s, i) for i in range(len(s["params"]))])
        return {"params": list(p), "shadows": [t for t in shadows if t is not None], "m": list(m), "v": list(v)}
    table = s["table"].detach()
    out = (table[s["ids"]].float() * case["scale"]).to(s["out_type"])
    if not case["train"]:
        return {"out": out}
    dtable = torch.zeros(table.shape, device=table.device).index_add_(0, s["ids"], s["dout"].float()) * case["scale"]
    if s["pad"] is not None:
        dtable[s["pad"]] = 0.0
    return {"out": out, "dtable": dtable.to(table.dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions, 64 bits ---------------------------------------------------------------------
def _largest(key, count):
    """Indices of the `count` largest of each row, the lowest index among equals."""
    left, found = key.clone(), []
    barred = torch.zeros_like(key, dtype=torch.bool)
    index = torch.arange(key.shape[1], device=key.device).expand_as(key)
    for _ in range(count):
        best = left.masked_fill(barred, float("-inf")).amax(1, keepdim=True)
        at = torch.where((left == best) & ~barred, index, key.shape[1]).amin(1, keepdim=True)
        barred = barred.scatter(1, at, True)
        found.append(at)
    return torch.cat(found, 1)


def _exact_scored(s):
    case = s["case"]
    T, E, k, G = (case[n] for n in ("tokens", "experts", "k", "groups"))
    l = s["logits"].detach().double().requires_grad_()
    none = torch.isinf(l.detach()).all(1, keepdim=True)
    is_open = ~torch.isinf(l.detach())
    safe = torch.where(is_open, l, torch.zeros_like(l))
    if case["score"] == "sigmoid":
        score = torch.sigmoid(safe) * is_open
        share_of = score / torch.where(none, torch.ones_like(l[:, :1]), score.sum(1, keepdim=True))
    else:
        score = share_of = torch.nan_to_num(torch.softmax(torch.where(none, torch.zeros_like(l), l), 1)) * is_open
    key = score.detach().float() if s["bias"] is not None or G > 1 else s["logits"].detach().float()
    if s["bias"] is not None:
        key = key + s["bias"]
    key = key.masked_fill(~is_open, float("-inf"))
    if G > 1:
        n = E // G
        of_group = torch.full((T, G), float("-inf"), device=l.device)
        for g in range(G):
            mine = key[:, g * n:(g + 1) * n]
            two = mine.gather(1, _largest(mine, min(2, n)))
            of_group[:, g] = torch.where(torch.isinf(two), 0.0, two).sum(1).masked_fill(torch.isinf(two).all(1), float("-inf"))
        stays = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter(1, _largest(of_group, case["top_groups"]), True)
        for g in range(G):
            key[:, g * n:(g + 1) * n].masked_fill_(~stays[:, g:g + 1], float("-inf"))
    chosen = _largest(key, k)
    made = ~torch.isinf(key.gather(1, chosen))
    got = score.gather(1, chosen) * made
    if case["normalize"]:
        got = got / torch.where(made.any(1, keepdim=True), got.sum(1, keepdim=True), torch.ones_like(got[:, :1]))
    weights = case["scale"] * got
    flat = torch.where(made, chosen, -1).reshape(-1).cpu()
    slots = torch.full((T * k,), -1, dtype=torch.int32)
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    offsets, counts = [0], []
    for e in range(E):
        mine = (flat == e).nonzero()[:, 0]
        counts.append(mine.numel())
        mine = mine[:s["capacity"]] if s["capacity"] else mine
        slots[mine] = offsets[-1] + torch.arange(mine.numel(), dtype=torch.int32)
        rows[offsets[-1]:offsets[-1] + mine.numel()] = mine.int()
        offsets.append(offsets[-1] + mine.numel())
    aux = E * (torch.tensor(counts, dtype=torch.float64, device=l.device) / (T * k) * share_of.mean(0)).sum()
    out = {"weights": weights.detach(), "experts": chosen.int(), "slots": slots.view(T, k), "offsets": torch.tensor(offsets, dtype=torch.int32),
           "rows": rows, "aux": aux.detach()}
    if case["train"]:
        ((weights * s["dweights"].double()).sum() + float(s["daux"]) * aux).backward()
        out["dlogits"] = l.grad
        if s["bias"] is not None:
            mean = sum(counts) / E
            out["bias"] = s["bias"].double() + torch.tensor([1e-3 * ((c < mean) - (c > mean)) for c in counts], dtype=torch.float64, device=l.device)
    return out


def _exact_values(codes, scales, which):
    c = codes.reshape(-1).long()
    size = c % 128 if which == "m" else c
    y = torch.ldexp(1.0 + (size % 8).double() / 8, (size // 8).double() - (15 if which == "m" else 31)) - FIRST[which]
    y = y * scales.double().repeat_interleave(BLOCK)[:c.numel()]
    return (torch.where(c >= 128, -y, y) if which == "m" else y).view(codes.shape)


def _exact_kept(x, which, bits):
    """What 8 bits stand for, of x in 64 bits."""
    n, low = x.numel(), -15 if which == "m" else -31
    b = torch.cat([x.reshape(-1), x.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    r = torch.cat([bits, bits.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    some = top >= 2.0 ** -100
    scale = torch.where(some, top, torch.ones_like(top)) / TOP[which]
    y = b.abs() / scale + FIRST[which]
    power = torch.floor(torch.log2(y)).clamp(low, 0)
    unit = torch.ldexp(torch.ones_like(y), power - 3)
    up = torch.floor(y / unit + r.double() / 65536)                       # goes up as often as the rest of the step is large
    kept = torch.minimum(up * unit, torch.full_like(y, 1.875)) - FIRST[which]
    if which == "v":
        kept = torch.where((b > 0) & (kept <= 0), FIRST[which] / 8, kept)
    return (torch.where(some, kept * scale, torch.zeros_like(kept)) * torch.where(b < 0, -1.0, 1.0)).view(-1)[:n].view(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "scored":
        return _exact_scored(s)
    if kind == "adamw8":
        t, b1, b2 = case["step"], HYPER["beta1"], HYPER["beta2"]
        out = {"params": [], "shadows": [], "m": [], "v": []}
        for i, p in enumerate(s["params"]):
            g = s["grads"][i].double() * (1.0 if s["clip"] is None else s["clip"].double())
            m = b1 * _exact_values(s["m_codes"][i], s["m_scales"][i], "m") + (1 - b1) * g
            v = b2 * _exact_values(s["v_codes"][i], s["v_scales"][i], "v") + (1 - b2) * g * g
            new = p.double() * (1 - HYPER["lr"] * HYPER["weight_decay"])
            new -= HYPER["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
            out["params"].append(new)
            if s["shadows"][i] is not None:
                out["shadows"].append(new)
            bits = _random_bits(p.numel(), s["seed"], t, i, p.device)
            out["m"].append(_exact_kept(m, "m", bits & 0xFFFF))
            out["v"].append(_exact_kept(v, "v", bits >> 16))
        return out
    table, ids = s["table"].detach().double(), s["ids"]
    out = {"out": table[ids] * case["scale"]}
    if case["train"]:
        keep = torch.ones_like(ids, dtype=torch.bool) if s["pad"] is None else ids != s["pad"]
        out["dtable"] = torch.zeros_like(table).index_add_(0, ids[keep], s["dout"].double()[keep] * case["scale"])
    return out


def work(case):
    kind = case["kind"]
    if kind == "scored":
        T, E, k = case["tokens"], case["experts"], case["k"]
        size = 2 if case["half"] else 4
        # logits in; weights, experts, slots and rows of each choice out; with the gradient that one out and the weights' in
        once = T * E * size + T * k * 16 + 4 * (E + 1) + (4 * E if case["bias"] else 0)
        return {"bytes": once + (T * E * size + T * k * 4 if case["train"] else 0), "flops": (12 if case["train"] else 6) * T * E}
    if kind == "adamw8":
        n = sum(math.prod(shape) for shape in _shapes(case))
        wide = sum(math.prod(shape) for shape in _shapes(case) if len(shape) > 1)
        grads = 4 * n - (2 * wide if case["half"] else 0)
        # parameters in and out, gradients in, codes and scales in and out, shadows out, both moments read back in bf16
        return {"bytes": 8 * n + grads + 4 * n + n // 8 + (2 * wide if case["shadow"] else 0) + 4 * n, "flops": 60 * n}
    T, V, D = case["tokens"], case["vocab"], case["width"]
    row, out = (2 if case["table_half"] else 4) * D, (2 if case["out_half"] else 4) * D
    once = 8 * T + min(T, V) * row + T * out
    return {"bytes": once + (T * out + V * row if case["train"] else 0), "flops": (2 if case["train"] else 1) * T * D}
