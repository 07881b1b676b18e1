"""Routing by scores: sigmoid or softmax, a bias for the choice, groups of experts, weights as they are or over their sum; the bias' update.

Choices have to be equal.  Weights and gradients come from fp32 arithmetic: exponentials within 2 units of 2^-23 of arguments that are off by
2^-24 |l| (|l| < 16: 2^-20), sums of at most 16 and 384 terms, two products: FP32 = 2^-18 relative in the 2-norm.  A result in bf16 is off by
at most half a step more, 2^-8 of each value and so of the norm (BF16); over many values about RMS."""

import math

import pytest
import torch

from torchure_b200 import ops
from torchure_b200.ops import debug, kernels, moe, oracle

FP32, BF16, RMS = 2.0 ** -18, 2.0 ** -8, 2.0 ** -9
GPU = pytest.param("cuda", marks=pytest.mark.gpu)


@pytest.fixture(autouse=True)
def _check_kernel_errors():
    yield
    if torch.cuda.is_available():
        kernels.check_error()


def inputs(T, E, dtype=torch.float32, seed=0, closed=0.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) * spread).to(dtype)
    if closed:
        off = torch.rand(T, E, generator=g) < closed
        off[::7] = True                     # no expert at all
        logits = logits.masked_fill(off, float("-inf"))
    return logits, torch.randn(E, generator=g) * 0.1


def choices(logits, k, score, bias, groups, top_groups):
    """The definition, one token after the other: [T][k] experts, -1 where the choice is not made."""
    found = []
    for row in logits.double().tolist():
        live = [l for l in row if l != -math.inf]
        if score == "sigmoid":
            s = [1 / (1 + math.exp(-l)) if l > -700 else 0.0 for l in row]
        else:
            top = max(live, default=0.0)
            whole = sum(math.exp(l - top) for l in live)
            s = [math.exp(l - top) / whole if l != -math.inf else 0.0 for l in row]
        c = torch.tensor(s, dtype=torch.float64).float()
        if bias is None and groups == 1:
            c = torch.tensor(row).float()
        elif bias is not None:
            c = c + bias
        c = [v if l != -math.inf else -math.inf for v, l in zip(c.tolist(), row)]
        n = len(row) // groups
        if groups > 1:
            total = []
            for g in range(groups):
                two = sorted((v for v in c[g * n:(g + 1) * n] if v != -math.inf), reverse=True)[:2]
                total.append(float(torch.tensor(two, dtype=torch.float32).sum()) if two else -math.inf)
            stay = sorted(range(groups), key=lambda g: (-total[g], g))[:top_groups]
            c = [v if e // n in stay else -math.inf for e, v in enumerate(c)]
        order = sorted(range(len(row)), key=lambda e: (-c[e], e))[:k]
        found.append([e if c[e] != -math.inf else -1 for e in order])
    return torch.tensor(found)


def exact(logits, k, experts, score, normalize, scale):
    """(weights, p) in 64 bits, differentiable, of the choices that were made (experts >= 0)."""
    l = logits.detach().double().requires_grad_()
    made = experts >= 0
    none = (l.detach() == -math.inf).all(1, keepdim=True)
    safe = torch.where(none, torch.zeros_like(l), l)
    log_s = torch.nn.functional.logsigmoid(safe) if score == "sigmoid" else torch.log_softmax(safe, 1)
    top = log_s.gather(1, experts.clamp_min(0))
    if normalize:
        top = torch.where(made, top, torch.full_like(top, -math.inf))
        w = torch.softmax(torch.where(made.any(1, keepdim=True), top, torch.zeros_like(top)), 1) * made
    else:
        w = torch.exp(torch.where(made, top, torch.zeros_like(top))) * made
    return l, scale * w, torch.softmax(log_s, 1) * ~none


def norm_off(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return float((got - want).norm() / want.norm().clamp_min(1e-30))


CASES = [      # T, E, k, score, biased, groups, top_groups, normalize, scale, closed
    (1, 1, 1, "sigmoid", False, 1, 1, True, 1.0, 0.0),
    (5, 2, 2, "softmax", True, 1, 0, True, 1.0, 0.0),
    (1, 8, 2, "sigmoid", True, 4, 2, True, 2.5, 0.0),
    (33, 9, 3, "sigmoid", True, 9, 5, False, 1.0, 0.3),
    (70, 15, 4, "softmax", True, 5, 2, True, 1.0, 0.3),
    (257, 24, 6, "softmax", False, 3, 2, False, 16.0, 0.2),
    (300, 63, 5, "sigmoid", False, 7, 3, True, 1.0, 0.0),
    (129, 64, 8, "sigmoid", True, 8, 4, True, 2.5, 0.0),
    (65, 160, 6, "softmax", False, 8, 3, False, 16.0, 0.1),
    (515, 128, 8, "sigmoid", True, 1, 0, True, 1.0, 0.0),
    (40, 256, 8, "sigmoid", True, 8, 4, True, 2.5, 0.0),
    (37, 374, 16, "softmax", True, 17, 4, True, 1.0, 0.1),      # groups of 22, two of 32 places each empty
    (37, 384, 16, "sigmoid", False, 1, 0, False, 1.0, 0.0),
    (37, 384, 7, "sigmoid", True, 32, 1, True, 1.0, 0.0),
    (64, 378, 4, "sigmoid", True, 9, 2, True, 1.0, 0.5),
    (900, 384, 8, "sigmoid", True, 8, 4, True, 2.5, 0.1),        # several tokens of a warp, 12, 16, 24 and 10 experts of a thread
    (700, 384, 6, "softmax", True, 3, 2, True, 1.0, 0.0),
    (600, 380, 8, "sigmoid", False, 20, 8, False, 1.0, 0.2),
    (777, 300, 8, "softmax", True, 1, 0, False, 1.0, 0.0),
]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, E, k, score, biased, groups, top_groups, normalize, scale, closed", CASES)
def test_against_the_definition(device, dtype, T, E, k, score, biased, groups, top_groups, normalize, scale, closed):
    logits, bias = inputs(T, E, dtype, seed=T + E, closed=closed)
    bias = bias if biased else None
    x = logits.to(device, copy=True).requires_grad_()
    r = moe.route(x, k, score=score, bias=None if bias is None else bias.to(device), groups=groups, top_groups=top_groups,
                  normalize=normalize, scale=scale)
    want = choices(logits, k, score, bias, groups, max(1, top_groups))
    made = r.slots.cpu() >= 0
    assert torch.equal(torch.where(made, r.experts.cpu().long(), -1), want)
    counts = torch.bincount(want[want >= 0], minlength=E)
    assert torch.equal(r.counts.cpu().long(), counts) and torch.equal(r.offsets.cpu().long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    flat, rows = want.reshape(-1), r.rows.cpu().long()
    order = sorted((i for i in range(T * k) if flat[i] >= 0), key=lambda i: (int(flat[i]), i))
    assert rows.tolist() == order + [-1] * (T * k - len(order))
    assert all(int(r.slots.view(-1)[i]) == n for n, i in enumerate(order))
    # weights, term and gradient
    l, w, p = exact(logits, k, want, score, normalize, scale)
    aux = E * (counts.double() / (T * k) * p.mean(0)).sum()
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
    ((w * dw).sum() + 0.3 * aux).backward()
    got, = torch.autograd.grad((r.weights, r.aux_loss), (x,), (dw.to(device), torch.tensor(0.3, device=device)))
    assert norm_off(r.weights, w) < FP32 and abs(float(r.aux_loss.detach() - aux.detach())) <= FP32 * abs(float(aux.detach()))
    assert got.dtype == dtype and torch.isfinite(got).all()
    if float(l.grad.norm()) > 1e-12:          # (one expert: the gradient is a difference of equals)
        slack = FP32 * float((w.detach() * dw).norm() + 0.3 * aux.detach()) / float(l.grad.norm())
        assert norm_off(got, l.grad) < slack + (BF16 if dtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("E, groups, top_groups, biased", [(64, 8, 4, True), (6, 3, 1, True), (128, 1, 0, True), (32, 4, 2, False)])
def test_ties_go_to_the_lowest_index(device, E, groups, top_groups, biased):
    """All equal: the first groups, the first experts; scores that round to 1 are equal too."""
    bias = torch.full((E,), 0.25, device=device) if biased else None
    for value in (0.0, 40.0, -3.0):
        r = moe.route(torch.full((9, E), value, device=device), 2, score="sigmoid", bias=bias, groups=groups, top_groups=top_groups)
        assert (r.experts.cpu() == torch.tensor([0, 1])).all() and torch.allclose(r.weights.cpu(), torch.tensor(0.5))
    logits = torch.tensor([[20.0, 30.0] * (E // 2)], device=device)          # both scores are 1 in fp32
    r = moe.route(logits, 2, score="sigmoid", bias=bias, groups=groups, top_groups=top_groups)
    assert r.experts.tolist() == [[0, 1]]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("normalize", [True, False])
def test_tiny_and_large_scores(device, normalize):
    """Scores that fp32 cannot hold keep their ratios; infinite logits have the score 1."""
    logits = torch.tensor([[-200.0, -201.0, -300.0, -200.5], [float("inf"), 0.0, -1.0, float("inf")], [-90.0, -95.0, 1.0, -2.0]], device=device)
    r = moe.route(logits.requires_grad_(), 2, score="sigmoid", normalize=normalize)
    assert r.experts.tolist() == [[0, 3], [0, 3], [2, 3]]
    if normalize:
        a = 1 / (1 + math.exp(-0.5))
        s2, s3 = 1 / (1 + math.exp(-1.0)), 1 / (1 + math.exp(2.0))
        want = torch.tensor([[a, 1 - a], [0.5, 0.5], [s2 / (s2 + s3), s3 / (s2 + s3)]])
    else:
        want = torch.tensor([[0.0, 0.0], [1.0, 1.0], [1 / (1 + math.exp(-1.0)), 1 / (1 + math.exp(2.0))]])
    assert torch.allclose(r.weights.detach().cpu(), want, rtol=2.0 ** -18, atol=1e-37)
    grad, = torch.autograd.grad((r.weights.sum(), r.aux_loss), (logits,), (torch.ones((), device=device), torch.ones((), device=device)))
    assert torch.isfinite(grad).all() and torch.isfinite(r.aux_loss).all()


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_bias_decides_the_choice_and_nothing_else(device):
    logits, _ = inputs(50, 16, seed=3)
    x = logits.to(device)
    bias = torch.zeros(16, device=device)
    bias[5], bias[6], bias[7] = 2.0, float("-inf"), -2.0
    r = moe.route(x, 3, score="sigmoid", bias=bias)
    assert (r.experts[:, 0] == 5).all() and not (r.experts == 6).any()
    s = torch.sigmoid(x.double()).gather(1, r.experts.long())
    assert norm_off(r.weights, s / s.sum(1, keepdim=True)) < FP32


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("E", [1, 3, 8, 384])
def test_balance_bias(device, E):
    g = torch.Generator().manual_seed(E)
    counts = torch.randint(0, 2 ** 30, (E,), generator=g, dtype=torch.int32)
    if E == 8:
        counts[:] = torch.tensor([4, 4, 4, 4, 4, 3, 5, 4])
    bias = torch.randn(E, generator=g)
    mean = sum(counts.tolist()) / E
    want = bias + torch.tensor([0.125 * ((c < mean) - (c > mean)) for c in counts.tolist()])
    b = bias.to(device)
    kept = b._version
    assert moe.balance_bias_(b, counts.to(device), 0.125) is b and torch.equal(b.cpu(), want) and b._version > kept


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_refusals(device):
    x = torch.randn(4, 12, device=device)
    bad = [dict(score="tanh"), dict(groups=5, top_groups=1), dict(groups=0), dict(groups=3), dict(groups=3, top_groups=4), dict(top_groups=2),
           dict(groups=6, top_groups=1), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=-1.0),
           dict(bias=torch.zeros(11, device=device)), dict(bias=torch.zeros(12, device=device, dtype=torch.bfloat16)),
           dict(bias=torch.zeros(1, 12, device=device))]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            moe.route(x, 3, **kw)
    for k in (0, 13):
        with pytest.raises(ValueError):
            moe.route(x, k, score="sigmoid")
    for bias, counts in ((torch.zeros(3), torch.zeros(4, dtype=torch.int32)), (torch.zeros(3), torch.zeros(3)),
                         (torch.zeros(3).bfloat16(), torch.zeros(3, dtype=torch.int32))):
        with pytest.raises((ValueError, TypeError)):
            moe.balance_bias_(bias.to(device), counts.to(device), 0.1)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_no_tokens(device):
    x = torch.randn(0, 8, device=device, requires_grad=True)
    r = moe.route(x, 2, score="sigmoid", bias=torch.zeros(8, device=device), groups=4, top_groups=2)
    assert r.weights.shape == (0, 2) and r.offsets.tolist() == [0] * 9 and float(r.aux_loss.detach()) == 0
    grad, = torch.autograd.grad((r.weights.sum() + r.aux_loss,), (x,))
    assert grad.shape == (0, 8)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_capacity_and_strides(device):
    """The first rows in token order keep their places, as without scores; logits in rows further apart, or in columns."""
    logits, bias = inputs(200, 16, seed=9)
    how = dict(score="sigmoid", bias=bias.to(device), groups=4, top_groups=2)
    r = moe.route(logits.to(device), 4, 20, **how)
    full = moe.route(logits.to(device), 4, **how)
    assert torch.equal(r.experts, full.experts) and int((r.offsets[1:] - r.offsets[:-1]).max()) == 20 and torch.equal(r.counts, full.counts)
    wide = torch.zeros(200, 40, device=device)
    wide[:, 3:19] = logits
    for x in (wide[:, 3:19], logits.to(device).t().contiguous().t()):
        s = moe.route(x, 4, 20, **how)
        assert all(torch.equal(a, b) for a, b in zip(s, r))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Along the gradient itself, in logits where no choice changes: a central difference in 64 bits of the plain statement."""
    logits, bias = inputs(32, 24, seed=4)
    for score in ("sigmoid", "softmax"):
        for normalize in (True, False):
            how = dict(score=score, bias=bias.cuda(), groups=4, top_groups=2, normalize=normalize, scale=2.0)
            x = logits.cuda().requires_grad_()
            r = moe.route(x, 3, **how)
            dw = torch.randn(32, 3, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
            grad, = torch.autograd.grad((r.weights, r.aux_loss), (x,), (dw, torch.ones((), device="cuda")))

            def value(l):
                _, w, p = exact(l, 3, r.experts.long().cpu(), score, normalize, 2.0)
                return float((w * dw.cpu()).sum() + 24 * (r.counts.cpu().double() / 96 * p.mean(0)).sum())

            d = grad.double().cpu() / grad.double().cpu().norm()
            h = 1e-4
            slope = (value(logits.double() + h * d) - value(logits.double() - h * d)) / (2 * h)
            # the difference is off by h^2 / 6 of a third derivative, bounded by the scale of the weights
            assert abs(slope - float(grad.norm())) < 1e-5 * float(grad.norm()) + 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 700])
def test_captured_and_replayed(T):
    """In a graph, with another stream's work in flight; the replay reads new logits and the bias that the step before left."""
    logits, bias = inputs(T, 32, seed=5)
    x, b = logits.cuda(), bias.cuda()
    how = dict(score="sigmoid", groups=4, top_groups=2)

    def step(l):
        l = l.detach().requires_grad_()
        r = moe.route(l, 4, bias=b, **how)
        dl, = torch.autograd.grad((r.weights.square().sum(), r.aux_loss), (l,), (torch.ones((), device="cuda"), torch.ones((), device="cuda")))
        moe.balance_bias_(b, r.counts, 0.01)
        return [r.weights.detach(), r.experts, r.rows, dl]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for seed in (6, 7):
        x.copy_(inputs(T, 32, seed=seed)[0])
        before = b.clone()
        graph.replay()
        after = b.clone()
        kept = [t.clone() for t in got]
        b.copy_(before)
        want = step(x)
        assert all(torch.equal(p, q) for p, q in zip(kept, want)) and torch.equal(b, after)


@pytest.mark.gpu
def test_every_output_is_written():
    debug.enable()
    try:
        for T in (1, 300):
            logits, bias = inputs(T, 48, seed=8)
            x = logits.cuda().requires_grad_()
            r = moe.route(x, 4, score="sigmoid", bias=bias.cuda(), groups=6, top_groups=3)
            torch.autograd.grad((r.weights.sum(), r.aux_loss), (x,), (torch.ones((), device="cuda"), torch.ones((), device="cuda")))
            assert debug.verify() >= 3
    finally:
        debug.enable(False)


def mlp_inputs(T, E, D, F, device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, D, generator=g)
    wgu, wd = torch.randn(E, 2 * F, D, generator=g) * D ** -0.5, torch.randn(E, D, F, generator=g) * F ** -0.5
    return [t.to(device, dtype) for t in (x, wgu, wd)] + [torch.randn(T, E, generator=g).to(device)]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 37, 600])
@pytest.mark.parametrize("act_bits", [16, 8])
def test_expert_mlp_with_scores(T, act_bits):
    """The whole feed-forward takes its routing from the scores, and its gradients reach logits and matrices through them.

    Against the plain statement in 64 bits at the same bf16 values: each of the chain's roundings (rows, activation, products, gradients) is
    2^-9 in the 2-norm, at most 8 of them in a row add to 8 RMS; in 8 bits gate and up are off by 2^-8 of their block's largest, some 3 of
    their own rms, which an activation and a product carry on: 16 RMS more."""
    E, D, F, k = 16, 64, 40, 3
    x, wgu, wd, logits = mlp_inputs(T, E, D, F, "cuda", torch.bfloat16, seed=T)
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 0.1
    how = moe.Scoring("sigmoid", bias, 4, 2, True, 2.5)
    with torch.no_grad():
        quiet, _ = moe.expert_mlp(x, logits, wgu, wd, k, scoring=how)
    leaves = [t.detach().requires_grad_() for t in (x, logits, wgu, wd)]
    out, aux = moe.expert_mlp(*leaves, k, act_bits=act_bits, scoring=how)
    dout = torch.randn(T, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    grads = torch.autograd.grad((out, aux), leaves, (dout, torch.tensor(0.1, device="cuda")))
    wide = [t.detach().double().requires_grad_() for t in (x, logits, wgu, wd)]
    want, want_aux = oracle.expert_mlp(*wide, k, scoring=how)
    wants = torch.autograd.grad((want, want_aux), wide, (dout.double(), torch.tensor(0.1, device="cuda", dtype=torch.float64)))
    assert norm_off(out, want) < 8 * RMS and norm_off(quiet, want) < 8 * RMS and abs(float(aux - want_aux)) < FP32 * float(want_aux)
    for got, w in zip(grads, wants):
        assert norm_off(got, w) < (24 if act_bits == 8 else 8) * RMS


def test_expert_mlp_plain_with_scores():
    x, wgu, wd, logits = mlp_inputs(9, 8, 16, 8, "cpu", torch.float64)
    how = moe.Scoring("sigmoid", torch.linspace(-0.2, 0.2, 8), 4, 2, False, 2.0)
    out, aux = moe.expert_mlp(x, logits, wgu, wd, 2, scoring=how)
    r = moe.route(logits, 2, score="sigmoid", bias=how.bias, groups=4, top_groups=2, normalize=False, scale=2.0)
    for t in range(9):
        y = torch.zeros(16, dtype=torch.float64)
        for j in range(2):
            e = int(r.experts[t, j])
            g, u = (x[t] @ wgu[e].t()).chunk(2)
            y += r.weights[t, j].double() * ((torch.nn.functional.silu(g) * u) @ wd[e].t())
        assert torch.allclose(out[t], y, rtol=1e-6, atol=1e-9)
    assert torch.equal(aux, r.aux_loss)


@pytest.mark.gpu
def test_forward_mode_and_second_gradients_are_refused():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    r = moe.route(x, 2, score="sigmoid")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(r.weights.square().sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError):
        moe.route(fwd.make_dual(x.detach(), torch.ones(4, 8, device="cuda")), 2, score="sigmoid")


@pytest.mark.gpu
def test_plain_and_native_choose_alike():
    """A long batch in both precisions: the same experts on the CPU and on the GPU."""
    for dtype in (torch.float32, torch.bfloat16):
        logits, bias = inputs(6000, 128, dtype, seed=11)
        for how in (dict(score="sigmoid", bias=bias), dict(score="softmax", bias=bias * 0.01, groups=8, top_groups=3),
                    dict(score="sigmoid", groups=4, top_groups=2), dict(score="softmax", normalize=False)):
            want = moe.route(logits, 6, **how)
            got = moe.route(logits.cuda(), 6, **{n: v.cuda() if torch.is_tensor(v) else v for n, v in how.items()})
            assert all(torch.equal(a.cpu(), b) for a, b in zip(got[2:], want[2:]))


def test_available_off_runs_the_plain_statements():
    ops.force_fallback(True)
    try:
        assert moe.route(torch.randn(3, 4), 2, score="sigmoid").weights.shape == (3, 2)
    finally:
        ops.force_fallback(False)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("T, E, k, score, biased, groups, top_groups", [
    (1, 8, 2, "softmax", False, 4, 2), (65, 160, 6, "softmax", False, 8, 3), (300, 63, 5, "sigmoid", False, 7, 3), (64, 9, 3, "sigmoid", True, 9, 5),
    (40, 256, 8, "sigmoid", True, 8, 4), (900, 384, 8, "softmax", False, 16, 4), (37, 374, 16, "softmax", True, 17, 4)])
def test_groups_by_their_largest_score(device, T, E, k, score, biased, groups, top_groups):
    """``group_scores`` 1, from its definition on whole tensors: the groups of the largest score, then the largest scores in them."""
    logits, bias = inputs(T, E, seed=E)
    s = (torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), 1)).float()
    c = s + bias if biased else s
    tops = c.view(T, groups, E // groups).amax(2)
    keep = torch.zeros(T, groups).scatter_(1, tops.topk(top_groups, 1).indices, 1).repeat_interleave(E // groups, 1) > 0
    want = c.masked_fill(~keep, float("-inf")).topk(k, 1).indices
    how = dict(score=score, bias=bias.to(device) if biased else None, groups=groups, top_groups=top_groups, normalize=False, scale=16.0)
    x = logits.to(device).requires_grad_()
    r = moe.route(x, k, group_scores=1, **how)
    assert torch.equal(r.experts.cpu().long(), want)
    _, w, _ = exact(logits, k, want, score, False, 16.0)
    assert norm_off(r.weights, w) < FP32
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
    l, w, _ = exact(logits, k, want, score, False, 16.0)
    (w * dw).sum().backward()
    got, = torch.autograd.grad(r.weights, x, dw.to(device))
    assert norm_off(got, l.grad) < FP32 * float((w.detach() * dw).norm()) / float(l.grad.norm())
    assert norm_off(moe.route(x, k, group_scores=2, **how).weights, moe.route(x, k, **how).weights) == 0


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_one_large_score_or_two_good_ones(device):
    """Where the two rules differ, and where a group has one open expert, or none."""
    inf = float("inf")
    logits = torch.tensor([[3.0, -3.0, 2.0, 2.0, 0.0, 0.0], [-inf, 1.0, 0.5, 0.5, -inf, -inf], [-inf] * 6], device=device)
    one = moe.route(logits, 2, score="sigmoid", groups=3, top_groups=1, group_scores=1)
    two = moe.route(logits, 2, score="sigmoid", groups=3, top_groups=1)
    assert one.experts[:2].tolist() == [[0, 1], [1, 0]] and two.experts[:2].tolist() == [[2, 3], [2, 3]]
    assert (one.slots >= 0).tolist() == [[True, True], [True, False], [False, False]]
    assert one.counts.tolist() == [1, 2, 0, 0, 0, 0] and float(one.weights[1, 0]) == 1.0


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_refusals_of_group_scores(device):
    x = torch.randn(4, 12, device=device)
    for bad in (0, 3, -1):
        with pytest.raises(ValueError):
            moe.route(x, 2, groups=3, top_groups=2, group_scores=bad)
        with pytest.raises(ValueError):
            moe.route(x, 2, group_scores=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 50])
def test_expert_mlp_with_group_scores(T):
    E, D, F, k = 16, 64, 40, 3
    x, wgu, wd, logits = mlp_inputs(T, E, D, F, "cuda", torch.bfloat16, seed=T)
    how = moe.Scoring("softmax", None, 4, 2, False, 2.5, 1)
    counts = torch.zeros(E, dtype=torch.int32, device="cuda")
    out, _ = moe.expert_mlp(x, logits, wgu, wd, k, scoring=how, counts=counts)
    want, _ = oracle.expert_mlp(*[t.double() for t in (x, logits, wgu, wd)], k, scoring=how)
    assert norm_off(out, want) < 8 * RMS
    assert torch.equal(counts, moe.route(logits, k, score="softmax", groups=4, top_groups=2, normalize=False, group_scores=1).counts)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("how", [dict(), dict(groups=2, top_groups=1), dict(groups=6, top_groups=3), dict(groups=3, top_groups=2, group_scores=1)])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("normalize", [False, True])
def test_rows_that_are_not_numbers(device, score, how, biased, normalize):
    """A NaN is no number to choose by, the largest there is: the lowest index has it first.  A term that such a row is part of is NaN, next to rows without experts
    too, and so are its weights; other rows are as without it."""
    inf, nan = float("inf"), float("nan")
    good = torch.tensor([[0.5, 1.0, 0.0, 2.0, 0.25, -1.0], [-inf] * 6])
    bias = torch.linspace(-0.1, 0.1, 6).to(device) if biased else None
    want = moe.route(good.to(device), 2, score=score, bias=bias, normalize=normalize, scale=2.0, **how)
    assert torch.isfinite(want.aux_loss)
    for row, first in (([nan] * 6, [0, 1]), ([-inf, -inf, nan, nan, -inf, -inf], [2, 3]), ([-inf, nan, nan, nan, nan, nan], None), ([nan, 0.0, 1.0, 2.0, 3.0, nan], None)):
        x = torch.cat([good, torch.tensor([row])]).to(device).requires_grad_()
        r = moe.route(x, 2, score=score, bias=bias, normalize=normalize, scale=2.0, **how)
        plain = moe.route(x.detach().cpu(), 2, score=score, bias=None if bias is None else bias.cpu(), normalize=normalize, scale=2.0, **how)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(r[2:], plain[2:]))
        assert first is None or how or r.experts[2].tolist() == first      # (groups: theirs have a say)
        assert torch.equal(r.weights[:2].detach(), want.weights) and torch.isnan(r.weights[2]).any() and torch.isnan(r.aux_loss)
        grad, = torch.autograd.grad((r.weights[:2].sum(), r.aux_loss), (x,), (torch.ones((), device=device), torch.zeros((), device=device)))
        assert torch.isfinite(grad[:2]).all() or device == "cpu"
