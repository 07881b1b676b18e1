"""Mixture-of-experts operators and 8-bit checkpoints on a GPU, at the edges: what is empty, refused, switched off or changed in place, and
gradients against differences along directions in which they are large.

Tolerances: RMS = 2^-9 is the 2-norm of a rounding to bf16, 2^-20 the router's fp32 arithmetic."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from torchure_b200 import ops
from torchure_b200.ops import act8, debug, kernels, moe

pytestmark = pytest.mark.gpu

RMS = 2.0 ** -9


@pytest.fixture(autouse=True)
def _check_kernel_errors():
    yield
    kernels.check_error()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(*shape, seed=0, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen(seed)) * std).bfloat16()


def mlp_inputs(T, E, D, F, seed=0):
    return (rand(T, D, seed=seed), torch.randn(T, E, device="cuda", generator=gen(seed + 1)),
            rand(E, 2 * F, D, seed=seed + 2, std=D ** -0.5), rand(E, D, F, seed=seed + 3, std=F ** -0.5))


def edges_of(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_combine_of_rows_without_columns():
    """A sum over no columns: the gradient of the weights is zero, not what lay in memory."""
    r = moe.route(torch.randn(5, 4, device="cuda", generator=gen(0)), 2)
    weights = r.weights.detach().requires_grad_()
    y = torch.empty(10, 0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    debug.enable()
    try:
        out = moe.combine(y, r._replace(weights=weights))
        dy, dw = torch.autograd.grad(out, (y, weights), torch.empty(5, 0, device="cuda", dtype=torch.bfloat16))
        debug.verify()
    finally:
        debug.enable(False)
    assert out.shape == (5, 0) and dy.shape == (10, 0) and dw.shape == (5, 2) and (dw == 0).all()


@pytest.mark.parametrize("name", ["route", "grouped_linear", "expert_mlp of a token", "expert_mlp", "expert_mlp by its matrices", "dispatch",
                                  "combine", "swiglu_8bit"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    """A tangent is never dropped without a word."""
    x, logits, wgu, wd = mlp_inputs(2 if name.endswith("token") else 40, 4, 64, 64)
    offsets = edges_of([0, 5, 10, 20, 40])
    r = moe.route(logits, 2)
    call, t = {
        "route": (lambda v: moe.route(v, 2), logits),
        "grouped_linear": (lambda v: moe.grouped_linear(v, wgu, offsets), x),
        "expert_mlp of a token": (lambda v: moe.expert_mlp(v, logits, wgu, wd, 2), x),
        "expert_mlp": (lambda v: moe.expert_mlp(x, v, wgu, wd, 2), logits),
        "expert_mlp by its matrices": (lambda v: moe.expert_mlp(x, logits, (wgu[:, :64], v), wd, 2), wgu[:, 64:]),
        "dispatch": (lambda v: moe.dispatch(v, r), x),
        "combine": (lambda v: moe.combine(v, r), rand(r.rows.numel(), 64)),
        "swiglu_8bit": (act8.swiglu_8bit, x),
    }[name]
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        call(t)


@pytest.mark.parametrize("N", [64, 33])
def test_grouped_linear_result_changes_in_place(N):
    offsets = edges_of([0, 7, 50])
    x, w, dy = rand(50, 64, seed=1).requires_grad_(), rand(2, N, 64, seed=2).requires_grad_(), rand(50, N, seed=3)
    y = moe.grouped_linear(x, w, offsets)
    y.mul_(2)
    got = torch.autograd.grad(y, (x, w), dy)
    want = torch.autograd.grad(moe.grouped_linear(x, w, offsets) * 2, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        y = moe.grouped_linear(x, w, offsets)
    y.mul_(torch.ones(N, device="cuda", requires_grad=True))
    assert y.requires_grad


@pytest.mark.parametrize("bits", [16, 8])
def test_experts_of_a_spread_layer_with_the_kernels_off(bits):
    """What runs on the buffers of a layer spread over ranks, on the plain statements on a GPU: in the layer's own precision."""
    from torchure_b200.parallel.expert_parallel import MoELayer

    torch.manual_seed(0)
    layer = MoELayer(64, 72, num_experts=4, top_k=2, experts="grouped", act_bits=bits).cuda()
    work = torch.randn(4, 9, 64, device="cuda", generator=gen(0))
    got = layer._grouped_products(work)
    ops.force_fallback(True)
    try:
        plain = layer._grouped_products(work)
        plain.sum().backward()
    finally:
        ops.force_fallback(False)
    assert plain.dtype == torch.float32 and layer.w_gate.grad is not None
    assert (got.double() - plain.double()).norm() < 5 * RMS * plain.double().norm()


def test_kernels_are_counted():
    """Few tokens are routed by one kernel, many by two."""
    for T, want in ((16, 1), (4096, 2)):
        logits = torch.randn(T, 8, device="cuda", generator=gen(0))
        moe.route(logits, 2)
        before = ops.launches()
        moe.route(logits, 2)
        assert ops.launches() - before == want


@pytest.mark.parametrize("rows,F,start", [(64, 256, 0), (1, 1, 0), (77, 519, 0), (9, 1000, 1), (33, 72, 3), (3, 4100, 1), (2, 5000, 0), (0, 64, 0)])
def test_swiglu_8bit_without_gradients(rows, F, start):
    """The bits of the activation are the same; a checkpoint that nobody will read is not made."""
    gu = rand(rows * 2 * F + start, seed=1)[start:].view(rows, 2 * F)
    want = act8.swiglu_8bit(gu.detach().requires_grad_()).detach()
    with torch.no_grad():
        assert torch.equal(act8.swiglu_8bit(gu), want)
    assert torch.equal(act8.swiglu_8bit(gu), want)


def test_swiglu_8bit_without_gradients_makes_no_checkpoint():
    gu = rand(2048, 2048, seed=1)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    act = act8.swiglu_8bit(gu)
    assert torch.cuda.max_memory_allocated() - before <= act.numel() * 2 + 4096


@pytest.mark.parametrize("edges,meant", [([0, 60, 20, 100], [0, 60, 60, 100]), ([0, -5, 50, 4000], [0, 0, 50, 100]),
                                         ([0, 2000000000, 2000000000, 7], [0, 100, 100, 100]), ([9, 30, 40, 90], [0, 30, 40, 90])])
@pytest.mark.parametrize("wide", [False, True])
def test_wrong_offsets_are_brought_into_range(edges, meant, wide):
    """Offsets that fall, are negative or pass the end count as the largest so far, within the rows; wide: by the kernels of many rows."""
    scale = 5 if wide else 1
    edges, meant = ([min(v * scale, 2 ** 31 - 1) for v in e] for e in (edges, meant))
    x, w, dy = rand(100 * scale, 64, seed=1), rand(3, 72, 64, seed=2), rand(100 * scale, 72, seed=3)

    def run(e):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = moe.grouped_linear(xl, wl, edges_of(e))
        return (y.detach(), *torch.autograd.grad(y, (xl, wl), dy))

    for a, b in zip(run(edges), run(meant)):
        assert torch.equal(a, b)


def test_grouped_gradients_against_differences_along_themselves():
    """The product is linear in rows and matrices: its value at (g, w), against dy, is the slope along g, which is |g|^2 where g is the gradient.
    The roundings of the result and of g are independent: their sum stays below 8 standard deviations, and the fp32 sums below 2^-20."""
    offsets = edges_of([0, 300, 300, 1000])
    x, w, dy = rand(1000, 256, seed=1).requires_grad_(), rand(3, 128, 256, seed=2).requires_grad_(), rand(1000, 128, seed=3)
    gx, gw = torch.autograd.grad(moe.grouped_linear(x, w, offsets), (x, w), dy)
    for g, y in ((gx, moe.grouped_linear(gx, w.detach(), offsets)), (gw, moe.grouped_linear(x.detach(), gw, offsets))):
        terms = y.double() * dy.double()
        want, own = g.double().square().sum(), g.double().square()
        assert (terms.sum() - want).abs() <= 8 * RMS * (terms.norm() + own.norm()) + 2.0 ** -20 * (terms.abs().sum() + want)


@pytest.mark.parametrize("T,E,k", [(300, 12, 3), (2000, 40, 8)])
def test_router_gradients_against_differences_along_themselves(T, E, k):
    """Both outputs of the router, apart: central differences of a step h along the sign of the gradient, so that the slope is the sum of its
    magnitudes.  Logits lie at least 4 h apart: no choice changes.  Along directions of entries +-1 the third derivative of a probability is at
    most 16 times the probability, so a difference is off by h^2 16 / 6 of the sum of |factor| times probability, and by 2^-20 / h of it for fp32."""
    h = 2.0 ** -5
    order = torch.rand(T, E, device="cuda", generator=gen(0)).add(torch.linspace(0, 0.8, E, device="cuda")).argsort(1).argsort(1)
    logits = (order.float() * (4 * h)).requires_grad_()
    dw = torch.randn(T, k, device="cuda", generator=gen(1))
    r = moe.route(logits, k)
    for name, g in (("weights", torch.autograd.grad(r.weights, logits, dw, retain_graph=True)[0]),
                    ("aux", torch.autograd.grad(r.aux_loss, logits, torch.tensor(2.0, device="cuda"))[0])):
        v = torch.sign(g)
        up, down = (moe.route((logits + s * h * v).detach(), k) for s in (1, -1))
        assert torch.equal(up.experts, r.experts) and torch.equal(down.experts, r.experts)
        if name == "weights":
            value, size = (lambda q: (q.weights.double() * dw.double()).sum()), (r.weights.detach().double() * dw.double().abs()).sum()
        else:
            value, size = (lambda q: 2 * q.aux_loss.double()), 2 * r.aux_loss.detach().double()
        slope, want = (value(up) - value(down)) / (2 * h), g.double().abs().sum()
        bound = size * (h * h * 16 / 6 + 2.0 ** -20 / h)
        assert want > 10 * bound and (slope - want).abs() <= bound + 2.0 ** -18 * want


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("T", [2, 100])
def test_expert_mlp_takes_logits_as_route_does(T, dtype):
    """A router under fp16 autocast, or one in fp64: as ``route``, in fp32, and the gradient in the logits' own type."""
    x, logits, wgu, wd = mlp_inputs(T, 6, 64, 64)
    leaf, same = logits.to(dtype).requires_grad_(), logits.to(dtype).float().requires_grad_()
    out, aux = moe.expert_mlp(x, leaf, wgu, wd, 2)
    want, waux = moe.expert_mlp(x, same, wgu, wd, 2)
    assert torch.equal(out, want) and torch.equal(aux, waux)
    dout = rand(T, 64, seed=9)
    got, = torch.autograd.grad((out, aux), (leaf,), (dout, torch.ones_like(aux)))
    ref, = torch.autograd.grad((want, waux), (same,), (dout, torch.ones_like(waux)))
    assert got.dtype == dtype and torch.equal(got, ref.to(dtype))
    with torch.no_grad():
        assert torch.equal(moe.expert_mlp(x, leaf, wgu, wd, 2)[0], moe.expert_mlp(x, same, wgu, wd, 2)[0])


@pytest.mark.parametrize("T", [300, 2500])
def test_expert_mlp_training_in_a_graph(T):
    """A pass with gradients is captured and replayed, with the second stream of many rows inside."""
    x, logits, wgu, wd = (t.requires_grad_() for t in mlp_inputs(T, 8, 128, 128))
    dout = rand(T, 128, seed=9)

    def once():
        out, aux = moe.expert_mlp(x, logits, wgu, wd, 2)
        return (out, *torch.autograd.grad((out, aux), (x, logits, wgu, wd), (dout, torch.ones_like(aux))))

    want = [t.detach().clone() for t in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))


def test_combine_needs_offsets():
    """The gradient reads the end of the last expert: a plan without experts is refused before a kernel looks for it."""
    r = moe.route(torch.randn(5, 4, device="cuda", generator=gen(0)), 2)
    y = rand(10, 16, seed=1).requires_grad_()
    with pytest.raises(ValueError, match="offsets"):
        moe.combine(y, r._replace(offsets=edges_of([])))
    with pytest.raises(ValueError, match="offsets"):
        moe.combine(y, r._replace(offsets=edges_of([10])))


def test_sizes_next_to_31_bits_are_refused():
    """Indexes of 32 bits run past the end by a tile, a block or a grid's stride.  Views without memory of their own: nothing is copied first."""
    long = 2 ** 31 - 100
    row = rand(1, 8, seed=1)
    tall = row.expand(long, 8)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    r = moe.route(torch.randn(4, 3, device="cuda", generator=gen(0)), 2)
    rows = torch.zeros(1, device="cuda", dtype=torch.int32)
    calls = {
        "quantize8": lambda: act8.quantize8(tall),
        "swiglu_8bit": lambda: act8.swiglu_8bit(tall),
        "route": lambda: moe.route(tall[:, :4], 1),
        "grouped_linear, rows": lambda: moe.grouped_linear(tall, row.view(1, 1, 8), edges_of([0, long])),
        "grouped_linear, matrices": lambda: moe.grouped_linear(row, row.view(1, 1, 8).expand(1, long, 8), edges_of([0, 1])),
        "expert_mlp, matrices": lambda: moe.expert_mlp(row, torch.zeros(1, 1, device="cuda"), row.view(1, 1, 8).expand(1, 2 ** 31, 8),
                                                       row[:, :1].expand(8, 2 ** 30).unsqueeze(0), 1),
        "dispatch": lambda: moe.dispatch(tall[:2 ** 30, :4], r._replace(slots=rows.expand(2 ** 30, 2), rows=rows.expand(2 ** 31))),
        "combine": lambda: moe.combine(tall[:, :4], r._replace(slots=rows.expand(1, long), weights=rows.float().expand(1, long))),
    }
    for name, call in calls.items():
        with pytest.raises((RuntimeError, ValueError), match="not supported|too many"):
            call()
        assert torch.cuda.max_memory_allocated() - before < 2 ** 20, name


def test_combine_of_no_choices():
    r = moe.route(torch.randn(5, 4, device="cuda", generator=gen(0)), 2)
    none = r._replace(weights=torch.empty(5, 0, device="cuda", requires_grad=True), slots=torch.empty(5, 0, device="cuda", dtype=torch.int32))
    y = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = moe.combine(y, none)
    dy, dw = torch.autograd.grad(out, (y, none.weights), torch.ones_like(out))
    assert (out == 0).all() and dy.shape == (0, 16) and dw.shape == (5, 0)
