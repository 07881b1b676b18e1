"""The mixture-of-experts kernels and the 8-bit checkpoints on a GPU, each against a plain statement in 64 bits.

Tolerances, from the number formats (U = 2^-8, the most that a rounding to bf16 takes; RMS = 2^-9, what many take in the 2-norm: an
error uniform in +-2^-8 / m for significands m in [1, 2) has 2^-9.2):
* one product: fp32 sums of bf16 products, rounded once: U |result| + 2^-18 sum |terms| (2^-23 for each addition of a chain that stays
  below 32 of them in a row per partial sum, with room).
* the whole feed-forward: at most five bf16 roundings in a row on the way to an output (gate / up, activation, product, weighted row,
  result), relative in the 2-norm: 5 RMS.
* router in fp32: 2^-20 relative (an exponential, a sum, a quotient).
"""

import math

import pytest
import torch

from torchure_b200.ops import act8, debug, kernels, moe, oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
RMS = 2.0 ** -9
NINF = float("-inf")


@pytest.fixture(autouse=True)
def _check_kernel_errors():
    yield
    kernels.check_error()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(*shape, seed=0, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen(seed)) * std).bfloat16()


def rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


# ---- router ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,k,capacity", [
    (1, 1, 1, 0), (1, 8, 2, 0), (1, 256, 8, 0), (5, 3, 3, 2), (64, 4, 4, 0), (129, 5, 1, 7), (300, 20, 3, 0), (1000, 33, 5, 100),
    (2049, 64, 8, 0), (4096, 8, 2, 1000), (777, 380, 16, 3), (9001, 128, 8, 600), (20000, 2, 1, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_route(T, E, k, capacity, dtype, masked):
    logits = torch.randn(T, E, device="cuda", generator=gen(T + E)).to(dtype)
    if masked:
        logits = logits.masked_fill(torch.rand(T, E, device="cuda", generator=gen(1)) < 0.4, NINF)
        logits[T // 2] = NINF
    dw = torch.randn(T, k, device="cuda", generator=gen(2))
    want = logits.cpu().double().requires_grad_()
    rw = oracle.route(want, k, capacity)
    (rw[0] * dw.cpu().double()).sum().add(0.5 * rw[6]).backward()
    leaf = logits.clone().requires_grad_()
    r = moe.route(leaf, k, capacity)
    for got, w in ((r.experts, rw[1]), (r.slots, rw[2]), (r.offsets, rw[3]), (r.rows, rw[4]), (r.counts, rw[5])):
        assert torch.equal(got.cpu(), w)
    assert rel(r.weights.cpu(), rw[0]) < 2.0 ** -20
    assert abs(r.aux_loss.item() - rw[6].item()) <= 2.0 ** -20 * abs(rw[6].item()) + 1e-12
    torch.autograd.backward((r.weights, r.aux_loss), (dw, torch.tensor(0.5, device="cuda")))
    tol = 2.0 ** -18 if dtype == torch.float32 else U
    # a gradient is a difference of terms as large as its row's largest weight times dw
    scale = max(want.grad.abs().max().item(), 1e-12)
    assert (leaf.grad.cpu().double() - want.grad).abs().max().item() <= tol * scale + 1e-7


def test_route_ties_and_signed_zeros():
    logits = torch.tensor([[0.0, -0.0, 0.0, -1.0], [-0.0, 0.0, -0.0, 0.0], [2.0, 2.0, 2.0, 2.0], [1.0, 3.0, 3.0, 1.0]], device="cuda")
    r = moe.route(logits, 3)
    assert r.experts.tolist() == [[0, 1, 2], [0, 1, 2], [0, 1, 2], [1, 2, 0]]


def test_route_rows_that_are_not_finite_stay_their_own():
    logits = torch.randn(40, 16, device="cuda", generator=gen(0))
    clean = moe.route(logits, 4)
    logits[3, 5] = float("nan")
    logits[9, 2] = float("inf")
    leaf = logits.clone().requires_grad_()
    r = moe.route(leaf, 4)
    assert torch.isnan(r.weights[3]).all() and r.experts[3, 0] == 5 and r.experts[9, 0] == 2
    keep = [t for t in range(40) if t not in (3, 9)]
    assert torch.equal(r.weights[keep], clean.weights[keep]) and torch.equal(r.experts[keep], clean.experts[keep])
    r.weights.sum().backward()
    assert torch.isfinite(leaf.grad[keep]).all() and torch.isnan(leaf.grad[3]).all()
    assert sorted(r.rows.tolist()) == list(range(160))


def test_route_no_tokens_and_strided_logits():
    r = moe.route(torch.empty(0, 4, device="cuda"), 2)
    assert r.offsets.tolist() == [0] * 5 and r.rows.numel() == 0 and r.aux_loss.item() == 0
    wide = torch.randn(50, 24, device="cuda", generator=gen(0))
    for part in (wide[:, 3:11], wide[::2, :8], wide.t()[:8].t()):
        a, b = moe.route(part, 2), moe.route(part.contiguous(), 2)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_route_same_bits_every_time():
    logits = torch.randn(8192, 64, device="cuda", generator=gen(0)).requires_grad_()
    first = None
    for _ in range(3):
        r = moe.route(logits, 8, 900)
        g, = torch.autograd.grad((r.weights.square().sum(), r.aux_loss), (logits,))
        now = [*r, g]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


# ---- rows ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,k,D,capacity", [(1, 4, 2, 8, 0), (37, 5, 3, 40, 0), (300, 8, 2, 1032, 60), (64, 8, 2, 7, 0), (513, 16, 4, 519, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dispatch_and_combine(T, E, k, D, capacity, dtype):
    r = moe.route(torch.randn(T, E, device="cuda", generator=gen(0)), k, capacity)
    weights = r.weights.detach().requires_grad_()
    r = r._replace(weights=weights)
    x = rand(T, D, seed=1).to(dtype).requires_grad_()
    dg = rand(T * k, D, seed=2)
    xg = moe.dispatch(x, r)
    want = oracle.dispatch(x.detach().double(), r.rows, k)
    assert xg.dtype == torch.bfloat16 and torch.equal(xg.double(), want)
    xg.backward(dg)
    xd = x.detach().double().requires_grad_()
    oracle.dispatch(xd, r.rows, k).backward(dg.double())
    assert rel(x.grad, xd.grad) < (U if dtype == torch.bfloat16 else 1e-6)

    y = rand(T * k, D, seed=3).requires_grad_()
    dout = rand(T, D, seed=4).to(dtype)
    out = moe.combine(y, r, dtype)
    yd, wd = y.detach().double().requires_grad_(), weights.detach().double().requires_grad_()
    ref = oracle.combine(yd, wd, r.slots)
    assert out.dtype == dtype and rel(out, ref.detach()) < (U if dtype == torch.bfloat16 else 1e-6)
    out.backward(dout)
    ref.backward(dout.double())
    assert rel(y.grad, yd.grad) < U and rel(weights.grad, wd.grad) < 1e-5


def test_combine_leaves_dropped_rows_out():
    """What lies in rows of no choice never reaches a sum, not even a NaN."""
    r = moe.route(torch.randn(64, 4, device="cuda", generator=gen(0)), 2, 8)
    y = rand(128, 16, seed=1)
    y[int(r.offsets[-1]):] = float("nan")
    assert torch.isfinite(moe.combine(y, r)).all()


# ---- grouped products -----------------------------------------------------------------------------------
def check_grouped(x, w, offsets, dy, fp32=False):
    """Forward, both gradients, element by element."""
    xl, wl = x.detach().requires_grad_(), (w.float() if fp32 else w.detach()).requires_grad_()
    y = moe.grouped_linear(xl, wl, offsets)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy)
    assert y.dtype == dx.dtype == torch.bfloat16 and dw.dtype == wl.dtype and dw.shape == w.shape
    xd, wd, dyd = x.double(), w.double(), dy.double()
    edge = offsets.tolist()
    for e, (a, b) in enumerate(zip(edge[:-1], edge[1:])):
        for got, p, q, u in ((y[a:b], xd[a:b], wd[e].t(), U), (dx[a:b], dyd[a:b], wd[e], U),
                             (dw[e], dyd[a:b].t(), xd[a:b], 2.0 ** -23 if fp32 else U)):
            want, size = p @ q, p.abs() @ q.abs()
            assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -18 * size + 1e-30).all()
    assert (y[edge[-1]:] == 0).all() and (dx[edge[-1]:] == 0).all()


GROUPS = [
    (64, 64, [0, 1]),
    (128, 256, [0, 0, 0, 5, 5]),
    (64, 128, [0, 16, 32, 48]),
    (520, 776, [0, 100, 100, 357, 1003]),
    (136, 72, [0, 255, 511, 512, 770]),
    (1024, 512, [0, 256, 512, 1024]),
    (256, 1544, [0, 700, 701, 703, 1500]),
    (8, 8, [0, 3, 130]),
]


@pytest.mark.parametrize("K,N,edges", GROUPS)
@pytest.mark.parametrize("fp32", [False, True])
def test_grouped_linear(K, N, edges, fp32):
    R, E = edges[-1], len(edges) - 1
    offsets = torch.tensor(edges, dtype=torch.int32, device="cuda")
    check_grouped(rand(R, K, seed=1), rand(E, N, K, seed=2, std=0.1), offsets, rand(R, N, seed=3), fp32)


@pytest.mark.parametrize("K,N", [(1, 1), (7, 9), (65, 130), (100, 33)])
def test_grouped_linear_widths_off_the_vectors(K, N):
    offsets = torch.tensor([0, 3, 3, 140], dtype=torch.int32, device="cuda")
    check_grouped(rand(140, K, seed=1), rand(3, N, K, seed=2), offsets, rand(140, N, seed=3))


def test_grouped_linear_rows_of_no_expert_and_no_rows():
    offsets = torch.tensor([0, 10, 90], dtype=torch.int32, device="cuda")
    check_grouped(rand(300, 64, seed=1), rand(2, 128, 64, seed=2), offsets, rand(300, 128, seed=3))
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    check_grouped(rand(70, 64, seed=1), rand(2, 128, 64, seed=2), offsets, rand(70, 128, seed=3))
    x, w = rand(0, 64).requires_grad_(), rand(2, 128, 64).requires_grad_()
    y = moe.grouped_linear(x, w, offsets)
    y.sum().backward()
    assert y.shape == (0, 128) and w.grad.abs().sum() == 0


def test_grouped_linear_strides():
    offsets = torch.tensor([0, 50, 200], dtype=torch.int32, device="cuda")
    wide, w = rand(400, 256, seed=1), rand(2, 96, 128, seed=2)
    for x in (wide[:200, 64:192], wide[::2, :128], wide[:200, 3:131], wide.t()[:128, :200].t(), wide[:1, :128].expand(200, 128)):
        check_grouped(x, w, offsets, rand(200, 96, seed=3))
    dy = rand(96, 200, seed=3).t()
    check_grouped(wide[:200, :128], w, offsets, dy)
    check_grouped(wide[:200, :128], rand(2, 128, 96, seed=2).transpose(1, 2), offsets, dy)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_grouped_linear_keeps_experts_apart(bad):
    """What one expert's rows or matrix hold reaches no other expert's results, also where their rows share a tile."""
    edges = [0, 37, 41, 41, 200]
    offsets = torch.tensor(edges, dtype=torch.int32, device="cuda")
    x, w, dy = rand(200, 128, seed=1), rand(4, 256, 128, seed=2), rand(200, 256, seed=3)

    def run(x, w, dy):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = moe.grouped_linear(xl, wl, offsets)
        return (y.detach(), *torch.autograd.grad(y, (xl, wl), dy))

    clean = run(x, w, dy)
    x[38], w[1], dy[39] = bad, bad, bad
    y, dx, dw = run(x, w, dy)
    rows = [r for r in range(200) if not 37 <= r < 41]
    assert torch.equal(y[rows], clean[0][rows]) and torch.equal(dx[rows], clean[1][rows])
    for e in (0, 2, 3):
        assert torch.equal(dw[e], clean[2][e])
    assert not torch.isfinite(y[37:41]).any() and not torch.isfinite(dw[1]).any()


def test_grouped_linear_does_not_follow_wrong_offsets_out_of_its_tensors():
    """Offsets that fall, are negative or pass the end: results are of no use, but other memory stays as it is."""
    x, w = rand(100, 64, seed=1), rand(3, 64, 64, seed=2)
    for edges in ([0, 60, 20, 100], [0, -5, 50, 4000], [0, 2000000000, 2000000000, 7]):
        offsets = torch.tensor(edges, dtype=torch.int32, device="cuda")
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        moe.grouped_linear(xl, wl, offsets).sum().backward()
        torch.cuda.synchronize()


def test_grouped_linear_same_bits_every_time():
    offsets = torch.tensor([0, 1000, 1100, 3000], dtype=torch.int32, device="cuda")
    x, w, dy = rand(3000, 512, seed=1).requires_grad_(), rand(3, 768, 512, seed=2).requires_grad_(), rand(3000, 768, seed=3)
    first = None
    for _ in range(3):
        y = moe.grouped_linear(x, w, offsets)
        now = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@pytest.mark.parametrize("E,R,K,N,seed", [(64, 5000, 256, 384, 0), (8, 12000, 512, 256, 1), (130, 3000, 128, 136, 2), (3, 40, 2048, 1024, 3)])
def test_grouped_linear_many(E, R, K, N, seed):
    cuts = torch.randint(0, R + 1, (E - 1,), generator=torch.Generator().manual_seed(seed)).sort().values.tolist()
    offsets = torch.tensor([0, *cuts, R], dtype=torch.int32, device="cuda")
    check_grouped(rand(R, K, seed=1), rand(E, N, K, seed=2, std=0.05), offsets, rand(R, N, seed=3))


# ---- 8-bit checkpoints -------------------------------------------------------------------------------------
def kept64(x):
    """What 8 bits stand for, in 64 bits."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -cols % 64)).view(rows, -1, 64)
    a = b.abs().amax(-1, keepdim=True)
    q = torch.where(a > 0, torch.floor(b.abs() * 127 / a.clamp_min(1e-300) + 0.5) * b.sign(), 0.0)
    return (q * a / 127).view(rows, -1)[:, :cols]


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 63), (2, 64), (77, 519), (5, 1000), (1000, 256), (4097, 72)])
def test_quantize8(rows, cols):
    x = rand(rows, cols, seed=rows)
    x[:, ::5] = (x[:, :1].float() / 2).bfloat16()         # half-way cases where the first value is the largest
    x[0, :] *= 1e-30
    kept = act8.quantize8(x)
    want = oracle.quantize8(x.cpu())
    assert torch.equal(kept.values.cpu(), want[0]) and torch.equal(kept.scales.cpu(), want[1])
    got = act8.dequantize8(kept)
    assert ((got.double() - kept64(x)).abs() <= U * kept64(x).abs()).all()


def test_quantize8_every_bf16_magnitude_and_ratio():
    """All pairs of 8-bit significands: the rounding is that of the exact quotient, halves away from zero."""
    a = torch.arange(128, 256, device="cuda").float()
    blocks = torch.cat([a[:, None].expand(128, 1), torch.zeros(128, 63, device="cuda")], 1)
    rows = []
    for shift in range(9):
        for part in range(0, 128, 63):
            b = blocks.clone()
            vals = a[part:part + 63] / 2.0 ** shift
            b[:, 1:1 + vals.numel()] = vals
            rows.append(torch.where(b <= b[:, :1], b, torch.zeros_like(b)))
    x = torch.cat(rows).bfloat16()
    x = torch.cat([x, -x])
    values = act8.quantize8(x).values.cpu().double()
    b = x.cpu().double()
    top = b.abs().amax(1, keepdim=True)
    want = torch.floor((2 * b.abs() * 127 + top) / (2 * top)) * b.sign()       # numerators and denominators are exact
    assert torch.equal(values, want)


def test_quantize8_not_finite_tiny_and_strided():
    x = torch.ones(4, 192, device="cuda", dtype=torch.bfloat16)
    x[0, :64] = 0.0
    x[1, 70], x[1, 130] = float("nan"), NINF
    x[2, :64] = 1e-39
    x[3, 5] = 3.3e38
    got = act8.dequantize8(act8.quantize8(x))
    assert (got[0, :64] == 0).all() and (got[0, 64:] == 1).all() and (got[1, :64] == 1).all() and torch.isnan(got[1, 64:]).all()
    assert (got[2, :64] == 0).all() and got[3, 5] == x[3, 5] and (got[3, 64:] == 1).all()
    wide = rand(60, 400, seed=1)
    for part in (wide[:, 8:136], wide[:, 3:200], wide[::3], wide.t()):
        a, b = act8.quantize8(part), act8.quantize8(part.contiguous())
        assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)
    assert act8.quantize8(x[:0]).values.shape == (0, 192)


@pytest.mark.parametrize("shape", [(1, 2), (3, 130), (333, 2000), (2, 5, 256), (1000, 384)])
def test_swiglu_8bit(shape):
    gu = rand(*shape, seed=1).requires_grad_()
    act = act8.swiglu_8bit(gu)
    dact = rand(*act.shape, seed=2)
    dgu, = torch.autograd.grad(act, (gu,), dact)
    F = shape[-1] // 2
    flat = gu.detach().reshape(-1, 2 * F)
    want = oracle.swiglu_plain(flat.double())
    # the activation: one rounding, and the sigmoid's 2^-20
    assert ((act.reshape(-1, F).double() - want).abs() <= (U + 2.0 ** -20) * want.abs() + 1e-38).all()
    k = torch.cat([kept64(flat[:, :F]), kept64(flat[:, F:])], 1).requires_grad_()
    oracle.swiglu_plain(k).backward(dact.reshape(-1, F).double())
    # d(gate) is d u s (1 + g (1 - s)): where the bracket vanishes what is left is the rounding of its terms
    d, u = dact.reshape(-1, F).double().abs(), k.detach()[:, F:].abs()
    slack = torch.cat([d * u, d * k.detach()[:, :F].abs()], 1) * 2.0 ** -20
    assert ((dgu.reshape(-1, 2 * F).double() - k.grad).abs() <= U * k.grad.abs() + slack + 1e-38).all()


@pytest.mark.parametrize("rows,cols", [(1, 7), (2000, 33), (300, 2557), (9, 8191), (3, 8193), (100, 64), (1777, 201)])
@pytest.mark.parametrize("start", [0, 1, 5])
def test_rows_on_any_boundary(rows, cols, start):
    """Widths off the vectors, rows that start anywhere and tiles of several rows give the bits of a padded, aligned copy."""
    def at(n, seed):        # n columns, the first of them `start` values past an aligned address
        return rand(rows * n + start, seed=seed)[start:].view(rows, n)

    x = at(cols, 1)
    room = -cols % 64
    a, b = act8.quantize8(x), act8.quantize8(torch.nn.functional.pad(x, (0, room)))
    assert torch.equal(a.values, b.values[:, :cols]) and torch.equal(a.scales, b.scales)
    assert torch.equal(act8.dequantize8(a), act8.dequantize8(b)[:, :cols])

    def halves(t):
        return torch.nn.functional.pad(t.view(rows, 2, cols), (0, room)).reshape(rows, -1)

    gu, dact = at(2 * cols, 2), at(cols, 3)
    odd, even = gu.clone().requires_grad_() if start == 0 else gu.requires_grad_(), halves(gu.detach()).requires_grad_()
    act, want = act8.swiglu_8bit(odd), act8.swiglu_8bit(even)
    assert torch.equal(act, want[:, :cols])
    d1, = torch.autograd.grad(act, (odd,), dact)
    d2, = torch.autograd.grad(want, (even,), torch.nn.functional.pad(dact, (0, room)))
    assert torch.equal(d1, d2.view(rows, 2, -1)[:, :, :cols].reshape(rows, -1))


def test_swiglu_8bit_keeps_half_the_bytes():
    gu = rand(4096, 2048, seed=1).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    act = act8.swiglu_8bit(gu)
    kept = torch.cuda.memory_allocated() - before - act.numel() * 2
    assert kept <= gu.numel() * (1 + 4 / 64) + 4096


# ---- the whole feed-forward ---------------------------------------------------------------------------------
def mlp_inputs(T, E, D, F, seed=0, dtype=torch.bfloat16):
    return (rand(T, D, seed=seed).to(dtype), torch.randn(T, E, device="cuda", generator=gen(seed + 1)),
            rand(E, 2 * F, D, seed=seed + 2, std=D ** -0.5), rand(E, D, F, seed=seed + 3, std=F ** -0.5))


def check_mlp(T, E, k, D, F, capacity=0, dtype=torch.bfloat16, bits=16, fp32=False, pair=False, masked=False):
    x, logits, wgu, wd = mlp_inputs(T, E, D, F, dtype=dtype)
    if masked:
        logits[::3] = NINF
    if fp32:
        wgu, wd = wgu.float(), wd.float()
    leaves = [t.clone().requires_grad_() for t in (x, logits, wgu, wd)]
    w = (leaves[2][:, :F], leaves[2][:, F:]) if pair else leaves[2]
    out, aux = moe.expert_mlp(leaves[0], leaves[1], w, leaves[3], k, capacity, bits)
    dout = rand(T, D, seed=9).to(dtype)
    torch.autograd.backward((out, aux), (dout, torch.tensor(0.3, device="cuda")))
    ref = [t.detach().cpu().double().requires_grad_() for t in (x, logits, wgu, wd)]
    want, waux = oracle.expert_mlp(*ref, k, capacity, bits)
    torch.autograd.backward((want, waux), (dout.cpu().double(), torch.tensor(0.3, dtype=torch.float64)))
    # 8 bits: gate and up off by 1 / 254 of the largest of 64 values (about 2.5 of their deviation), flips between neighbours
    # included on either side
    tol = 5 * RMS if bits == 16 else 5 * RMS + 2 * 2.5 / 127
    assert out.dtype == dtype and rel(out.cpu(), want.detach()) < 5 * RMS
    assert abs(aux.item() - waux.item()) < 2.0 ** -20 * waux.item()
    for got, r in zip(leaves, ref):
        assert got.grad.dtype == got.dtype and rel(got.grad.cpu(), r.grad) < tol
    with torch.no_grad():
        again, aux2 = moe.expert_mlp(x, logits, (wgu[:, :F], wgu[:, F:]) if pair else wgu, wd, k, capacity, bits)
    assert rel(again.cpu(), want.detach()) < 5 * RMS and torch.equal(aux2, aux.detach())


@pytest.mark.parametrize("T,E,k,D,F,capacity", [
    (1, 8, 2, 256, 192, 0), (3, 4, 1, 64, 64, 0), (16, 8, 2, 128, 72, 0), (61, 16, 4, 256, 136, 0), (300, 8, 2, 520, 264, 80),
    (1024, 5, 3, 256, 512, 0), (2000, 32, 4, 128, 128, 300)])
def test_expert_mlp(T, E, k, D, F, capacity):
    check_mlp(T, E, k, D, F, capacity)


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32, fp32=True), dict(fp32=True, pair=True), dict(bits=8), dict(masked=True),
                                dict(bits=8, dtype=torch.float32, fp32=True, pair=True, capacity=90)])
def test_expert_mlp_forms(kw):
    check_mlp(400, 6, 2, 256, 200, **kw)


@pytest.mark.parametrize("T,E,k,D,F,capacity", [(1, 8, 2, 1024, 264, 0), (2, 1, 1, 8, 8, 0), (3, 40, 7, 520, 136, 0), (4, 300, 8, 264, 72, 0),
                                                (4, 4, 2, 64, 64, 1), (2, 16, 16, 128, 32, 0)])
@pytest.mark.parametrize("dtype,logit", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_expert_mlp_of_a_few_tokens(T, E, k, D, F, capacity, dtype, logit):
    """Without gradients up to four tokens take kernels of their own: no rounding but the result's."""
    x, logits, wgu, wd = mlp_inputs(T, E, D, F, dtype=dtype)
    logits = logits.to(logit)
    if E > 4:
        logits[0, :E - k + 1] = NINF          # the last choice of the first token is not made
    for closed in (False, True):
        if closed:
            logits[T - 1] = NINF
        with torch.no_grad():
            out, aux = moe.expert_mlp(x, logits, wgu, wd, k, capacity)
        want, waux = oracle.expert_mlp(*(t.cpu().double() for t in (x, logits, wgu, wd)), k, capacity)
        assert out.dtype == dtype and aux.dtype == torch.float32
        size = want.abs().max(1, keepdim=True).values
        assert ((out.cpu().double() - want).abs() <= (U if dtype == torch.bfloat16 else 2.0 ** -16) * size).all()
        assert abs(aux.item() - waux.item()) <= 2.0 ** -20 * waux.item()
        assert not closed or (out[T - 1] == 0).all()


@pytest.mark.parametrize("T,E,k,D,F", [(100, 8, 2, 256, 136), (130, 40, 4, 72, 64), (61, 16, 4, 1024, 200), (300, 20, 2, 264, 72)])
@pytest.mark.parametrize("bits", [16, 8])
def test_expert_mlp_of_uneven_groups(T, E, k, D, F, bits):
    """Few rows per expert on average, but one expert has every token (more than one tile of rows), others have none."""
    x, logits, wgu, wd = mlp_inputs(T, E, D, F)
    logits[:, E // 2] += 100
    logits[:, ::3] = NINF
    leaves = [t.clone().requires_grad_() for t in (x, logits, wgu, wd)]
    out, aux = moe.expert_mlp(*leaves, k, act_bits=bits)
    dout = rand(T, D, seed=9)
    out.backward(dout)
    ref = [t.detach().cpu().double().requires_grad_() for t in (x, logits, wgu, wd)]
    want, _ = oracle.expert_mlp(*ref, k, 0, bits)
    want.backward(dout.cpu().double())
    assert rel(out.detach().cpu(), want.detach()) < 5 * RMS
    for got, r in list(zip(leaves, ref))[2:]:
        assert rel(got.grad.cpu(), r.grad) < (5 * RMS if bits == 16 else 5 * RMS + 2 * 2.5 / 127)
        assert not got.grad[moe.route(logits, k).counts == 0].any()
    with torch.no_grad():
        assert rel(moe.expert_mlp(x, logits, wgu, wd, k)[0].cpu(), want.detach()) < 5 * RMS


def test_expert_mlp_reads_matrices_that_were_just_written():
    """The kernels of a pass overlap, and read matrices early: never before what wrote them has ended, whoever wrote them."""
    E, D, F = 8, 512, 384
    x, logits, _, _ = mlp_inputs(64, E, D, F)
    r = moe.route(torch.randn(4096, 8, device="cuda", generator=gen(5)), 1)
    sources = [rand(4096, E * F * D * 3 // 4096, seed=s, std=D ** -0.5) for s in range(4)]

    def split(flat):
        flat = flat.reshape(-1)
        return flat[:E * 2 * F * D].view(E, 2 * F, D), flat[E * 2 * F * D:].view(E, D, F)

    with torch.no_grad():
        order = [src[r.rows.long()] for src in sources]
        want = [moe.expert_mlp(x, logits, *split(o), 2)[0] for o in order]
        torch.cuda.synchronize()
        held = torch.empty_like(order[0])
        for i in range(40):
            if i % 2:
                held.copy_(order[i % 4])
                got = moe.expert_mlp(x, logits, *split(held), 2)[0]
            else:
                got = moe.expert_mlp(x, logits, *split(moe.dispatch(sources[i % 4], r)), 2)[0]
            assert torch.equal(got, want[i % 4])


def test_expert_mlp_gradient_of_aux_alone_and_no_tokens():
    x, logits, wgu, wd = mlp_inputs(32, 4, 64, 64)
    logits.requires_grad_()
    out, aux = moe.expert_mlp(x, logits, wgu, wd, 2)
    aux.backward()
    ref = logits.detach().cpu().double().requires_grad_()
    oracle.route(ref, 2)[6].backward()
    assert rel(logits.grad.cpu(), ref.grad) < 1e-5
    out, aux = moe.expert_mlp(x[:0], logits[:0], wgu.clone().requires_grad_(), wd, 2)
    assert out.shape == (0, 64) and aux.item() == 0
    leaves = [t.detach().clone().requires_grad_() for t in (x[:0], logits[:0], wgu, wd)]
    out, aux = moe.expert_mlp(*leaves, 2)
    (out.sum() + aux).backward()
    assert all(t.grad.shape == t.shape and t.grad.abs().sum() == 0 for t in leaves)


def test_operators_on_another_stream():
    """Inputs made on one stream, used on another, in order: the kernels run on the current stream."""
    x, logits, wgu, wd = mlp_inputs(500, 8, 256, 256)
    want, _ = moe.expert_mlp(x, logits, wgu, wd, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = moe.expert_mlp(x, logits, wgu, wd, 2)
        kept = act8.dequantize8(act8.quantize8(got))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(kept, act8.dequantize8(act8.quantize8(want)))


def test_expert_mlp_in_a_graph():
    x, logits, wgu, wd = mlp_inputs(64, 8, 256, 256)
    with torch.no_grad():
        want, _ = moe.expert_mlp(x, logits, wgu, wd, 2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            moe.expert_mlp(x, logits, wgu, wd, 2)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, _ = moe.expert_mlp(x, logits, wgu, wd, 2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        logits.copy_(logits.roll(1, 1))          # other groups through the same graph
        graph.replay()
        assert torch.equal(got, moe.expert_mlp(x, logits, wgu, wd, 2)[0])


def test_every_output_is_written():
    """With outputs poisoned beforehand, no poison is left: rows of dropped choices and ragged tiles included."""
    debug.enable()
    try:
        for T, capacity, bits in ((1, 0, 16), (200, 30, 16), (200, 0, 8), (2000, 300, 8)):
            x, logits, wgu, wd = (t.requires_grad_() for t in mlp_inputs(T, 8, 264, 136))
            out, aux = moe.expert_mlp(x, logits, wgu, wd, 2, capacity, bits)
            torch.autograd.grad((out, aux), (x, logits, wgu, wd), (torch.ones_like(out), torch.ones_like(aux)))
            r = moe.route(logits, 2, capacity)
            y = moe.grouped_linear(moe.dispatch(x, r), wgu, r.offsets)
            torch.autograd.grad(moe.combine(y, r).float().sum(), (x, logits, wgu))
            act8.dequantize8(act8.quantize8(y))
            assert debug.verify() > 10
    finally:
        debug.enable(False)


def test_layer_and_model_on_the_operators():
    """The mixture layer in mixed precision, padded buffers against grouped products; then a model's step on them."""
    from torchure_b200.models import build_model
    from torchure_b200.objectives import ARObjective
    from torchure_b200.parallel.expert_parallel import MoELayer

    torch.manual_seed(0)
    old = MoELayer(256, 192, num_experts=8, top_k=2, capacity_factor=1.25).cuda()
    x = torch.randn(2, 150, 256, device="cuda")
    for bits in (16, 8):
        new = MoELayer(256, 192, num_experts=8, top_k=2, capacity_factor=1.25, experts="grouped", act_bits=bits).cuda()
        new.load_state_dict(old.state_dict())
        res = []
        for layer in (old, new):
            layer.zero_grad()
            xi = x.clone().requires_grad_()
            with torch.autocast("cuda", dtype=torch.bfloat16):
                out = layer(xi)
            (out.square().sum() + layer.aux_loss).backward()
            res.append([out.detach(), xi.grad, layer.w_gate.grad, layer.w_up.grad, layer.w_down.grad])
        for a, b in zip(*res):
            assert a.dtype == b.dtype == torch.float32 and rel(b, a) < 10 * RMS + (0.04 if bits == 8 else 0)
    cfg = dict(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, head_dim=128, vocab_size=512, num_experts=8, top_k=2,
               moe_ffn_dim=128, capacity_factor=1.25, experts="grouped", act_bits=8)
    model = build_model("qwen3_moe", cfg).cuda()
    model.init_weights()
    ids = torch.randint(0, 512, (2, 128), device="cuda")
    opt = torch.optim.SGD(model.parameters(), lr=0.05)
    losses = []
    for _ in range(8):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = ARObjective(fused_linear_ce=True, ce_chunk_size=256).compute_loss(model, {"input_ids": ids, "labels": ids})
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < losses[0]


def test_refusals_on_the_gpu():
    x, w = rand(4, 64), rand(3, 64, 64)
    offsets = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError, match="bf16 rows"):
        moe.grouped_linear(x.float(), w, offsets)
    with pytest.raises(ValueError, match="int32"):
        moe.grouped_linear(x, w, offsets.long())
    with pytest.raises(ValueError, match="GPU"):
        moe.grouped_linear(x, w, offsets.cpu())
    with pytest.raises(ValueError, match="experts"):
        moe.route(torch.randn(4, 385, device="cuda"), 2)
    with pytest.raises(ValueError, match="top_k"):
        moe.route(torch.randn(4, 64, device="cuda"), 17)
    xs, logits, wgu, wd = mlp_inputs(4, 3, 64, 64)
    with pytest.raises(ValueError, match="multiples of 8"):
        moe.expert_mlp(xs[:, :60].contiguous(), logits, wgu[:, :, :60].contiguous(), wd[:, :60].contiguous(), 2)
    with pytest.raises(TypeError, match="one type"):
        moe.expert_mlp(xs, logits, wgu.float(), wd, 2)
    with pytest.raises(TypeError, match="bf16"):
        act8.swiglu_8bit(torch.randn(4, 64, device="cuda"))
    kept = act8.quantize8(x)
    with pytest.raises(RuntimeError, match="do not match"):
        act8.dequantize8(act8.Act8(kept.values, kept.scales[:2]))
    with pytest.raises(ValueError, match="int32"):
        moe.combine(rand(8, 64), moe.route(logits, 2)._replace(slots=torch.zeros(4, 2, dtype=torch.int64, device="cuda")))


def test_expert_mlp_backward_on_another_stream_under_allocation_pressure():
    """The backward pass of many rows uses a second stream inside; to the caller and the allocator there is one.  Blocks that are freed
    right behind it and overwritten on the caller's stream must not reach what the pass still reads or has returned."""
    x, logits, wgu, wd = (t.requires_grad_() for t in mlp_inputs(2500, 8, 256, 256))
    dout = rand(2500, 256, seed=9)

    def once():
        out, aux = moe.expert_mlp(x, logits, wgu, wd, 2)
        return torch.autograd.grad((out, aux), (x, logits, wgu, wd), (dout, torch.ones_like(aux)))

    want = [g.clone() for g in once()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            for _ in range(6):
                got = once()
                junk = [torch.full((5000, n), float("nan"), device="cuda", dtype=torch.bfloat16) for n in (256, 512, 256, 1024)]
                for g, w in zip(got, want):
                    assert torch.equal(g, w)
                del got, junk


def test_offsets_beyond_31_bits():
    """Matrices of more than 2^31 elements: the last rows are those of a small call."""
    R, K, N = 1_100_000, 64, 2048
    x, w = rand(R, K, seed=1), rand(3, N, K, seed=2)
    edges = [0, 500_000, 1_099_000, R]
    y = moe.grouped_linear(x, w, torch.tensor(edges, dtype=torch.int32, device="cuda"))
    tail = moe.grouped_linear(x[-1000:], w[2:], torch.tensor([0, 1000], dtype=torch.int32, device="cuda"))
    assert y.numel() > 2 ** 31 and torch.equal(y[-1000:], tail)
    act = act8.swiglu_8bit(y)
    assert torch.equal(act[-1000:], act8.swiglu_8bit(tail))
    kept = act8.quantize8(y)
    small = act8.quantize8(tail)
    assert torch.equal(kept.values[-1000:], small.values) and torch.equal(kept.scales[-1000:], small.scales)
    assert torch.equal(act8.dequantize8(kept)[-1000:], act8.dequantize8(small))
    r = moe.route(torch.randn(R, 2, device="cuda", generator=gen(3)), 1)
    rows = moe.dispatch(y, r)
    out = moe.combine(rows, r)          # one choice of weight 1: what went in comes out
    assert torch.equal(out[-1000:], y[-1000:]) and torch.equal(out[:1000], y[:1000])


def test_gradients_against_differences():
    """The operators' own gradients against differences of their own outputs along random directions, where a step is large against
    the rounding: grouped products are linear, so that a step of any size gives the slope."""
    offsets = torch.tensor([0, 300, 300, 1000], dtype=torch.int32, device="cuda")
    x, w, dy = rand(1000, 256, seed=1), rand(3, 128, 256, seed=2), rand(1000, 128, seed=3)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(moe.grouped_linear(xl, wl, offsets), (xl, wl), dy)
    loss = lambda a, b: (moe.grouped_linear(a, b, offsets).double() * dy.double()).sum().item()
    vx, vw = rand(1000, 256, seed=4), rand(3, 128, 256, seed=5)
    for slope, g, v, scale in ((loss(vx, w), gx, vx, (vx.double() @ w[0].double().t()).norm()),
                               (loss(x, vw), gw, vw, (x.double() @ vw[0].double().t()).norm())):
        want = (g.double() * v.double()).sum().item()
        assert abs(slope - want) <= 4 * RMS * scale.item() * dy.double().norm().item() / 10
    logits = torch.randn(300, 12, device="cuda", generator=gen(6)).requires_grad_()
    dw = torch.randn(300, 3, device="cuda", generator=gen(7))
    r = moe.route(logits, 3)
    g, = torch.autograd.grad((r.weights, r.aux_loss), (logits,), (dw, torch.tensor(2.0, device="cuda")))
    v = torch.randn(300, 12, device="cuda", generator=gen(8))
    h = 2.0 ** -8           # smaller than the gaps between chosen and unchosen logits of the rows compared below

    def value(t):
        q = moe.route(t, 3)
        return q, (q.weights.double() * dw.double()).sum(1)

    (qp, up), (qm, down) = value(logits.detach() + h * v), value(logits.detach() - h * v)
    same = ((qp.experts == r.experts) & (qm.experts == r.experts)).all(1)
    aux = 2.0 * (qp.aux_loss.double() - qm.aux_loss.double()) / (2 * h)
    slope = ((up - down) / (2 * h))[same].sum().item() + (aux.item() if same.all() else 0.0)
    only = torch.autograd.grad(moe.route(logits, 3).weights, (logits,), dw)[0]
    want = (only.double() * v.double())[same].sum().item()
    # second-order term h^2 / 6 of functions bounded by |dw| with |v| of a few, and 2^-22 / h from the weights' rounding, over 900 terms
    assert same.sum() > 200 and abs(slope - (aux.item() if same.all() else 0.0) - want) <= 900 * (h * h * 4 + 2.0 ** -22 / h)
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("T", [40, 2100])
@pytest.mark.parametrize("pair", [False, True])
def test_expert_mlp_gradients_one_at_a_time(T, pair):
    """What is asked for alone has the bits it has among all; what is not asked for is not computed."""
    from torchure_b200 import ops

    x, logits, wgu, wd = (t.requires_grad_() for t in mlp_inputs(T, 6, 128, 72))
    gate, up = (wgu.detach()[:, i:i + 72].clone().requires_grad_() for i in (0, 72))
    leaves = [x, logits, gate, up, wd] if pair else [x, logits, wgu, wd]
    dout = rand(T, 128, seed=9)

    def grads(of):
        out, aux = moe.expert_mlp(x, logits, (gate, up) if pair else wgu, wd, 2)
        before = ops.launches()
        got = torch.autograd.grad((out, aux), of, (dout, torch.ones_like(aux)))
        return got, ops.launches() - before

    want, launches = grads(leaves)
    for leaf, w in zip(leaves, want):
        (got,), fewer = grads([leaf])
        assert torch.equal(got, w) and fewer < launches


def test_gradients_have_no_gradient():
    x, w = rand(8, 64).requires_grad_(), rand(2, 64, 64).requires_grad_()
    offsets = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(moe.grouped_linear(x, w, offsets).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(act8.swiglu_8bit(x).sum(), x, create_graph=True)
