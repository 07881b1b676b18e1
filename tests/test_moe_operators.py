"""Router, grouped products, expert feed-forward and 8-bit checkpoints on the CPU path: the plain statements against loops in 64
bits and against differences, the layer that uses them, and what the entry points refuse."""

import math

import pytest
import torch

from tests.dist_utils import run_distributed
from torchure_b200.ops import act8, moe, oracle

NINF = float("-inf")


def plain_route(logits, k, capacity):
    """(experts, slots, offsets, rows, counts) by loops over Python numbers."""
    T, E = len(logits), len(logits[0])
    experts, per = [], [[] for _ in range(E)]
    for t, row in enumerate(logits):
        order = sorted(range(E), key=lambda e: (-row[e], e))[:k]
        experts.append(order)
        for j, e in enumerate(order):
            if row[e] != NINF:
                per[e].append(t * k + j)
    slots, offsets, rows = [[-1] * k for _ in range(T)], [0], []
    for e in range(E):
        for i in (per[e][:capacity] if capacity else per[e]):
            slots[i // k][i % k] = len(rows)
            rows.append(i)
        offsets.append(len(rows))
    return experts, slots, offsets, rows + [-1] * (T * k - len(rows)), [len(p) for p in per]


@pytest.mark.parametrize("T,E,k,capacity", [(1, 1, 1, 0), (1, 8, 2, 0), (9, 3, 3, 0), (17, 5, 2, 4), (40, 12, 4, 1), (0, 4, 2, 0)])
def test_route_against_loops(T, E, k, capacity):
    g = torch.Generator().manual_seed(T * 31 + E)
    logits = torch.randint(-3, 4, (T, E), generator=g).double()            # many ties
    if T > 8:
        logits[2] = NINF
        logits[5, 1:] = NINF
        logits[7, 0] = NINF
    r = moe.route(logits, k, capacity)
    if T:
        experts, slots, offsets, rows, counts = plain_route(logits.tolist(), k, capacity)
        assert r.experts.tolist() == experts and r.slots.tolist() == slots and r.rows.tolist() == rows
        assert r.offsets.tolist() == offsets and r.counts.tolist() == counts
        for t in range(T):
            e = [math.exp(logits[t, i]) for i in experts[t]]
            want = [v / sum(e) if sum(e) else 0.0 for v in e]
            assert torch.allclose(r.weights[t], torch.tensor(want, dtype=torch.float64), rtol=1e-12, atol=0)
    else:
        assert r.offsets.tolist() == [0] * (E + 1) and r.aux_loss.item() == 0


def test_route_gradient_by_differences():
    logits = torch.randn(7, 5, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    logits[3, 2] = -40.0
    logits.requires_grad_()

    def f(x):
        r = moe.route(x, 2)
        return r.weights, r.aux_loss

    assert torch.autograd.gradcheck(f, (logits,), eps=1e-6, atol=1e-7)


def test_closed_rows_have_no_gradient():
    logits = torch.randn(4, 6, generator=torch.Generator().manual_seed(1))
    logits[1] = NINF
    logits[2, 3:] = NINF
    logits.requires_grad_()
    r = moe.route(logits, 4)
    assert r.weights[1].tolist() == [0.0] * 4 and r.slots[1].tolist() == [-1] * 4 and r.slots[2, 3] == -1
    (r.weights.square().sum() + r.aux_loss).backward()
    assert torch.isfinite(logits.grad).all() and logits.grad[1].abs().sum() == 0


def test_expert_mlp_gradient_by_differences():
    g = torch.Generator().manual_seed(2)
    T, D, F, E, k = 6, 8, 16, 4, 2
    x, logits = (torch.randn(T, n, generator=g, dtype=torch.float64).requires_grad_() for n in (D, E))
    wgu = torch.randn(E, 2 * F, D, generator=g, dtype=torch.float64).requires_grad_()
    wd = torch.randn(E, D, F, generator=g, dtype=torch.float64).requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: moe.expert_mlp(*a, k, 3), (x, logits, wgu, wd), eps=1e-6, atol=1e-6)


def test_grouped_linear_rows_of_no_expert():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 4, generator=g).requires_grad_()
    w = torch.randn(3, 5, 4, generator=g).requires_grad_()
    y = moe.grouped_linear(x, w, torch.tensor([0, 2, 2, 7], dtype=torch.int32))
    torch.testing.assert_close(y[:2], x[:2] @ w[0].t())
    torch.testing.assert_close(y[2:7], x[2:7] @ w[2].t())
    assert y[7:].abs().sum() == 0
    y.sum().backward()
    assert w.grad[1].abs().sum() == 0 and x.grad[7:].abs().sum() == 0


def test_dispatch_and_combine_are_inverse():
    g = torch.Generator().manual_seed(4)
    r = moe.route(torch.randn(11, 5, generator=g), 3)
    x = torch.randn(11, 6, generator=g)
    torch.testing.assert_close(moe.combine(moe.dispatch(x, r), r), x)          # the weights of a token add up to 1


def quantized(x):
    """The values that 8 bits stand for, by loops in 64 bits; None for a block that is not finite."""
    out = []
    for row in x.double().tolist():
        done = []
        for lo in range(0, len(row), 64):
            b = row[lo:lo + 64]
            a = max(abs(v) for v in b)
            if not all(math.isfinite(v) for v in b):
                done += [None] * len(b)
            else:
                done += [math.copysign(math.floor(abs(v) * 127 / a + 0.5), v) * a / 127 if a else 0.0 for v in b]
        out.append(done)
    return out


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 63), (2, 64), (5, 200)])
def test_quantize8_against_loops(rows, cols):
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(rows, cols, generator=g).bfloat16()
    x[0, 0] = 2.0
    x[0, -1] = -1.0          # half the largest: a half-way case
    kept = act8.quantize8(x)
    assert kept.values.dtype == torch.int8 and kept.scales.shape == (rows, -(-cols // 64))
    got = oracle.dequantize8(*kept).double()
    torch.testing.assert_close(got, torch.tensor(quantized(x), dtype=torch.float64), rtol=2e-7, atol=0)


def test_quantize8_blocks_of_zeros_and_of_what_is_not_finite():
    x = torch.ones(2, 192, dtype=torch.bfloat16)
    x[0, :64] = 0.0
    x[1, 70] = float("nan")
    x[1, 130] = float("inf")
    got = act8.dequantize8(act8.quantize8(x))
    assert got[0, :64].abs().sum() == 0 and (got[0, 64:] == 1).all() and (got[1, :64] == 1).all()
    assert torch.isnan(got[1, 64:]).all()


def test_swiglu_8bit_takes_its_gradient_at_the_kept_values():
    g = torch.Generator().manual_seed(5)
    gu = torch.randn(3, 140, generator=g).bfloat16()
    leaf = gu.clone().requires_grad_()
    act = act8.swiglu_8bit(leaf)
    act.backward(torch.ones_like(act))
    kept = torch.tensor([a + b for a, b in zip(quantized(gu[:, :70]), quantized(gu[:, 70:]))], dtype=torch.float64).requires_grad_()
    oracle.swiglu_plain(kept).sum().backward()
    assert (leaf.grad.double() - kept.grad).norm() < 2 ** -7 * kept.grad.norm()          # a few bf16 roundings


@pytest.mark.parametrize("factor,bits", [(0.0, 16), (1.0, 16), (8.0, 8)])
def test_grouped_layer_equals_the_padded_one(factor, bits):
    """Same choices, same drops, same loss and gradients in fp32 (8 bits: gate and up off by 1 / 254 of a block's largest)."""
    from torchure_b200.parallel.expert_parallel import MoELayer

    torch.manual_seed(0)
    old = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=factor or 8.0)
    new = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=factor, experts="grouped", act_bits=bits)
    new.load_state_dict(old.state_dict())
    x = torch.randn(3, 7, 16)
    grads = []
    for layer in (old, new):
        xi = x.clone().requires_grad_()
        out = layer(xi)
        (out.square().sum() + layer.aux_loss).backward()
        grads.append([out.detach(), xi.grad, *(p.grad for p in layer.parameters())])
    for a, b in zip(*grads):
        assert (a - b).norm() <= (1e-5 if bits == 16 else 1e-2) * a.norm()


def test_grouped_model_trains_on_cpu():
    from torchure_b200.models import build_model
    from torchure_b200.objectives import ARObjective

    cfg = dict(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=32, head_dim=8, vocab_size=64, num_experts=4, top_k=2,
               moe_ffn_dim=32, capacity_factor=1.25)
    ids = torch.randint(0, 64, (2, 16), generator=torch.Generator().manual_seed(0))
    losses = []
    for kind in ("capacity", "grouped"):
        torch.manual_seed(0)
        model = build_model("qwen3_moe", dict(cfg, experts=kind))
        model.init_weights()
        loss = ARObjective(fused_linear_ce=True, ce_chunk_size=16).compute_loss(model, {"input_ids": ids, "labels": ids})
        loss.backward()
        losses.append(loss.item())
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert abs(losses[0] - losses[1]) < 1e-5


def test_refusals():
    x, w = torch.randn(4, 8), torch.randn(3, 6, 8)
    r = moe.route(torch.randn(4, 3), 2)
    with pytest.raises(ValueError, match="top_k"):
        moe.route(torch.randn(4, 3), 4)
    with pytest.raises(ValueError, match="top_k"):
        moe.route(torch.randn(4, 3), 0)
    with pytest.raises(ValueError, match="capacity"):
        moe.route(torch.randn(4, 3), 1, -1)
    with pytest.raises(ValueError, match="logits"):
        moe.route(torch.randn(3), 1)
    with pytest.raises(ValueError, match="logits"):
        moe.route(torch.ones(3, 3, dtype=torch.int64), 1)
    with pytest.raises(ValueError, match="do not fit"):
        moe.grouped_linear(x, torch.randn(3, 6, 7), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="offsets"):
        moe.grouped_linear(x, w, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="routed"):
        moe.dispatch(torch.randn(5, 8), r)
    with pytest.raises(ValueError, match="rows expected"):
        moe.combine(torch.randn(7, 8), r)
    wgu, wd = torch.randn(3, 12, 8), torch.randn(3, 8, 6)
    with pytest.raises(ValueError, match="bits"):
        moe.expert_mlp(x, torch.randn(4, 3), wgu, wd, 2, act_bits=4)
    with pytest.raises(ValueError, match="do not fit"):
        moe.expert_mlp(x, torch.randn(4, 2), wgu, wd, 2)
    with pytest.raises(ValueError, match="differ"):
        moe.expert_mlp(x, torch.randn(4, 3), (wgu, wgu[:, :6]), wd, 2)
    with pytest.raises(TypeError, match="bf16"):
        act8.quantize8(torch.randn(4, 8))
    with pytest.raises(ValueError, match="matrix"):
        act8.quantize8(torch.randn(8).bfloat16())
    with pytest.raises(ValueError, match="gate and up"):
        act8.swiglu_8bit(torch.randn(4, 7).bfloat16())
    from torchure_b200.parallel.expert_parallel import MoELayer

    with pytest.raises(ValueError, match="grouped"):
        MoELayer(8, 8, 2, experts="dense")
    with pytest.raises(ValueError, match="grouped experts"):
        MoELayer(8, 8, 2, act_bits=8)


def _spread(rank, world):
    from torchure_b200.core.mesh import Mesh
    from torchure_b200.parallel.expert_parallel import MoELayer

    mesh = Mesh({"ep": world})
    torch.manual_seed(0)
    full = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=8.0, experts="grouped")
    spread = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=8.0, experts="grouped")
    spread.load_state_dict(full.state_dict())
    spread.shard_(mesh, "ep")
    x = torch.randn(6, 16, generator=torch.Generator().manual_seed(rank))
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    out, want = spread(a), full(b)
    torch.testing.assert_close(out, want, rtol=1e-4, atol=1e-5)
    out.square().sum().backward()
    want.square().sum().backward()
    torch.testing.assert_close(a.grad, b.grad, rtol=1e-4, atol=1e-5)
    # this rank's experts saw the tokens of all ranks
    grads = [torch.zeros_like(full.w_down) for _ in range(world)]
    torch.distributed.all_gather(grads, full.w_down.grad)
    torch.testing.assert_close(spread.w_down.grad, sum(grads)[rank * 2:rank * 2 + 2], rtol=1e-4, atol=1e-5)


def test_grouped_layer_spread_over_ranks():
    run_distributed(_spread, 2, timeout_s=120)
