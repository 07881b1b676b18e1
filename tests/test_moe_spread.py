"""The grouped mixture layer spread over ranks (CPU, gloo): settings under which it has to equal the layer in one piece.

Tolerance: both sides compute in fp32 and differ in the order of sums of at most 128 terms; 2^-24 for each addition and a dozen operations in
a row stay below 2^-16 of the tensor's 2-norm."""

import pytest
import torch

from tests.dist_utils import run_distributed


def _same(got, want):
    assert (got.detach() - want.detach()).norm() <= 2.0 ** -16 * want.detach().norm()


def _against_one_piece(rank, world, favourite, **kw):
    from torchure_b200.core.mesh import Mesh
    from torchure_b200.parallel.expert_parallel import MoELayer

    torch.manual_seed(0)
    full, spread = (MoELayer(16, 32, num_experts=4, top_k=2, experts="grouped", **kw) for _ in range(2))
    with torch.no_grad():
        for w in (full.w_gate, full.w_up, full.w_down):
            w.mul_(10 * 64).round_().div_(64)      # gate and up come out exact in any order of the sums, and so do their 8 bits
        if favourite:      # every token prefers one expert
            full.router.weight[:, 0] = torch.tensor([0.0, 9.0, 0.0, 0.0])
    spread.load_state_dict(full.state_dict())
    spread.shard_(Mesh({"ep": world}), "ep")
    x = torch.randn(64, 16, generator=torch.Generator().manual_seed(rank)).mul(16).round().div(16)
    if favourite:
        x[:, 0] = 1.0
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    out, want = spread(a), full(b)
    assert not (want == 0).all(1).any()
    _same(out, want)
    out.square().sum().backward()
    want.square().sum().backward()
    _same(a.grad, b.grad)
    for name in ("w_gate", "w_up", "w_down"):      # this rank's experts saw the tokens of all ranks
        grads = [torch.zeros_like(getattr(full, name)) for _ in range(world)]
        torch.distributed.all_gather(grads, getattr(full, name).grad)
        _same(getattr(spread, name).grad, sum(grads)[rank * 2:rank * 2 + 2])


@pytest.mark.parametrize("favourite", [False, True])
def test_capacity_factor_0_drops_nothing(favourite):
    run_distributed(_without_limit, 2, favourite, timeout_s=120)


def _without_limit(rank, world, favourite):
    _against_one_piece(rank, world, favourite, capacity_factor=0.0)


def test_8_bit_checkpoints_are_taken():
    run_distributed(_in_8_bits, 2, timeout_s=120)


def _in_8_bits(rank, world):
    _against_one_piece(rank, world, False, capacity_factor=8.0, act_bits=8)
