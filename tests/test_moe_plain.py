"""The plain path of the mixture-of-experts operators takes the arguments that the kernels take."""

import pytest
import torch

from torchure_b200.ops import moe


@pytest.mark.parametrize("have", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("want", [None, torch.bfloat16, torch.float32])
def test_combine_gives_the_type_that_was_asked_for(have, want):
    g = torch.Generator().manual_seed(0)
    r = moe.route(torch.randn(9, 4, generator=g), 2)
    y = torch.randn(18, 6, generator=g).to(have)
    out = moe.combine(y, r) if want is None else moe.combine(y, r, want)
    assert out.dtype == (want or have)
    exact = (r.weights.double()[:, :, None] * y.double()[r.slots.long()]).sum(1)
    # terms and sum of two of them, each rounded to the narrower type: 2^-8 (bf16) or 2^-23 of the terms' magnitudes
    size = (r.weights.double()[:, :, None] * y.double()[r.slots.long()].abs()).sum(1)
    unit = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -23
    assert ((out.double() - exact).abs() <= 4 * unit * size).all()


@pytest.mark.parametrize("edges,meant", [([0, 60, 20, 100], [0, 60, 60, 100]), ([0, -5, 50, 4000], [0, 0, 50, 100]), ([9, 30, 40, 90], [0, 30, 40, 90])])
def test_wrong_offsets_count_as_on_the_gpu(edges, meant):
    """Offsets that fall, are negative or pass the end: the largest so far, within the rows, from 0 on."""
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(100, 6, generator=g), torch.randn(3, 5, 6, generator=g)
    got, want = (moe.grouped_linear(x, w, torch.tensor(e, dtype=torch.int32)) for e in (edges, meant))
    assert got.shape == (100, 5) and torch.equal(got, want)


@pytest.mark.parametrize("rows,matrices", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("pair", [False, True])
def test_rows_and_matrices_of_two_types(rows, matrices, pair):
    """As on a GPU: bf16 rows of a model whose parameters are fp32, and the other way round; gradients have their tensors' types."""
    g = torch.Generator().manual_seed(3)
    x, logits = torch.randn(20, 16, generator=g).to(rows).requires_grad_(), torch.randn(20, 4, generator=g).requires_grad_()
    gate, up = (torch.randn(4, 24, 16, generator=g).mul(0.25).to(matrices).requires_grad_() for _ in range(2))
    down = torch.randn(4, 16, 24, generator=g).mul(0.2).to(matrices).requires_grad_()
    first = (gate, up) if pair else torch.cat([gate, up], 1)
    out, aux = moe.expert_mlp(x, logits, first, down, 2)
    assert out.dtype == rows and aux.dtype == torch.float32
    (out.float().sum() + aux).backward()
    assert all(t.grad is not None and t.grad.dtype == t.dtype for t in (x, logits, gate, up, down))
    exact, _ = moe.expert_mlp(x.detach().double(), logits.detach().double(), torch.cat([gate, up], 1).detach().double(), down.detach().double(), 2)
    # at most six roundings to bf16 in a row (matrices, gate / up, activation, product, weighted row, sum): 6 2^-9 in the 2-norm
    assert (out.detach().double() - exact).norm() <= 6 * 2.0 ** -9 * exact.norm()
    if rows == torch.bfloat16:
        y = moe.grouped_linear(x, gate, torch.tensor([0, 3, 3, 9, 20], dtype=torch.int32))
        assert y.dtype == rows and torch.autograd.grad(y.float().sum(), gate)[0].dtype == matrices
