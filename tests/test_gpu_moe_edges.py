"""Mixture-of-experts operators and 8-bit checkpoints on a GPU, at the edges: what is empty, refused, switched off or changed in place, and
gradients against differences along directions in which they are large.

Tolerances: U = 2^-8 and RMS = 2^-9 are the most and the 2-norm's share of a rounding to bf16, 2^-20 the router's fp32 arithmetic."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from torchure_b200 import ops
from torchure_b200.ops import act8, debug, kernels, moe, oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
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
