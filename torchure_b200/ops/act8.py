"""Activation checkpoints in 8 bits: what a backward pass needs of an activation, at half the bytes of bf16.

``quantize8`` keeps a bf16 matrix as int8 values and one fp32 scale for every 64 values of a row; ``dequantize8`` reads it back;
``swiglu_8bit`` is SwiGLU whose backward pass reads gate and up from such a checkpoint, written by the forward pass as it goes.

With a the largest magnitude of a block: q = sign(x) floor(127 |x| / a + 1/2), scale = a / 127.  The value kept is off by at most
a / 254.  A block of zeros reads back as zeros; a block that holds a NaN or an infinity reads back as NaN, all of it.

On tensors that are not on a GPU the plain statements of ``ops/oracle.py`` run.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from torchure_b200 import ops
from torchure_b200.ops import debug, oracle
from torchure_b200.ops.kernels import _C

BLOCK = oracle.ACT8_BLOCK


class Act8(NamedTuple):
    """A matrix in 8 bits: ``values`` int8 [rows, columns], ``scales`` fp32 [rows, ceil(columns / 64)]."""

    values: torch.Tensor
    scales: torch.Tensor


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """``x`` as a matrix of contiguous rows."""
    if x.dim() < 1:
        raise ValueError(f"{what}: a tensor of at least one dimension expected")
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{what}: bf16 expected, got {x.dtype}")
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def quantize8(x: torch.Tensor) -> Act8:
    """A bf16 matrix [rows, columns] (any row stride) in 8 bits."""
    if ops.available() and x.is_cuda:
        return Act8(*_C().quantize8(x))
    if x.dim() != 2:
        raise ValueError(f"quantize8: a matrix expected, got {x.dim()} dimensions")
    return Act8(*oracle.quantize8(_rows(x.detach(), "quantize8")))


def dequantize8(kept: Act8) -> torch.Tensor:
    """bf16 [rows, columns] of what ``quantize8`` kept."""
    values, scales = kept
    if ops.available() and values.is_cuda:
        return _C().dequantize8(values, scales, debug.enabled())
    return oracle.dequantize8(values, scales).bfloat16()


def swiglu_8bit(gu: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up of ``gu`` [..., 2F] = gate | up (bf16), [..., F].  Until the backward pass ``gu`` is kept in 8 bits, gate and
    up in blocks of their own; the gradient is the formula's at the values read back.  Without gradients nothing is kept."""
    if ops.available() and gu.is_cuda:
        return _C().swiglu_8bit(gu, debug.enabled())
    if gu.dim() < 1 or gu.shape[-1] % 2:
        raise ValueError(f"swiglu_8bit: gate and up columns expected, got {tuple(gu.shape)}")
    act = oracle.swiglu_8bit(_rows(gu, "swiglu_8bit")).to(gu.dtype)
    return act.view(*gu.shape[:-1], gu.shape[-1] // 2)
