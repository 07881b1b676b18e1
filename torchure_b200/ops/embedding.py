"""Token embedding: rows of a table by id, scaled, and the table's gradient by sorted tokens.

The gradient is dense, [V, D] in the table's type: every row the sum over its tokens in fp32, in an order that does not depend on what else
runs, and rounded once.  However often a token occurs, many SMs share its sum.

On tensors that are not on a GPU the plain statement of ``ops/oracle.py`` runs.
"""

from __future__ import annotations

import torch

from torchure_b200 import ops
from torchure_b200.ops import debug, oracle
from torchure_b200.ops.kernels import _C


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale * table[ids], [..., D] in ``out_dtype`` (bf16 or fp32; None: the table's).

    ids int64 or int32 of any shape, table [V, D] bf16 or fp32 (rows with any stride).  ``padding_idx``: a row that gets no gradient.  On a GPU
    an id outside the table gives a row of NaN and no gradient (on the CPU an IndexError)."""
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.bfloat16, torch.float32) and (table.is_cuda or out_dtype != torch.float64):
        raise TypeError(f"embedding: rows in bf16 or fp32, not {out_dtype}")
    if ops.available() and (table.is_cuda or ids.is_cuda):
        return _C().embedding(ids, table, scale, padding_idx, out_dtype == torch.bfloat16, debug.enabled())
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding: ids in int64 or int32 expected, got {ids.dtype}")
    if table.dim() != 2 or table.shape[0] < 1:
        raise ValueError(f"embedding: a table [rows, width] expected, got {tuple(table.shape)}")
    if padding_idx is not None and not -table.shape[0] <= padding_idx < table.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} in a table of {table.shape[0]} rows")
    if not abs(scale) < float("inf"):
        raise ValueError(f"embedding: scale {scale}")
    return oracle.embedding(ids, table, scale, padding_idx, out_dtype)
