from typing import Optional

import torch

from ... import _ops

__all__ = ["embedding"]


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[indices]``: a learnt vector for the label of every voxel or point.

    ``indices`` int32 or int64 of any shape, ``table`` [rows, C] (fp32, fp16 or bf16); the result has the table's dtype
    and the shape of ``indices`` with C behind it.  An index that is no row of the table (a negative one, say) gives
    zeros and no gradient.  ``padding_idx`` names a row that gets no gradient (negative: counted from the end).
    The gradient is accumulated in fp32 in the order of the indices and rounded once: the same call gives the same
    bits.  It cannot be differentiated again."""
    if padding_idx is None:
        return _ops.embedding(table, indices, scale, -1)
    rows = table.shape[0]
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} is no row of a table of {rows}")
    return _ops.embedding(table, indices, scale, padding_idx % rows)
