from typing import Optional

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ... import backend

__all__ = ["embedding"]


class _Embedding(Function):
    """Lookup of table rows and the gradient of the table, summed token by token in a fixed order."""

    @staticmethod
    def forward(ctx, table: torch.Tensor, indices: torch.Tensor, scale: float, padding_idx: Optional[int]) -> torch.Tensor:
        ctx.save_for_backward(indices)
        ctx.args = table.shape[0], scale, padding_idx
        return backend.embedding_forward_cuda(indices, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output: torch.Tensor):
        (indices,) = ctx.saved_tensors
        num_rows, scale, padding_idx = ctx.args
        return backend.embedding_backward_cuda(grad_output, indices, num_rows, scale, padding_idx), None, None, None


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[indices]``: a learnt vector for the label of every voxel or point.

    ``indices`` int32 or int64 of any shape, ``table`` [rows, C] (fp32, fp16 or bf16); the result has the table's dtype
    and the shape of ``indices`` with C behind it.  An index that is no row of the table (a negative one, say) gives
    zeros and no gradient.  ``padding_idx`` names a row that gets no gradient (negative: counted from the end).
    The gradient is accumulated in fp32 in the order of the indices and rounded once: the same call gives the same
    bits."""
    if padding_idx is not None:
        if not -table.shape[0] <= padding_idx < table.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is no row of a table of {table.shape[0]}")
        padding_idx = padding_idx % table.shape[0]
    flat = indices if indices.dim() == 1 else indices.reshape(-1)
    if torch.is_grad_enabled() and table.requires_grad:
        out = _Embedding.apply(table, flat, scale, padding_idx)
    else:
        out = backend.embedding_forward_cuda(flat, table, scale)
    return out if indices.dim() == 1 else out.view(*indices.shape, table.shape[1])
