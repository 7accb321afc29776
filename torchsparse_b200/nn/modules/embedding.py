"""Learnt vectors for categorical voxel features."""
from typing import Optional, Union

import torch
from torch import nn

from ...tensor import SparseTensor
from .. import functional as F
from ..utils import fapply

__all__ = ["Embedding"]


class Embedding(nn.Embedding):
    """``scale * weight[label]`` for the integer label of every voxel: ``forward`` takes a SparseTensor whose features
    are labels [N] or [N, 1] (int32 or int64) and keeps its coordinates, or a plain tensor of labels.  A label that is no
    row of the table gives zeros.  Constructor arguments are those of ``nn.Embedding`` that name the table, and
    ``scale``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, scale: float = 1.0,
                 device=None, dtype=None) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: Optional[int] = None, *,
                        scale: float = 1.0) -> "Embedding":
        """A layer on the rows of ``embeddings`` [rows, C], which it shares; not trained where ``freeze`` is set."""
        if embeddings.dim() != 2:
            raise ValueError(f"from_pretrained expects a table [rows, channels], not {tuple(embeddings.shape)}")
        layer = cls(*embeddings.shape, padding_idx, scale, device="meta", dtype=embeddings.dtype)
        layer.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return layer

    def forward(self, input: Union[SparseTensor, torch.Tensor]) -> Union[SparseTensor, torch.Tensor]:
        if isinstance(input, SparseTensor):
            return fapply(input, self._labels)
        return F.embedding(input, self.weight, self.scale, self.padding_idx)

    def _labels(self, feats: torch.Tensor) -> torch.Tensor:
        if feats.dim() == 2 and feats.shape[1] == 1:
            feats = feats[:, 0]
        if feats.dim() != 1:
            raise ValueError(f"Embedding expects one label per voxel, not features {tuple(feats.shape)}")
        return F.embedding(feats, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")
