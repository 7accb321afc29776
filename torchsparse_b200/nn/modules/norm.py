from typing import Optional

import torch
from torch import nn

from ...tensor import SparseTensor
from .. import functional as F
from ..functional.group_norm import activation_code
from ..utils import fapply

__all__ = ["BatchNorm", "GroupNorm", "InstanceNorm"]

_KERNEL_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class BatchNorm(nn.BatchNorm1d):
    """BatchNorm1d over the feature matrix (torchsparse/nn/modules/norm.py:15-17)."""

    def forward(self, input: SparseTensor) -> SparseTensor:
        return fapply(input, super().forward)


class InstanceNorm(nn.InstanceNorm1d):
    def forward(self, input: SparseTensor) -> SparseTensor:
        return fapply(input, super().forward)


class GroupNorm(nn.GroupNorm):
    """Group normalisation per batch sample (torchsparse/nn/modules/norm.py:25-57): the rows of every sample are
    normalised on their own, as ``nn.GroupNorm`` does for one [1, C, rows] input.

    ``activation`` ("relu", "leaky_relu", "silu") is applied in the same kernel.  ``forward`` takes the rows grouped by
    sample (``F.sample_rows``) when the caller has them; else it groups them and reads the batch size from the device.
    As in ``nn.GroupNorm`` a group of one value is then a ValueError; with ``rows`` it becomes ``act(bias)``.
    fp32, fp16 and bf16 features on a GPU run on the library's kernels, with parameters of the same or another of these
    dtypes; other features run through torch, sample by sample."""

    activation: Optional[str] = None      # also of modules that were pickled without one
    negative_slope = 0.01

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, device=None, dtype=None,
                 *, activation: Optional[str] = None, negative_slope: float = 0.01) -> None:
        super().__init__(num_groups, num_channels, eps, affine, device, dtype)
        activation_code(activation)      # refuses an unknown one
        self.activation, self.negative_slope = activation, negative_slope

    def forward(self, input: SparseTensor, rows: Optional[F.RowGroups] = None) -> SparseTensor:
        feats = input.feats
        if feats.shape[1] != self.num_channels:
            raise ValueError(f"expected {self.num_channels} channels, got {feats.shape[1]}")
        if feats.is_cuda and feats.dtype in _KERNEL_DTYPES:
            if rows is None:
                rows = F.sample_rows(input)
                if self.num_groups == self.num_channels and bool((rows.offsets.diff() == 1).any()):
                    raise ValueError("Expected more than 1 value per channel: a sample of one row in groups of one channel")
            nfeats = F.group_norm(feats, rows.offsets, self.num_groups, self.weight, self.bias, self.eps, self.activation,
                                  self.negative_slope, rows.order)
        else:
            nfeats = self._by_sample(input)
        return SparseTensor._from_parts(nfeats, input.coords, input.stride, input.spatial_range, input._caches)

    def _by_sample(self, input: SparseTensor) -> torch.Tensor:
        coords, feats = input.coords, input.feats
        batch_size = int(torch.max(coords[:, 0]).item()) + 1 if coords.shape[0] else 0
        num_channels = feats.shape[1]
        nfeats = torch.zeros_like(feats)
        for k in range(batch_size):
            rows = coords[:, 0] == k
            sample = feats[rows].transpose(0, 1).reshape(1, num_channels, -1)
            sample = super().forward(sample)
            if self.activation == "relu":
                sample = nn.functional.relu(sample)
            elif self.activation == "leaky_relu":
                sample = nn.functional.leaky_relu(sample, self.negative_slope)
            elif self.activation == "silu":
                sample = nn.functional.silu(sample)
            nfeats[rows] = sample.reshape(num_channels, -1).transpose(0, 1)
        return nfeats

    def extra_repr(self) -> str:
        more = f", activation={self.activation}" if self.activation else ""
        return super().extra_repr() + more
