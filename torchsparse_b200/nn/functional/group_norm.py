from typing import NamedTuple, Optional

import torch

from ... import _ops
from ...tensor import SparseTensor

__all__ = ["RowGroups", "group_rows", "sample_rows", "group_norm"]


class RowGroups(NamedTuple):
    """Rows grouped by an index (both int32): ``order`` [N] the row at each grouped position, ``offsets`` [groups + 1]
    the first position of each group.  Rows of no group stand behind ``offsets[-1]``."""

    order: torch.Tensor
    offsets: torch.Tensor


def group_rows(keys: torch.Tensor, num_groups: int) -> RowGroups:
    """Group rows by ``keys`` (int32 or int64 [N]); rows of one group keep their order, a key outside
    [0, num_groups) belongs to no group."""
    return RowGroups(*_ops.group_rows(keys, num_groups))


def sample_rows(input: SparseTensor, batch_size: Optional[int] = None) -> RowGroups:
    """The rows of a tensor grouped by batch sample.  Without ``batch_size`` the largest batch index is read from the
    device.  The result serves every layer on the same coordinates."""
    batch = input.coords[:, 0].to(input.feats.device)
    if batch.dtype not in (torch.int32, torch.int64):
        batch = batch.long()
    if batch_size is None:
        batch_size = int(batch.max().item()) + 1 if batch.numel() else 0
    return group_rows(batch, max(int(batch_size), 1))


_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "leaky_relu": 2, "silu": 3}


def activation_code(activation: Optional[str]) -> int:
    """The library's number of an activation that a norm can be fused with."""
    try:
        return _ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(k for k in _ACTIVATIONS if k)}") from None


def group_norm(feats: torch.Tensor, offsets: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: Optional[str] = None,
               negative_slope: float = 0.01, order: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(group_norm(feats))`` over the rows of each sample, features [N, C] (fp32, fp16 or bf16).

    ``offsets`` int32 [samples + 1], ascending: sample s is rows ``offsets[s]`` to ``offsets[s + 1]``, or, with
    ``order`` int32 [N], a permutation, the rows ``order[offsets[s] : offsets[s + 1]]`` (see ``group_rows``).  A sample may be empty;
    rows of no sample become zero.  A group with one value becomes ``act(bias)``.  ``weight`` and ``bias`` [C] may have a
    dtype of their own (fp32 beside 16-bit features).  ``activation``: None, "relu", "leaky_relu" or "silu".
    Statistics and sums are fp32 and run in a fixed order.  Differentiable as often as wanted, in forward mode and under
    ``torch.func`` too; beyond the plain gradient it is then composed of slower operations."""
    return _ops.group_norm(feats, weight, bias, offsets, order, num_groups, eps, activation_code(activation), negative_slope)
