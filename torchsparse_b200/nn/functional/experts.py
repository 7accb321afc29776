from typing import NamedTuple

import torch

from ... import _ops

__all__ = ["ExpertRows", "expert_sort", "expert_dispatch", "expert_combine"]


class ExpertRows(NamedTuple):
    """The N * k choices of N rows sorted by expert (all int32): ``order`` [N * k] the choice at each sorted position,
    ``inverse`` [N, k] the position of each choice, ``offsets`` [experts + 1] the first position of each expert.
    Choices without an expert stand behind ``offsets[-1]``."""

    order: torch.Tensor
    inverse: torch.Tensor
    offsets: torch.Tensor


def expert_sort(experts: torch.Tensor, num_experts: int) -> ExpertRows:
    """Sort the choices of a router: ``experts`` int32 or int64 [N, k] (or [N]) names the weight matrices that row i is
    sent to.  Choices of one expert keep their order; a choice outside [0, num_experts) (-1, say, for one dropped for
    want of room) goes to no expert."""
    return ExpertRows(*_ops.expert_sort(experts, num_experts))


def expert_dispatch(feats: torch.Tensor, rows: ExpertRows) -> torch.Tensor:
    """[N * k, C]: the rows of ``feats`` sorted by expert, those of expert e at positions ``offsets[e]`` to
    ``offsets[e + 1]``; zeros behind the last expert.  The gradient adds up a row's k copies in their order."""
    return _ops.expert_dispatch(feats, rows.inverse, rows.offsets)


def expert_combine(feats: torch.Tensor, weights: torch.Tensor, rows: ExpertRows) -> torch.Tensor:
    """[N, C]: row i is the sum over its choices of ``weights[i, j]`` times the sorted row of that choice (``feats``
    [N * k, C], what the experts made of the dispatched rows); a choice without an expert adds nothing.  Products and
    sums are fp32.  ``weights`` fp32, fp16 or bf16 [N, k].  The gradients of this and of ``expert_dispatch`` cannot be
    differentiated again."""
    return _ops.expert_combine(feats, weights, rows.inverse, rows.offsets)
