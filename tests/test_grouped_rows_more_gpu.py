"""More of the operators over grouped rows on the GPU: cases that their first tests did not reach."""
import pytest
import torch

from test_grouped_rows_gpu import TYPES, U, affine, check_norm, features

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ group norm
@pytest.mark.parametrize("n", [900, 200_000])      # one block per sample and group, and chunks of rows
def test_an_empty_sample_without_eps_leaves_the_parameters_gradients(n):
    """An empty sample has no deviation: 1 / sqrt(0 + 0) must reach nothing."""
    from torchsparse_b200.nn import functional as F

    w, b = affine(24)
    x = features(n, 24, torch.float32)
    check_norm(x, [0, n // 3, n // 3, n], 3, w, b, "silu", eps=0.0)
    leaf = w.clone().requires_grad_()
    y = F.group_norm(x, ints([0, 0]), 3, leaf, b, eps=0.0)      # nothing but an empty sample
    assert bool((y == 0).all()) and bool((torch.autograd.grad(y.sum(), leaf)[0] == 0).all())
