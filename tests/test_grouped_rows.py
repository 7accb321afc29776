"""The operators over grouped rows without a GPU: argument checks of the C entries, refusals of CPU tensors, and what
the modules do on the CPU."""
import numpy as np
import pytest
import torch


def test_c_entries_refuse_bad_arguments_before_any_cuda_call():
    from torchsparse_b200._lib import lib

    x = 256      # an address that is never read: every call below is refused before a launch
    assert lib.tsb_group_rows(None, 0, 1, 5, 2, None, None, x, None, 0, None) == 1
    assert lib.tsb_group_rows(x, 0, 1, 5, 0, x, None, x, x, 1 << 20, None) == 1
    assert lib.tsb_group_rows(x, 0, -1, 5, 2, x, None, x, x, 1 << 20, None) == 1
    assert lib.tsb_group_rows(x, 0, 1, 1 << 31, 2, x, None, x, x, 1 << 20, None) == 5
    assert lib.tsb_group_rows(x, 0, 1, 5, 600, x, None, x, x, 0, None) == 3
    norm = lambda n=100_000, c=8, g=2, b=1, act=0, dtype=0, p=0, ws=1 << 26: lib.tsb_group_norm_fwd(      # noqa: E731
        x, None, x, None, None, n, c, g, b, 1e-5, act, 0.1, dtype, p, x, x, x, x, ws, None)
    assert [norm(n=-1), norm(c=0), norm(g=3), norm(g=0), norm(b=-1), norm(act=4)] == [1] * 6
    assert [norm(dtype=3), norm(p=9)] == [2, 2] and norm(ws=0) == 3
    assert [norm(n=1 << 31), norm(c=1 << 17)] == [5, 5]
    grad = lambda n=100_000, c=8, g=2, ws=1 << 26, dx=x: lib.tsb_group_norm_bwd(      # noqa: E731
        x, x, None, x, None, None, x, x, n, c, g, 1, 0, 0.1, 0, 0, dx, None, None, x, ws, None)
    assert [grad(g=3), grad(n=-1), grad(dx=None), grad(ws=0)] == [1, 1, 1, 3]
    assert lib.tsb_embedding_fwd(None, x, 0, 5, 3, 8, 1.0, 0, x, None) == 1
    assert lib.tsb_embedding_fwd(x, x, 0, 5, 3, 0, 1.0, 0, x, None) == 1
    assert lib.tsb_embedding_fwd(x, x, 0, 5, 3, 8, 1.0, 7, x, None) == 2
    assert lib.tsb_embedding_fwd(x, x, 0, 0, 3, 8, 1.0, 0, None, None) == 0
    assert lib.tsb_embedding_bwd(x, x, 0, 5, 3, 8, 1.0, -1, 0, None, x, 1 << 20, None) == 1
    assert lib.tsb_embedding_bwd(x, x, 0, 5, 3, 8, 1.0, -1, 0, x, x, 16, None) == 3
    assert lib.tsb_embedding_bwd(x, x, 0, 1 << 31, 3, 8, 1.0, -1, 0, x, x, 16, None) == 5
    assert lib.tsb_expert_dispatch(x, None, x, 5, 2, 8, 0, x, None) == 1
    assert lib.tsb_expert_dispatch(x, x, x, 5, 0, 8, 0, x, None) == 1
    assert lib.tsb_expert_dispatch(x, x, x, 1 << 30, 2, 8, 0, x, None) == 5
    assert lib.tsb_expert_combine(x, x, 5, x, x, 5, 2, 8, 0, x, None) == 2
    assert lib.tsb_expert_combine(None, x, 0, x, x, 5, 2, 8, 0, x, None) == 1
    assert lib.tsb_expert_combine_bwd(x, x, x, 0, x, x, 5, 2, 8, 0, x, None, None) == 1
    assert lib.tsb_expert_combine_bwd(None, None, None, 0, None, None, 0, 2, 8, 0, None, None, None) == 0


def test_workspaces_grow_with_the_sizes():
    from torchsparse_b200._lib import lib

    assert lib.tsb_group_rows_workspace_bytes(1_000_000, 300) >= 5 * 4_000_000
    assert lib.tsb_group_norm_fwd_workspace_bytes(1_000_000, 64, 8, 10_000, 0) >= 10_000 * 8 * 8
    assert lib.tsb_group_norm_bwd_workspace_bytes(1_000_000, 64, 8, 10_000, 0) >= 2 * 10_000 * 64 * 8
    assert lib.tsb_group_norm_fwd_workspace_bytes(1000, 64, 8, 1, 0) == 0      # one block per sample and group
    assert lib.tsb_embedding_bwd_workspace_bytes(100_000, 50, 64, 1) > lib.tsb_embedding_bwd_workspace_bytes(1000, 50, 64, 1)


def test_cpu_tensors_are_refused():
    from torchsparse_b200.nn import functional as F

    x, idx = torch.randn(4, 8), torch.zeros(4, dtype=torch.int32)
    rows = F.ExpertRows(idx, idx[:, None], idx[:2])
    for call in (lambda: F.group_rows(idx, 2), lambda: F.group_norm(x, idx[:2], 2), lambda: F.embedding(idx, x),
                 lambda: F.expert_sort(idx, 2), lambda: F.expert_dispatch(x, rows), lambda: F.expert_combine(x, x[:, :1], rows)):
        with pytest.raises(RuntimeError, match="CUDA tensors required"):
            call()


@pytest.mark.parametrize("activation", [None, "relu", "leaky_relu", "silu"])
def test_group_norm_module_on_the_cpu_normalises_sample_by_sample(activation):
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    g = torch.Generator().manual_seed(0)
    coords = torch.randint(0, 9, (200, 4), generator=g).int()
    coords[:, 0] = torch.randint(0, 3, (200,), generator=g)
    x = ts.SparseTensor(torch.randn(200, 12, generator=g, dtype=torch.float64), coords)
    m = spnn.GroupNorm(3, 12, activation=activation, negative_slope=0.2).double()
    y = m(x)
    fn = {None: lambda t: t, "relu": torch.relu, "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, 0.2),
          "silu": torch.nn.functional.silu}[activation]
    for s in range(3):
        rows = coords[:, 0] == s
        want = fn(torch.nn.functional.group_norm(x.feats[rows].t()[None], 3, m.weight, m.bias, m.eps))
        assert torch.allclose(y.feats[rows], want[0].t(), atol=1e-12)
    assert y.coords is x.coords and y._caches is x._caches
    with pytest.raises(ValueError):
        spnn.GroupNorm(3, 15)(x)
    with pytest.raises(ValueError):
        spnn.GroupNorm(3, 12, activation="tanh")


def test_embedding_module_refuses_features_that_are_no_labels():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    m = spnn.Embedding(5, 4, padding_idx=0, scale=2.0)
    assert m.weight.shape == (5, 4) and bool((m.weight[0] == 0).all()) and "scale=2.0" in repr(m)
    with pytest.raises(ValueError):
        m(ts.SparseTensor(torch.zeros(6, 2, dtype=torch.int64), torch.zeros(6, 4, dtype=torch.int32)))
