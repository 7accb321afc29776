"""Modules and imports of the operators over grouped rows, without a GPU."""
import pytest
import torch


def test_embedding_from_a_pretrained_table():
    from torchsparse_b200 import nn as spnn

    table = torch.randn(6, 4)
    m = spnn.Embedding.from_pretrained(table, padding_idx=-1, scale=2.0)
    assert m.weight.data_ptr() == table.data_ptr() and not m.weight.requires_grad
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (6, 4, 5, 2.0)
    assert bool((table[5] != 0).all())                           # as in torch the padding row keeps its values
    trained = spnn.Embedding.from_pretrained(table.half(), freeze=False)
    assert trained.weight.requires_grad and trained.weight.dtype == torch.float16 and trained.scale == 1.0
    for bad in (table[0], table[None]):
        with pytest.raises(ValueError):
            spnn.Embedding.from_pretrained(bad)


def test_the_package_imports_without_the_torch_operators():
    """A missing or unusable module is an error of the operators that it holds, and of nothing else."""
    import subprocess
    import sys
    import textwrap

    code = """
        import os
        import torch

        found = os.path.exists
        os.path.exists = lambda path: not str(path).endswith("_bindings.so") and found(path)
        import torchsparse_b200 as ts
        from torchsparse_b200 import _ops, nn as spnn
        from torchsparse_b200.nn import functional as F

        spnn.Conv3d(4, 4, 3)
        y = spnn.GroupNorm(2, 4)(ts.SparseTensor(torch.randn(5, 4), torch.zeros(5, 4, dtype=torch.int32)))
        assert y.feats.shape == (5, 4)
        try:
            F.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(2, 4))
        except ImportError as e:
            assert "_bindings.so is missing" in str(e)
        else:
            raise AssertionError("no error")
        try:
            _ops.nothing
        except AttributeError:
            print("as expected")
    """
    got = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "as expected" in got.stdout, got.stderr


def test_one_block_per_sample_and_group_only_where_every_split_of_the_rows_suits_it():
    """The kernels of one block need no workspace.  They are taken by what a batch can hold, not by its mean alone: a batch
    of many nominal samples may have all its rows in one."""
    from torchsparse_b200._lib import lib

    small = lambda n, c, g, b, dtype: lib.tsb_group_norm_fwd_workspace_bytes(n, c, g, b, dtype) == 0      # noqa: E731
    assert small(1217, 256, 32, 1, 1) and small(4000, 64, 8, 1, 1) and small(16384, 64, 8, 16, 1) and small(8000, 256, 32, 16, 1)
    assert not small(16384, 64, 8, 64, 0)                  # 32768 vectors of a group: on 8 blocks if one sample has them
    assert not small(130_000, 32, 8, 64, 1)
    assert not small(16000, 64, 64, 16, 1)                 # groups of one 16-bit channel: 33 MB in reads of 32 bytes


def test_sizes_whose_flat_index_a_launch_cannot_hold_are_refused():
    from torchsparse_b200._lib import lib

    x, n, c = 256, (1 << 31) - 1, 1 << 20      # addresses are never read: every call is refused before a launch
    for channels in (c, c - 1):
        assert lib.tsb_embedding_fwd(x, x, 0, n, 3, channels, 1.0, 1, x, None) == 5
        assert lib.tsb_expert_dispatch(x, x, x, n, 1, channels, 1, x, None) == 5
    assert lib.tsb_embedding_fwd(x, x, 0, 5, 3, c + 1, 1.0, 1, x, None) == 5


def test_workspaces_of_wide_rows_go_by_the_blocks_that_run():
    from torchsparse_b200._lib import lib

    fwd, bwd = lib.tsb_group_norm_fwd_workspace_bytes, lib.tsb_group_norm_bwd_workspace_bytes
    # at most 256 column tiles, 444 blocks over all of them and a slot more for each tile and sample
    for n, c, g, b in ((10, 65536, 65536, 1), (300, 4096, 4096, 4), (300, 4096, 4096, 1000), (5000, 2048, 32, 4), (1_000_000, 64, 8, 8)):
        for dtype in (0, 1, 2):
            tiles = -(-c // 256)
            assert fwd(n, c, g, b, dtype) <= (444 + 2 * tiles + tiles * b) * g * 8 + 3 * 256 + 2 * b * g * 4
            assert bwd(n, c, g, b, dtype) <= (min(444, -(-n // 4)) + 2 * b) * c * 8 + b * g * 8 + 3 * 256
    assert fwd(10, 65536, 65536, 1, 1) < 512 << 20
