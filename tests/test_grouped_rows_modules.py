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
