"""CPU tests of the training modules' construction: what nn.Embedding's and nn.LayerNorm's users call."""

import copy
import pickle

import pytest
import torch
import torch.nn as nn

import genie_tk


def test_embedding_from_pretrained():
    table = torch.randn(7, 5)
    m = genie_tk.Embedding.from_pretrained(table)
    ref = nn.Embedding.from_pretrained(table)
    assert type(m) is genie_tk.Embedding and m.weight.data_ptr() == table.data_ptr()
    assert m.weight.requires_grad is ref.weight.requires_grad is False
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (7, 5, None, 1.0)
    m = genie_tk.Embedding.from_pretrained(table, freeze=False, padding_idx=-2, scale=2.0)
    assert m.weight.requires_grad and m.padding_idx == 5 and m.scale == 2.0
    assert torch.equal(m.weight, table)  # a given padding row stays
    for t in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert t.scale == 2.0 and t.padding_idx == 5 and torch.equal(t.weight, table)
    with pytest.raises(ValueError, match="2-D"):
        genie_tk.Embedding.from_pretrained(table[0])


def test_options_of_nn_embedding_that_are_not_offered():
    """They raise by name; the values that nn.Embedding has by default are accepted."""
    table = torch.randn(7, 5)
    for bad in ({"max_norm": 1.0}, {"max_norm": 0.0}, {"scale_grad_by_freq": True}, {"sparse": True}):
        with pytest.raises(ValueError, match=next(iter(bad))):
            genie_tk.Embedding.from_pretrained(table, **bad)
    genie_tk.Embedding.from_pretrained(table, max_norm=None, norm_type=2.0, scale_grad_by_freq=False, sparse=False)
