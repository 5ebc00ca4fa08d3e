"""The decoder layer's attention refuses a call before it changes the cache."""
import pytest
import torch

import monarch_attention_b200 as ma


def layer_inputs(device):
    x = torch.ones(1, 2, 3, 64, dtype=torch.bfloat16, device=device)
    table, lengths, parents = (torch.tensor(t, dtype=torch.int32, device=device) for t in ([[0, 1, 2]], [3], [[-1, 0, 1]]))
    return x, ma.PagedKV.allocate(3, 2, 64, 16, device=device), table, lengths, parents


def test_trees_need_a_causal_layer():
    x, cache, table, lengths, parents = layer_inputs("cpu")
    for key in (x, None):   # (nothing has looked at the tensors yet, which are the host's)
        with pytest.raises(ValueError, match="causal"):
            ma.CachedAttention(causal=False)(x, key, key, cache, table, lengths, None, parents)


@pytest.mark.gpu
def test_a_refused_tree_leaves_the_cache():
    x, cache, table, lengths, parents = layer_inputs("cuda")
    layer = ma.CachedAttention(causal=False)
    with pytest.raises(ValueError, match="causal"):
        layer(x, x, x, cache, table, lengths, None, parents)
    assert not any(bool(t.view(torch.uint8).any()) for t in cache)
    layer(x, x, x, cache, table, lengths)
    assert bool(cache.k.view(torch.uint8).any())
