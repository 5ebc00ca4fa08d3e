"""Definitions of the decoder's side that need no GPU: modules from before, rotations that are none."""
import torch

import monarch_attention_b200 as ma


def test_a_module_pickled_without_a_rotary_has_none():
    """A whole module's pickle is its dictionary, which from before the rotary positions does not name them."""
    module = ma.MonarchAttention(16, 2, ma.PadType.post)
    module._impl_fn = lambda q, k, v, m, T, B, pre_pad: q + k + v
    old = ma.MonarchAttention.__new__(ma.MonarchAttention)
    old.__setstate__({k: v for k, v in module.__dict__.items() if k != "rotary"})
    x = torch.ones(1, 1, 2, 4)
    assert old.rotary is None and torch.equal(old(x, x, x), 3 * x) and torch.equal(module(x, x, x), 3 * x)
