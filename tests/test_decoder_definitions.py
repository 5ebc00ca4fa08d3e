"""Definitions of the decoder's side that need no GPU: modules from before, rotations that are none."""
import pytest
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


@pytest.mark.parametrize("factor", [0.99, 0.5, 1e-5])
def test_yarn_is_for_longer_contexts(factor):
    """Below one its multiplier of sines would shrink scores, and end below zero."""
    with pytest.raises(ValueError, match="factor"):
        ma.RotaryPositions(64, scaling="yarn", factor=factor, trained_length=4096)
    assert ma.RotaryPositions(64, scaling="yarn", factor=1.0, trained_length=4096).magnitude == 1.0


@pytest.mark.parametrize("kw", [dict(base=1e300, scaling="ntk", factor=1e300), dict(base=1e200, scaling="ntk", factor=1e150), dict(base=1e-200, scaling="ntk", factor=1e-200), dict(base=1e-320), dict(base=1e-300, scaling="linear", factor=1e-100)])
def test_frequencies_that_are_no_numbers_are_refused(kw):
    with pytest.raises(ValueError, match="frequencies"):
        ma.RotaryPositions(64, **kw)
