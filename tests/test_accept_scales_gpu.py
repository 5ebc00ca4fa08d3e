"""Acceptance of tokens whose block has a scale that is no number."""
import pytest
import torch

from decoder_reference import held

pytestmark = pytest.mark.gpu


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_tokens_of_a_scale_of_nan_stay_nan(bad, width):
    """A token moves with what it stands for, NaN in all its features: its place does not keep the codes of a rejected token."""
    import monarch_attention_b200 as ma
    g = torch.Generator(device="cuda").manual_seed(bad)
    cache = ma.PagedKV.allocate(4, 2, width, 16)
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        c.view(torch.uint8).copy_(torch.randint(0, 0x7f, c.shape, generator=g, device="cuda"))
        s.copy_(2.0 ** torch.randint(-3, 4, s.shape, generator=g, device="cuda"))
    page = on_gpu([[2, 0, 3]])
    cache.k_scale[page[0, bad].long(), 1] = float("nan")   # of one head's block, keys only
    before = [held(c, s, page[0], 40, 16) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    # 30 tokens behind 10: token 0 stands where it is, 7 (place 17) and 25 (place 35) take places 11 and 12, in block 0
    parents, tokens, answers = torch.zeros(1, 30, dtype=torch.int32, device="cuda"), torch.arange(30, dtype=torch.int32, device="cuda")[None], on_gpu([[-5] * 30])
    parents[0, 0], parents[0, 25] = -1, 7
    answers[0, 0], answers[0, 7] = 7, 25
    got = ma.accept_drafts_b200(cache, page, on_gpu([40]), on_gpu([30]), parents, tokens, answers)
    assert got.path[0, :4].tolist() == [0, 7, 25, -1] and got.lengths.tolist() == [13]
    place = list(range(11)) + [17, 35]
    for j, (c, s) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        now, want = held(c, s, page[0], 13, 16), before[j][:, place]
        assert torch.equal(torch.isnan(now), torch.isnan(want)) and torch.isnan(want).any() == (j == 0)
        # exact but for values that become subnormal: half a step of those
        scale = torch.nan_to_num(s[2].cpu().double(), nan=0.0)[:, :, None]
        assert bool(((now - want).nan_to_num(nan=0.0).abs() <= 2.0 ** -10 * scale).all())
