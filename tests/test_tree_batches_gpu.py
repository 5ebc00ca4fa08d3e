"""The append of trees of many sequences at once has the bits of one sequence at a time, however its heads are spread over the GPU."""
import pytest
import torch

from drafts_reference import trees
from test_kv_cache_gpu import heads, new_cache, raw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,H,Hk,N,D", [(30, 32, 8, 61, 128), (38, 32, 8, 61, 128), (48, 32, 8, 61, 128), (66, 32, 8, 61, 128), (100, 32, 8, 61, 128), (74, 40, 8, 20, 128), (64, 12, 12, 25, 64), (123, 12, 12, 25, 64),
                                        (80, 12, 12, 9, 64), (60, 24, 8, 40, 64), (90, 16, 16, 40, 64), (200, 28, 2, 7, 128), (75, 44, 1, 15, 128)])
def test_a_batch_of_trees_is_its_sequences(E, H, Hk, N, D):
    import monarch_attention_b200 as ma
    page, per, rotary = 64, 3, ma.RotaryPositions(D)
    table = torch.randperm(E * per, generator=torch.Generator().manual_seed(E)).view(E, per).to(torch.int32).cuda()
    g = torch.Generator().manual_seed(N)
    counts = torch.randint(0, N + 1, (E,), generator=g).to(torch.int32).cuda()
    counts[::3] = N
    lengths = counts + torch.randint(0, 60, (E,), generator=g).to(torch.int32).cuda()
    q, k, v = (heads(E, h, N, D, torch.bfloat16, "tokens", s) for s, h in ((1, H), (2, Hk), (3, Hk)))
    parents = trees(E, N, "random", 1)
    whole, single = (new_cache(E * per, Hk, D, page, "tokens") for _ in range(2))
    out = ma.append_kv_b200(whole, k, v, table, lengths, counts, query=q, rotary=rotary, parents=parents)
    for e in range(E):
        one = ma.append_kv_b200(single, k[e:e + 1], v[e:e + 1], table[e:e + 1], lengths[e:e + 1], counts[e:e + 1], query=q[e:e + 1], rotary=rotary, parents=parents[e:e + 1])
        assert torch.equal(one[0], out[e])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(raw(whole), raw(single)))
