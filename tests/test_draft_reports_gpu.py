"""What the append of a tree reports of its parents, whichever kernel takes it."""
import pytest
import torch

from drafts_reference import trees
from test_kv_cache_gpu import heads, new_cache, raw

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("N,bad,parent", [(1, 0, 0), (1, 0, 5), (1, 0, -2), (2, 1, 1), (20, 0, 19), (20, 17, 17), (20, 19, -7), (300, 299, 300)])
def test_parents_that_cannot_be_are_reported_by_the_append(N, bad, parent, rotated, width):
    import monarch_attention_b200 as ma
    rotary = ma.RotaryPositions(width) if rotated else None
    k, v, q = (heads(3, h, N, width, BF, "tokens", s) for s, h in ((1, 2), (2, 2), (3, 4)))
    table, lengths = on_gpu([list(range(e * 20, e * 20 + 20)) for e in range(3)]), on_gpu([N + 3, N, N + 15])
    got = []
    for wrong in (False, True):   # (what cannot be counts as none)
        cache, parents = new_cache(60, 2, width, 16), trees(3, N, "random", 2)
        parents[2, bad] = parent if wrong else -1
        got.append([ma.append_kv_b200(cache, k, v, table, lengths, query=q if rotated else None, rotary=rotary, parents=parents), *raw(cache)])
        torch.cuda.synchronize()
        if wrong:
            with pytest.raises(RuntimeError, match="parent"):
                ma.append_kv_b200(cache, k, v, table, lengths)
        ma.append_kv_b200(cache, k, v, table, lengths)   # (nothing is left to report)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("N", [1, 20])
def test_parents_of_padding_are_not_looked_at(N, rotated):
    import monarch_attention_b200 as ma
    k, v = (heads(2, 2, N, 64, BF, "tokens", s) for s in (1, 2))
    parents = trees(2, N, "random", 2)
    parents[1] = 1000
    for _ in range(2):
        ma.append_kv_b200(new_cache(8, 2, 64, 16), k, v, on_gpu([[0, 1, 2, 3], [4, 5, 6, 7]]), on_gpu([N, 9]), on_gpu([N, 0]), rotary=ma.RotaryPositions(64) if rotated else None, parents=parents)
        torch.cuda.synchronize()
