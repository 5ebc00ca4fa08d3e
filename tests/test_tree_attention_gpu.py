"""Attention of drafted trees over the paged cache, and their append, against the definitions in 64 bits."""
import pytest
import torch

from decoder_reference import HALF_STEP, SUBNORMAL, close, held, rotate, rotation_bound
from drafts_reference import line, power_for, seen_by_tree, tree_attention, trees
from test_cached_attention_gpu import filled, queries
from test_kv_cache_gpu import heads, new_cache, raw

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def on_gpu(*lists):
    return [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in lists]


def check(out, q, cache, table, lengths, counts, page, parents, window=0, softcap=0.0):
    E, H, N, D = q.shape
    assert out.shape == q.shape and out.dtype == q.dtype
    for e in range(E):
        L, n = lengths[e], N if counts is None else counts[e]
        assert not bool(out[e, :, n:].any()), "rows of padding are zero"
        if n == 0:
            continue
        k, v = held(cache.k, cache.k_scale, table[e], L, page), held(cache.v, cache.v_scale, table[e], L, page)
        want, bound = tree_attention(q[e, :, :n].double().cpu(), k, v, seen_by_tree(parents[e].tolist(), L, n, window), D ** -0.5, softcap)
        close(out[e, :, :n], want, bound + HALF_STEP[q.dtype] * (want.abs() + bound) + SUBNORMAL[q.dtype], f"sequence {e} of {L} tokens")


CASES = [  # E, H, Hk, N, D, page, lengths, counts
    (1, 1, 1, 1, 64, 16, [1], None), (2, 4, 4, 2, 128, 16, [2, 40], None), (3, 12, 12, 7, 64, 16, [7, 500, 129], [7, 5, 0]), (2, 8, 2, 8, 128, 64, [300, 8], [8, 3]),
    (2, 2, 2, 32, 64, 32, [32, 170], [32, 31]), (1, 6, 2, 9, 128, 128, [1025], None), (4, 5, 1, 5, 64, 16, [70, 5, 33, 2], [5, 5, 1, 5]), (20, 8, 8, 17, 128, 64, list(range(17, 417, 20)), None),
    (1, 3, 1, 10, 64, 64, [9000], None),
    (2, 1, 1, 33, 64, 16, [33, 129], [33, 30]), (2, 16, 4, 61, 128, 64, [700, 61], [61, 7]), (1, 8, 1, 25, 64, 32, [4100], None), (1, 2, 2, 128, 128, 128, [128], None), (1, 3, 1, 300, 64, 64, [1000], None),
    (1, 1, 1, 512, 128, 16, [600], None), (2, 2, 1, 400, 64, 32, [401, 30], [400, 40])]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["forest", "random", "wide", "star"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_trees_match_the_definition(case, kind, dtype):
    import monarch_attention_b200 as ma
    E, H, Hk, N, D, page, lengths, counts = CASES[case]
    cache, table = filled(E, max(lengths) // page + 2, Hk, D, page, lengths, "tokens" if case % 2 else "heads", seed=case)
    q, parents = queries(E, H, N, D, dtype, "tokens" if case % 2 else "heads"), trees(E, N, kind, case)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents, token_major_output=bool(case % 2))
    check(out, q, cache, table, lengths, counts, page, parents)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N,window,softcap", [(1, 1, 0.0), (6, 1, 0.0), (6, 2, 20.0), (8, 100, 0.0), (8, 10 ** 9, 0.0), (60, 1, 0.0), (60, 3, 15.0), (60, 200, 0.0), (300, 5, 0.0)])
@pytest.mark.parametrize("kind", ["random", "chain", "forest"])
def test_windows_are_of_positions(N, window, softcap, kind, dtype):
    import monarch_attention_b200 as ma
    lengths, counts, page = [N, 333, 1025, 150 + N], [N, max(N - 3, 1), 0, N], 32
    lengths[1] = max(lengths[1], N)
    cache, table = filled(4, 50, 2, 64, page, lengths)
    q, parents = queries(4, 8, N, 64, dtype, "tokens"), trees(4, N, kind, N)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), window=window, softcap=softcap, parents=parents)
    check(out, q, cache, table, lengths, counts, page, parents, window, softcap)


@pytest.mark.parametrize("H,Hk,N,lengths,counts,window,softcap", [(4, 4, 1, [700], None, 0, 0.0), (8, 2, 8, [4000, 20], [8, 6], 0, 10.0), (4, 4, 32, [900], None, 50, 0.0), (2, 1, 100, [5000, 100], None, 0, 0.0),
                                                                 (1, 1, 500, [600], None, 300, 0.0)])
def test_a_chain_is_what_ordinary_tokens_are(H, Hk, N, lengths, counts, window, softcap):
    import monarch_attention_b200 as ma
    E = len(lengths)
    cache, table = filled(E, max(lengths) // 64 + 2, Hk, 128, 64, lengths)
    q, sizes = queries(E, H, N, 128, BF, "tokens"), on_gpu(lengths, counts)
    kw = dict(window=window, softcap=softcap)
    parents = trees(E, N, "chain")
    out = ma.cached_attention_b200(q, cache, table, *sizes, parents=parents, **kw)
    if N * H // Hk <= 8:   # the same kernel, with another mask
        assert torch.equal(out, ma.cached_attention_b200(q, cache, table, *sizes, **kw))
    check(out, q, cache, table, lengths, counts, 64, parents, **kw)


@pytest.mark.parametrize("N", [6, 60])
def test_keys_of_nan_reach_their_descendants_only(N):
    import monarch_attention_b200 as ma
    lengths, page = [200 + N], 32
    cache, table = filled(1, 12, 2, 64, page, lengths)
    q, parents = queries(1, 8, N, 64, BF, "heads"), trees(1, N, "random", 3)
    bad = next(n for n in range(N - 1, 0, -1) if n in parents[0].tolist())
    position = 200 + bad
    clean = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths), parents=parents)
    cache.k.view(torch.uint8)[table[0, position // page].long(), :, position % page] = 0x7f
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths), parents=parents)
    below = torch.tensor([bad in line(parents[0].tolist(), n) for n in range(N)], device="cuda")
    assert torch.isnan(out[:, :, below]).all() and torch.equal(out[:, :, ~below], clean[:, :, ~below]) and below.any() and not below.all()


@pytest.mark.parametrize("N", [5, 70])
def test_scores_of_any_magnitude(N):
    """Rows whose scores lie far from zero take paths of their own: the mask holds there too."""
    import monarch_attention_b200 as ma
    lengths, page = [300 + N, 128 + N], 64
    cache, table = filled(2, 8, 2, 128, page, lengths)
    cache.k_scale.mul_(2.0 ** 9)
    q, parents = queries(2, 4, N, 128, BF, "tokens"), trees(2, N, "forest", 5)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths), parents=parents)
    check(out, q, cache, table, lengths, None, page, parents)


@pytest.mark.parametrize("N", [4, 50])
def test_rows_in_front_of_the_sequence_see_nothing(N):
    """A count above the length puts tokens in front of the first place: they are zero, and nobody's ancestors."""
    import monarch_attention_b200 as ma
    lengths, page = [N // 2, 1], 16
    cache, table = filled(2, N // 16 + 2, 1, 64, page, lengths)
    q, parents = queries(2, 2, N, 64, HF, "heads"), trees(2, N, "random", 1)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths), parents=parents)
    check(out, q, cache, table, lengths, None, page, parents)


@pytest.mark.parametrize("N", [6, 40])
def test_parents_that_cannot_be_count_as_none_and_are_reported(N):
    import monarch_attention_b200 as ma
    lengths, page = [100 + N], 32
    cache, table = filled(1, 8, 2, 64, page, lengths)
    q, parents = queries(1, 4, N, 64, BF, "heads"), trees(1, N, "random", 1)
    parents[0, 3], parents[0, 4], parents[0, 5] = 3, N + 5, -7
    sizes = on_gpu(lengths)
    out = ma.cached_attention_b200(q, cache, table, *sizes, parents=parents)
    check(out, q, cache, table, lengths, None, page, parents)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="parent"):
        ma.cached_attention_b200(q, cache, table, *sizes)
    ma.cached_attention_b200(q, cache, table, *sizes)


@pytest.mark.parametrize("N", [8, 60, 130])
def test_one_tree_for_all_and_results_in_place(N):
    """Parents with a batch stride of zero; a result in the query's place and beside its rows; a call on a stream of its own."""
    import monarch_attention_b200 as ma
    lengths, page = [N, 900, 2000], 32
    cache, table = filled(3, 70, 2, 64, page, lengths)
    both = torch.empty(3, N, 2, 4, 64, dtype=BF, device="cuda")   # rows of queries beside those of results
    q, beside = (both[:, :, i].transpose(1, 2) for i in range(2))
    q.copy_(queries(3, 4, N, 64, BF, "heads"))
    one = trees(1, N, "random", 2)
    sizes, alone = on_gpu(lengths), q.clone()
    want = ma.cached_attention_b200(alone, cache, table, *sizes, parents=one.repeat(3, 1))
    check(want, alone, cache, table, lengths, None, page, one.repeat(3, 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ma.cached_attention_b200(q, cache, table, *sizes, parents=one.expand(3, N), out=beside) is not None
        in_place = ma.cached_attention_b200(q, cache, table, *sizes, parents=one.expand(3, N), out=q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(beside, want) and torch.equal(in_place, want)


@pytest.mark.parametrize("E,H,Hk,N,D,lengths,counts", [(16, 4, 4, 33, 128, [1400] * 16, None), (20, 4, 4, 50, 64, list(range(50, 2050, 100)), [50, 7] * 10), (40, 8, 8, 64, 64, [2100] * 20 + [70] * 20, None),
                                                       (16, 8, 4, 64, 128, [5000] * 15 + [64], None), (3, 8, 8, 128, 64, [128, 9000, 300], [128, 0, 100]), (148, 1, 1, 40, 64, list(range(40, 188)), None)])
def test_many_rows_in_any_shares(E, H, Hk, N, D, lengths, counts):
    """Even pieces of ragged lengths, tiles of the same rows in turns, more heads than SMs."""
    import monarch_attention_b200 as ma
    page, per = 64, max(lengths) // 64 + 20
    cache, table = filled(E, per, Hk, D, page, lengths, spare=1)
    q, parents = queries(E, H, N, D, HF, "tokens"), trees(E, N, "random", 4)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents)
    look = [0, E // 2, E - 1]   # (the definition in 64 bits takes a second a sequence)
    check(out[look], q[look], cache, table[look], [lengths[i] for i in look], None if counts is None else [counts[i] for i in look], page, parents[look])
    assert torch.isfinite(out).all()
    again = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents)
    assert torch.equal(out, again)


# --- the append --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("E,H,Hk,N,D,page,dim,pairs,dtype,layout", [
    (2, 4, 2, 7, 64, 16, 64, "half", BF, "heads"), (3, 6, 2, 20, 128, 64, 128, "interleaved", HF, "tokens"), (1, 12, 12, 61, 64, 32, 32, "half", HF, "tokens"),
    (2, 4, 1, 200, 128, 128, 64, "half", BF, "tokens"), (1, 2, 2, 512, 64, 16, 64, "interleaved", BF, "heads"), (2, 3, 3, 1, 64, 16, 64, "half", BF, "heads")])
@pytest.mark.parametrize("kind", ["random", "forest", "star"])
def test_trees_are_appended_at_the_positions_of_their_depth(E, H, Hk, N, D, page, dim, pairs, dtype, layout, kind):
    import monarch_attention_b200 as ma
    rotary = ma.RotaryPositions(dim, pairs=pairs)
    first = [5, 0, 30][:E]
    counts = [N, max(N - 2, 1), N][:E]
    per = (30 + N) // page + 2
    table = torch.randperm(E * per, generator=torch.Generator().manual_seed(1)).view(E, per).to(torch.int32).cuda()
    cache = new_cache(E * per, Hk, D, page, layout)
    k0, v0 = (heads(E, Hk, 30, D, dtype, layout, s) for s in (1, 2))
    ma.append_kv_b200(cache, k0, v0, table, *on_gpu(first, first))
    before = [[held(c, s, table[e], first[e], page) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))] for e in range(E)]
    k, v, q = (heads(E, h, N, D, dtype, layout, s) for s, h in ((3, Hk), (4, Hk), (5, H)))
    parents = trees(E, N, kind, 2)
    lengths = [a + b for a, b in zip(first, counts)]
    q_out = ma.append_kv_b200(cache, k, v, table, *on_gpu(lengths, counts), query=q, rotary=rotary, parents=parents)
    for e in range(E):
        n, rows = counts[e], parents[e].tolist()
        place = torch.tensor([first[e] + len(line(rows, i)) - 1 for i in range(n)])
        want, size = rotate(q[e, :, :n], place, rotary)
        close(q_out[e, :, :n], want, rotation_bound(want, size, dtype), f"query of {e}")
        assert not bool(q_out[e, :, n:].any())
        want_k, size_k = rotate(k[e, :, :n], place, rotary)
        for j, (c, s, want, off) in enumerate(((cache.k, cache.k_scale, want_k, 8 * 2.0 ** -24 * size_k), (cache.v, cache.v_scale, v[e, :, :n].double().cpu(), 0.0))):
            got = held(c, s, table[e], lengths[e], page)
            scale = s.cpu()[table[e].long().cpu()].double().transpose(0, 1).flatten(1, 2).repeat_interleave(16, -1)[:, :lengths[e], None]
            # half a step of e4m3, or of its subnormal codes, of which older tokens may have taken one more
            bound = 2.0 ** -4 * want.abs() + scale[:, first[e]:] * 2.0 ** -10 + 2 * off
            close(got[:, first[e]:], want, bound, f"{'kv'[j]} of {e}")
            close(got[:, :first[e]], before[e][j], scale[:, :first[e]] * 2.0 ** -10, f"older {'kv'[j]} of {e}")
            for b in range(-(-first[e] // 16), -(-lengths[e] // 16)):   # blocks of nothing but the call's tokens have the smallest scale that holds them
                most = want[:, b * 16 - first[e]:b * 16 + 16 - first[e]].abs().amax((-1, -2))
                for h in range(Hk):
                    assert float(scale[h, b * 16, 0]) in (power_for(float(most[h]) * (1 - 2.0 ** -20)), power_for(float(most[h]) * (1 + 2.0 ** -20)))


def test_a_chain_is_appended_like_ordinary_tokens():
    import monarch_attention_b200 as ma
    rotary = ma.RotaryPositions(128)
    k, v, q = (heads(2, h, 50, 128, BF, "tokens", s) for s, h in ((3, 2), (4, 2), (5, 4)))
    table = torch.arange(10, dtype=torch.int32, device="cuda").view(2, 5)
    got = []
    for parents in (None, trees(2, 50, "chain")):
        cache = new_cache(10, 2, 128, 32)
        got.append([ma.append_kv_b200(cache, k, v, table, *on_gpu([60, 50], [50, 41]), query=q, rotary=rotary, parents=parents), *raw(cache)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_without_a_rotation_parents_change_nothing():
    import monarch_attention_b200 as ma
    k, v = (heads(1, 2, 20, 64, BF, "tokens", s) for s in (3, 4))
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    got = []
    for parents in (None, trees(1, 20, "star")):
        cache = new_cache(4, 2, 64, 16)
        ma.append_kv_b200(cache, k, v, table, *on_gpu([25], [20]), parents=parents)
        got.append(raw(cache))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals():
    import monarch_attention_b200 as ma
    cache, table = filled(1, 40, 1, 64, 16, [600])
    sizes = on_gpu([600])
    q = queries(1, 1, 4, 64, BF, "heads")
    good = trees(1, 4, "chain")
    for bad in (good.long(), good[:, :3], good[0], good.expand(2, 4), good.cpu(), trees(1, 8, "chain")[:, ::2]):
        with pytest.raises(ValueError):
            ma.cached_attention_b200(q, cache, table, *sizes, parents=bad)
        with pytest.raises(ValueError):
            ma.append_kv_b200(cache, q, q, table, *sizes, parents=bad)
    with pytest.raises(ValueError, match="causal"):
        ma.cached_attention_b200(q, cache, table, *sizes, causal=False, parents=good)
    q = queries(1, 1, 513, 64, BF, "heads")
    for call in (lambda: ma.cached_attention_b200(q, cache, table, *sizes, parents=trees(1, 513, "chain")),
                 lambda: ma.append_kv_b200(cache, q, q, table, *sizes, parents=trees(1, 513, "chain"))):
        with pytest.raises(ValueError, match="512"):
            call()
