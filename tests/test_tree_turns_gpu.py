"""Trees of up to 128 rows whose two tiles take the steps in turns, against the definition in 64 bits: windows, caps, far scores, keys of NaN.

The tiles go in turns where there are 16 heads or more and a CTA has steps enough: by the columns of the table, 10 for up to 64 rows and 24 for up to 128 with a CTA for each
of 148 SMs, 16 with more heads than SMs (up to 64 rows).
"""
import pytest
import torch

from decoder_reference import HALF_STEP, SUBNORMAL
from drafts_reference import line, seen_by_tree, trees
from test_cached_attention_gpu import filled, queries
from test_tree_attention_gpu import on_gpu

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
PAGE = 64


def held_on_gpu(codes, scales, table, length):
    """(heads, length, D) in 64 bits: what a sequence's cached tokens stand for."""
    used = table[:-(-length // PAGE)].long()
    x = codes.view(torch.uint8)[used].view(torch.float8_e4m3fn).double() * scales[used].double().repeat_interleave(16, -1)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def definition(q, k, v, seen, softcap):
    """Result and bound: ``decoder_reference.attention`` for rows with a line of keys each, on the GPU.  (Scores that are off by `off` change a weight, and the sum that it is
    divided by, by factors of up to exp(off) each; far from zero that is more than 1 + off.)"""
    H, n, D = q.shape
    q, k, v = q.double(), *(t.repeat_interleave(H // t.shape[0], 0) for t in (k, v))
    s, size = q @ k.mT * D ** -0.5, (q.abs() @ k.abs().mT) * D ** -0.5
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -torch.inf), -1), nan=0.0)
    off = (size * (1.5 * D + 8) * 2.0 ** -24 + softcap * 2.0 ** -22).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    return w @ v, ((1 + 2.0 ** -11 + 2.0 ** -20) * torch.exp(2 * off) - 1) * (w @ v.abs()) + seen.shape[1] * 2.0 ** -24 * v.abs().amax()


def check(out, q, cache, table, lengths, counts, parents, window=0, softcap=0.0):
    E, H, N, D = q.shape
    for e in range(E):
        L, n = lengths[e], counts[e]
        assert not bool(out[e, :, n:].any()), "rows of padding are zero"
        if n == 0:
            continue
        k, v = held_on_gpu(cache.k, cache.k_scale, table[e], L), held_on_gpu(cache.v, cache.v_scale, table[e], L)
        want, bound = definition(q[e, :, :n], k, v, seen_by_tree(parents[e].tolist(), L, n, window).cuda(), softcap)
        got, bound = out[e, :, :n].double(), bound + HALF_STEP[q.dtype] * (want.abs() + bound) + SUBNORMAL[q.dtype]
        assert torch.isfinite(got).all()
        over = (got - want).abs() - bound
        assert bool((over <= 0).all()), f"sequence {e} of {L} tokens: {float((over > 0).double().mean()):.2e} of the elements over the bound, off by {float((got - want).abs().max()):.3e}"


SHAPES = {  # E, H, Hk, N, columns of the table (of 64 tokens)
    "64 rows": (16, 4, 2, 32, 98), "128 rows": (16, 8, 4, 64, 122), "33 rows": (16, 2, 2, 33, 98), "more heads than SMs": (40, 8, 4, 32, 34), "125 rows": (20, 5, 1, 25, 360)}


def case(shape, D, dtype, seed=0):
    E, H, Hk, N, columns = SHAPES[shape]
    g = torch.Generator().manual_seed(seed)
    most = columns * PAGE
    counts = [N if e % 3 else int(torch.randint(0, N + 1, (), generator=g)) for e in range(E)]
    # full, of any length, of one step or less, and with an odd number of steps
    lengths = [max(c, (most, int(torch.randint(1, most, (), generator=g)), int(torch.randint(1, 129, (), generator=g)), 128 * 3 - 5)[e % 4]) for e, c in enumerate(counts)]
    cache, table = filled(E, columns, Hk, D, PAGE, lengths, "tokens", seed)
    return cache, table, lengths, counts, queries(E, H, N, D, dtype, "tokens", seed + 1), trees(E, N, "random", seed)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (0, 20.0), (3, 0.0), (130, 15.0), (700, 0.0), (2500, 0.0)])
def test_turns_match_the_definition(shape, D, dtype, window, softcap):
    import monarch_attention_b200 as ma
    cache, table, lengths, counts, q, parents = case(shape, D, dtype)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents, window=window, softcap=softcap)
    check(out, q, cache, table, lengths, counts, parents, window, softcap)
    assert torch.equal(out, ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents, window=window, softcap=softcap))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("power", [9, 10])
def test_scores_far_from_zero_in_turns(shape, D, dtype, window, power):
    """The path of rows apart, from the first step of a tile on, and (a quarter of the blocks) from a later one."""
    import monarch_attention_b200 as ma
    cache, table, lengths, counts, q, parents = case(shape, D, dtype, 3)
    if power == 9:
        cache.k_scale.mul_(2.0 ** 9)
    else:
        cache.k_scale.view(-1)[::4].mul_(2.0 ** power)
    out = ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents, window=window)
    check(out, q, cache, table, lengths, counts, parents, window)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_keys_of_nan_in_turns(shape, D, dtype):
    """A key of NaN among the call's tokens reaches its descendants, one in front of them all rows of its sequence; the others keep their bits."""
    import monarch_attention_b200 as ma
    cache, table, lengths, counts, q, parents = case(shape, D, dtype, 5)
    call = lambda: ma.cached_attention_b200(q, cache, table, *on_gpu(lengths, counts), parents=parents)  # noqa: E731
    clean = call()
    reached = torch.zeros(q.shape[0], q.shape[2], dtype=torch.bool)
    for e, (L, n) in enumerate(zip(lengths, counts)):
        if n < 2 or e % 4 == 3:
            continue
        rows = parents[e].tolist()
        if e % 4 == 0 and L > n:
            place = (L - n) // 2
            reached[e, :n] = True
        else:
            bad = n // 2
            place = L - n + bad
            reached[e, :n] = torch.tensor([bad in line(rows, i) for i in range(n)])
        cache.k.view(torch.uint8)[table[e, place // PAGE].long(), :, place % PAGE] = 0x7f
    out, reached = call(), reached.cuda()[:, None, :, None].expand_as(clean)
    assert torch.equal(torch.isnan(out), reached) and torch.equal(out[~reached], clean[~reached]) and reached.any() and not reached.all()
