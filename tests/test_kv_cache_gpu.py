"""The append to the paged 8-bit cache: codes and scales against the definition in 64 bits, over several calls of all sizes."""
import pytest
import torch

from decoder_reference import HALF_STEP, held, rotate, rotation_bound

pytestmark = pytest.mark.gpu


def heads(E, H, N, D, dtype, layout, seed, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (E, N, H, D) if layout == "tokens" else (E, H, N, D)
    t = (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)
    return t.permute(0, 2, 1, 3) if layout == "tokens" else t


def new_cache(pages, Hk, D, page, layout="heads"):
    """A pool with other owners' leavings in it, NaN among them."""
    import monarch_attention_b200 as ma
    g = torch.Generator(device="cuda").manual_seed(7)
    shape = (pages, Hk, page, D) if layout == "heads" else (pages, page, Hk, D)
    codes = [torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    if layout == "tokens":
        codes = [c.permute(0, 2, 1, 3) for c in codes]
    scales = [torch.rand(pages, Hk, page // 16, generator=g, device="cuda") for _ in range(2)]
    return ma.PagedKV(*codes, *scales)


def raw(cache):
    return [t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone() for t in cache]


STEPS = [  # tokens of each call
    [1] * 20, [5, 1, 1, 40, 1], [16, 16, 1], [33, 15], [100], [1, 130, 1, 2]]


@pytest.mark.parametrize("steps", STEPS)
@pytest.mark.parametrize("E,H,Hk,D,page,dim,pairs,dtype,layout", [
    (1, 1, 1, 64, 16, 64, "half", torch.bfloat16, "heads"), (3, 6, 2, 128, 64, 128, "interleaved", torch.bfloat16, "tokens"),
    (2, 12, 12, 64, 32, 32, "half", torch.float16, "tokens"), (2, 5, 5, 128, 16, 0, "half", torch.float16, "heads"),
    (4, 8, 1, 128, 128, 64, "half", torch.bfloat16, "tokens"), (2, 3, 3, 64, 64, 16, "interleaved", torch.float16, "tokens"), (1, 4, 9, 128, 32, 16, "half", torch.bfloat16, "heads")])
def test_append_matches_the_definition(E, H, Hk, D, page, dim, pairs, dtype, layout, steps):
    import monarch_attention_b200 as ma
    total = sum(steps)
    per = total // page + 2
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(E * per + 3, generator=g)[:E * per].view(E, per).to(torch.int32).cuda()
    cache = new_cache(E * per + 3, Hk, D, page, layout)
    rotary = ma.RotaryPositions(dim, pairs=pairs) if dim else None
    lengths = torch.randint(0, 3, (E,), generator=g).mul(0)
    truth = {n: torch.zeros(E, Hk, 0, D, dtype=torch.float64) for n in "kv"}
    truth = {n: [truth[n][e] for e in range(E)] for n in "kv"}
    slack = {n: [torch.zeros(Hk, 0, D, dtype=torch.float64) for e in range(E)] for n in "kv"}
    for i, N in enumerate(steps):
        # all of the call's tokens, or fewer, none among them
        counts = torch.randint(0, N + 1, (E,), generator=g) if i % 2 else torch.full((E,), N)
        growth = 4.0 ** (min(i, 8) if dtype == torch.float16 else i)   # (f16 ends at 65504: the definition of more is not finite itself)
        k, v, q = (heads(E, h, N, D, dtype, layout, 10 * i + j, std=0.01 * growth) for j, h in enumerate((Hk, Hk, H)))
        lengths = lengths + counts
        before = raw(cache)
        out = ma.append_kv_b200(cache, k, v, table, lengths.to(torch.int32).cuda(), counts.to(torch.int32).cuda() if i % 2 else None, query=q, rotary=rotary)
        assert out.shape == q.shape and out.dtype == dtype
        after = raw(cache)
        for e in range(E):
            n, start = int(counts[e]), int(lengths[e] - counts[e])
            place = torch.arange(start, start + n)
            new = {}
            for name, x in (("k", k), ("v", v), ("q", q)):
                x = x[e, :, :n]
                if rotary is not None and name != "v":
                    new[name] = rotate(x, place, rotary)
                else:
                    new[name] = x.double().cpu(), torch.zeros(x.shape, dtype=torch.float64)
            want, size = new["q"]
            got = out[e].double().cpu()
            assert bool(((got[:, :n] - want).abs() <= rotation_bound(want, size, dtype)).all()) and not bool(got[:, n:].any())
            for name in "kv":
                truth[name][e] = torch.cat((truth[name][e], new[name][0]), 1)
                slack[name][e] = torch.cat((slack[name][e], 8 * 2.0 ** -24 * new[name][1]), 1)
        # nothing but the sequences' own slots and blocks has changed
        mine = torch.zeros(E * per + 3, page, dtype=torch.bool)
        for e in range(E):
            p = torch.arange(int(lengths[e] - counts[e]) // 16 * 16 if counts[e] else int(lengths[e]), int(lengths[e]))
            mine[table[e].cpu().long()[p // page], p % page] = True
        for a, b in zip(before[:2], after[:2]):
            assert torch.equal(a.cpu().transpose(1, 2)[~mine], b.cpu().transpose(1, 2)[~mine])
        blocks = mine.view(-1, page // 16, 16).any(-1)
        for a, b in zip(before[2:], after[2:]):
            assert torch.equal(a.cpu().transpose(1, 2)[~blocks], b.cpu().transpose(1, 2)[~blocks])
    for e in range(E):
        L = int(lengths[e])
        for name, codes, scales in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
            got = held(codes, scales, table[e], L, page)
            s = scales.cpu()[table[e].cpu().long()].double().transpose(0, 1).flatten(1).repeat_interleave(16, -1)[:, :L, None]
            # half a step of the type, twice in the subnormal range, where a code may have been re-expressed (each raise rounds again)
            bound = truth[name][e].abs() * 2.0 ** -4 + s * 2.0 ** -10 * 4 + slack[name][e] * (1 + 2.0 ** -4)
            assert bool(((got - truth[name][e]).abs() <= bound).all()), (name, float(((got - truth[name][e]).abs() - bound).max()))
            # scales: powers of two, and no larger than the largest magnitude since the block began asks for
            assert bool((torch.frexp(s)[0] == 0.5).all())
            for b in range((L + 15) // 16):
                most = truth[name][e][:, 16 * b:16 * b + 16].abs().amax((-1, -2))
                block = s[:, 16 * b, 0]
                assert bool((most <= 448 * block * (1 + 1e-5)).all()) and bool(((most >= 224 * block * (1 - 1e-5)) | (block <= 2.0 ** -40)).all())


def test_raised_scales_move_older_codes_without_a_second_rounding():
    """Codes that stay normal are the same values after their block's scale has risen eightfold."""
    import monarch_attention_b200 as ma
    cache = new_cache(2, 1, 64, 16)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    x = torch.linspace(1.0, 1.9, 64, device="cuda").to(torch.bfloat16).view(1, 1, 1, 64)
    ma.append_kv_b200(cache, x, x, table, torch.tensor([1], dtype=torch.int32, device="cuda"))
    first = held(cache.k, cache.k_scale, table[0], 1, 16)
    ma.append_kv_b200(cache, 8 * x, 8 * x, table, torch.tensor([2], dtype=torch.int32, device="cuda"))
    both = held(cache.k, cache.k_scale, table[0], 2, 16)
    assert torch.equal(both[:, :1], first) and torch.equal(both[:, 1:], 8 * first)
    ma.append_kv_b200(cache, 0 * x, 0 * x, table, torch.tensor([3], dtype=torch.int32, device="cuda"))   # a smaller token does not lower it
    assert torch.equal(held(cache.k, cache.k_scale, table[0], 2, 16), both)


def test_extreme_values():
    import monarch_attention_b200 as ma
    D = 64
    table = torch.tensor([[0]], dtype=torch.int32, device="cuda")
    one = torch.tensor([1], dtype=torch.int32, device="cuda")
    for fill, want in ((0.0, 0.0), (2.0 ** -100, 0.0), (3.0e38, 448 * 2.0 ** 60), (1e-9, 1e-9), (1e20, 1e20)):
        cache = new_cache(1, 1, D, 16)
        x = torch.full((1, 1, 1, D), fill, device="cuda").to(torch.bfloat16)
        ma.append_kv_b200(cache, x, -x, table, one)
        k, v = (held(c, s, table[0], 1, 16) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        want = torch.full_like(k, min(float(x[0, 0, 0, 0]), want) if want > 1e20 else float(x[0, 0, 0, 0]))
        bound = want.abs() * 2.0 ** -4 + 2.0 ** -50   # half a subnormal step of the smallest scale
        assert bool(((k - want).abs() <= bound).all()) and bool(((v + want).abs() <= bound).all())
    cache = new_cache(1, 1, D, 16)
    x = torch.ones(1, 1, 1, D, device="cuda", dtype=torch.bfloat16)
    x[..., 3], x[..., 4], x[..., 5] = float("nan"), float("inf"), float("-inf")
    ma.append_kv_b200(cache, x, x, table, one)
    k = cache.k[0, 0, 0].float()
    assert bool(torch.isnan(k[3])) and float(k[4]) == 448.0 and float(k[5]) == -448.0 and bool(torch.isfinite(k[6:]).all())
    assert float(cache.k_scale[0, 0, 0]) == 2.0 ** 60


def test_a_call_again_on_the_same_tokens_changes_nothing():
    import monarch_attention_b200 as ma
    cache = new_cache(8, 2, 128, 32)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    rotary = ma.RotaryPositions(128)
    k, v = heads(2, 2, 40, 128, torch.bfloat16, "heads", 1), heads(2, 2, 40, 128, torch.bfloat16, "heads", 2)
    lengths = torch.tensor([50, 77], dtype=torch.int32, device="cuda")
    cache.k_scale.fill_(2.0 ** -8), cache.v_scale.fill_(2.0 ** -8)
    cache.k.zero_(), cache.v.zero_()
    ma.append_kv_b200(cache, k, v, table, lengths, rotary=rotary)
    first = raw(cache)
    ma.append_kv_b200(cache, k, v, table, lengths, rotary=rotary)
    assert all(torch.equal(a, b) for a, b in zip(first, raw(cache)))


def test_unaligned_and_strided_inputs():
    import monarch_attention_b200 as ma
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    lengths = torch.tensor([21], dtype=torch.int32, device="cuda")
    wide = heads(1, 2, 21, 67, torch.bfloat16, "heads", 1)
    turned = heads(1, 2, 64, 21, torch.bfloat16, "heads", 2).transpose(-1, -2)
    rotary = ma.RotaryPositions(64)
    for x in (wide[..., 1:65], wide[..., 3:67], turned, heads(1, 1, 21, 64, torch.bfloat16, "heads", 3).expand(1, 2, 21, 64)):
        a, b = new_cache(4, 2, 64, 16), new_cache(4, 2, 64, 16)
        qa = ma.append_kv_b200(a, x, x, table, lengths, query=x, rotary=rotary)
        y = x.contiguous()
        qb = ma.append_kv_b200(b, y, y, table, lengths, query=y, rotary=rotary)
        assert all(torch.equal(s, t) for s, t in zip(raw(a), raw(b))) and torch.equal(qa, qb)


def test_bad_pages_and_lengths_are_left_out_and_reported():
    import monarch_attention_b200 as ma
    k = heads(3, 2, 4, 64, torch.bfloat16, "heads", 1)
    good = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([4, 20, 32], dtype=torch.int32, device="cuda")
    want = new_cache(6, 2, 64, 16)
    start = raw(want)
    ma.append_kv_b200(want, k, k, good, lengths)
    for table, length, counts in [([[0, 1], [2, 6], [4, 5]], [4, 20, 32], None), ([[0, 1], [2, -1], [4, 5]], [4, 20, 32], None),
                                  ([[0, 1], [2, 2 ** 31 - 1], [4, 5]], [4, 20, 32], None), (good.tolist(), [4, 3, 32], None),
                                  (good.tolist(), [4, -5, 32], None), (good.tolist(), [4, 1000, 32], [4, 4, 4]), (good.tolist(), [4, 20, 32], [4, 9, 4]),
                                  (good.tolist(), [4, 20, 32], [4, -1, 4]), (good.tolist(), [4, 2 ** 31 - 1, 32], None)]:
        cache = new_cache(6, 2, 64, 16)
        ma.append_kv_b200(cache, k, k, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(length, dtype=torch.int32, device="cuda"),
                          None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="earlier call"):
            ma.append_kv_b200(cache, k, k, good, lengths)
        for a, b, s in zip(raw(cache), raw(want), start):   # the others' tokens are there, the bad sequence's are not
            assert torch.equal(a[[0, 1, 4, 5]], b[[0, 1, 4, 5]]) and torch.equal(a[[2, 3]], s[[2, 3]])
    cache = new_cache(6, 2, 64, 16)
    ma.append_kv_b200(cache, k, k, good, lengths)   # and the next call is an ordinary one
    assert all(torch.equal(a, b) for a, b in zip(raw(cache), raw(want)))


def test_half_step_of_the_code():
    assert torch.finfo(torch.float8_e4m3fn).eps / 2 == 2.0 ** -4 and HALF_STEP[torch.float16] == 2.0 ** -11
