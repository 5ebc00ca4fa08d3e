"""The append to the 8-bit cache and the attention over it at the ends of their ranges: infinities, NaN, scales and scores far apart."""
import math

import pytest
import torch

from decoder_reference import HALF_STEP, SUBNORMAL, attention, close, held
from test_cached_attention_gpu import check, filled, queries

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("N", [1, 2, 20])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_and_nan_stay_in_features_that_are_not_rotated(D, pairs, dim, N):
    """Values, and what lies behind ``dim`` in keys and queries, are passed on feature by feature whatever is in them."""
    import monarch_attention_b200 as ma
    if dim > D:
        pytest.skip("wider than the head")
    E, H, Hk = 2, 3, 2
    rotary = ma.RotaryPositions(dim, pairs=pairs)
    q, k, v = (torch.ones(E, h, N, D, device="cuda", dtype=BF) for h in (H, Hk, Hk))
    for t, first in ((q, dim), (k, dim), (v, 0)):
        for i, x in enumerate((INF, NAN, -INF)):
            at = first + (D - first) * (2 * i + 1) // 7
            if at < D:
                t[:, i % t.shape[1], N // 2, at] = x
    cache = ma.PagedKV.allocate(8, Hk, D, 32)
    table, lengths = torch.arange(8, dtype=torch.int32, device="cuda").view(E, 4), ints(N + 3, N + 60)
    out = ma.append_kv_b200(cache, k, v, table, lengths, query=q, rotary=rotary)
    assert bool(((out == q) | (out.isnan() & q.isnan()))[..., dim:].all()) and bool(out[..., :dim].isfinite().all())
    for codes, x, first in ((cache.k, k, dim), (cache.v, v, 0)):
        for e in range(E):
            place = torch.arange(int(lengths[e]) - N, int(lengths[e]), device="cuda")
            got = codes.view(torch.uint8)[table[e].long()[place // 32], :, place % 32].view(torch.float8_e4m3fn).float().transpose(0, 1)
            assert torch.equal(got.isnan(), x[e].isnan())
            assert bool((got[x[e] == INF] == 448.0).all()) and bool((got[x[e] == -INF] == -448.0).all())


@pytest.mark.parametrize("N", [1, 2, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_a_row_of_nan_leaves_the_others_of_its_block(D, N):
    """A block's scale is that of its numbers: a token that is NaN throughout is stored as that, and the tokens beside it keep their values."""
    import monarch_attention_b200 as ma
    cache = ma.PagedKV.allocate(4, 2, D, 16)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    x = torch.linspace(1.0, 1.75, 8, device="cuda").to(BF).repeat(D // 8).expand(1, 2, 5, D).contiguous()
    ma.append_kv_b200(cache, x, -x, table, ints(5))
    bad = x[:, :, :1].expand(1, 2, N, D).clone()
    bad[:, 1, N // 2] = NAN
    ma.append_kv_b200(cache, bad, -bad, table, ints(5 + N))
    alone = ma.PagedKV.allocate(4, 2, D, 16)
    ma.append_kv_b200(alone, torch.full_like(x[:, :, :1], NAN), torch.full_like(x[:, :, :1], NAN), table, ints(1))
    for codes, scales, sign in ((cache.k, cache.k_scale, 1.0), (cache.v, cache.v_scale, -1.0)):
        got = held(codes, scales, table[0], 5 + N, 16)
        want = sign * torch.cat((x, bad), 2)[0].to(torch.float8_e4m3fn).double().cpu()   # (the scale is a power of two, so the rounding is the type's)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    # with nothing but NaN the smallest scale of all, which the next token raises as far as it asks for
    assert float(alone.k_scale[0, 0, 0]) == 2.0 ** -40 and bool(alone.k[0, 0, 0].float().isnan().all())


@pytest.mark.parametrize("place", range(16))
@pytest.mark.parametrize("N,softcap", [(1, 0.0), (5, 0.0), (40, 0.0), (40, 20.0)])
def test_a_key_of_nan_reaches_all_rows_that_see_it(N, softcap, place):
    """Whichever of a block's 16 places it has, and however many rows there are; rows in front of it do not see it."""
    import monarch_attention_b200 as ma
    L, D, page = 300, 64, 32
    cache, table = filled(2, 12, 2, D, page, [L, L])
    spots = (160 + place, L - N // 2 - 1 if N > 1 else 3)   # in the middle; among the call's own tokens
    for e, t in enumerate(spots):
        cache.k.view(torch.uint8)[int(table[e, t // page]), :, t % page, 7] = 0x7f
    q = queries(2, 8, N, D, BF, "heads")
    out = ma.cached_attention_b200(q, cache, table, ints(L, L), softcap=softcap)
    for e, t in enumerate(spots):
        sees = torch.arange(L - N, L) >= t
        assert bool(out[e][:, sees.cuda()].isnan().all())
        if not sees.all():
            k, v = (held(c, s, table[e], L, page) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            n = int((~sees).sum())
            want, bound = attention(q[e, :, :n], k[:, :t], v[:, :t], L - N, True, D ** -0.5, softcap)
            close(out[e, :, :n], want, bound + HALF_STEP[BF] * (want.abs() + bound) + SUBNORMAL[BF])


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [3, 40])
def test_a_query_of_nan_or_infinity_is_its_own_rows_matter(N, dtype, bad):
    import monarch_attention_b200 as ma
    cache, table = filled(1, 8, 2, 128, 64, [400])
    q = queries(1, 4, N, 128, dtype, "heads")
    want = ma.cached_attention_b200(q, cache, table, ints(400))
    broken = q.clone()
    broken[0, 1, N // 2, 70] = bad
    out = ma.cached_attention_b200(broken, cache, table, ints(400))
    assert bool(out[0, 1, N // 2].isnan().all())   # (of scores of plus and minus infinity, or NaN)
    rest = torch.ones(1, 4, N, dtype=torch.bool, device="cuda")
    rest[0, 1, N // 2] = False
    assert bool(out[rest].isfinite().all())
    # (the other rows of its tile may get another reference and so other roundings of their weights: 2^-11 and the type's)
    assert bool(((out[rest].float() - want[rest].float()).abs() <= 2 ** -10 * 16 + 2 * HALF_STEP[dtype] * want[rest].float().abs()).all())


def one_hot_keys(L, D, page, far):
    """A cache of keys that give scores of 0 (an early token, of value 0) and ``-far`` in units of log2 (all others, of value 1) to the query (1, 0, ..)."""
    import monarch_attention_b200 as ma
    pages = -(-L // page)
    cache = ma.PagedKV.allocate(pages, 1, D, page)
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    raw = cache.k.view(torch.uint8)
    raw[..., 0] = 0xb8                     # -1
    raw[0, :, 5, 0] = 0
    cache.v.view(torch.uint8).fill_(0x38)  # 1
    cache.v.view(torch.uint8)[0, :, 5] = 0
    return cache, torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages), far * math.log(2.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("E,N", [(1, 1), (1, 40), (1000, 1), (500, 5), (160, 40)])
@pytest.mark.parametrize("L,far", [(131071, 25.1), (131071, 24.4), (60000, 25.0), (60000, 27.0), (3000, 22.6), (3000, 26.0)])
def test_a_long_tail_of_small_weights_is_not_lost(L, far, E, N, dtype):
    """One key far above all others, whose values are what the result has: tail / (1 + tail), tail = (L - 1) 2^-far.

    The largest weight is 2^7 at least, so that those of the tail are 2^(7 - far) or more and rounded to 2^-25: 2^(far - 32) of themselves, 2^-11 at normal
    weights.  An addend to a 32-bit sum of products loses up to 2^-25 of the sum: L 2^-25 of it, and sums of weights L 2^-24 of the tail."""
    import monarch_attention_b200 as ma
    cache, table, scale = one_hot_keys(L, 64, 128, far)
    q = torch.zeros(E, 4, N, 64, dtype=dtype, device="cuda")   # (many sequences over the same pages: a head stays with one CTA)
    q[..., 0] = 1.0
    out = ma.cached_attention_b200(q, cache, table.expand(E, -1), ints(*[L] * E), causal=False, scale=scale)
    tail = (L - 1) * 2.0 ** -far
    want = tail / (1 + tail)
    bound = want * (2.0 ** (far - 32) + 2.0 ** -11 + L * 2.0 ** -24)
    close(out, torch.full((E, 4, N, 64), want, dtype=torch.float64), torch.tensor(bound + HALF_STEP[dtype] * (want + bound) + SUBNORMAL[dtype]))


def one_hot(q, k, v, first, scale, softcap=0.0):
    """Values of the best key of each row, and whether it stands so far above the others that nothing else counts, whatever 32-bit sums do to scores."""
    q, D = q.double().cpu(), q.shape[-1]
    k, v = (t.repeat_interleave(q.shape[0] // t.shape[0], 0) for t in (k, v))
    s, size = q @ k.mT * scale, q.abs() @ k.abs().mT * abs(scale)
    if softcap:
        s, size = softcap * torch.tanh(s / softcap), size + softcap
    seen = torch.arange(k.shape[1]) <= first + torch.arange(q.shape[1])[:, None]
    top, best = s.masked_fill(~seen, -math.inf).topk(2, -1)
    # (D + 8) 2^-24 of the sum of magnitudes each, D 2^-25 more of a row brought to f16; 100 more is 2^-144 of the weight
    clear = top[..., 0] - top[..., 1] > 2 * (1.5 * D + 8) * 2.0 ** -24 * size.amax(-1) + 100
    return v.gather(1, best[..., :1].expand(-1, -1, D)), clear


@pytest.mark.parametrize("dtype,size", [(BF, 3e4), (BF, 1e8), (BF, 1e20), (BF, 1e30), (HF, 3e2), (HF, 6e4 / 5)])
@pytest.mark.parametrize("N", [1, 20, 80])
@pytest.mark.parametrize("scale", [128 ** -0.5, 1e4])
@pytest.mark.parametrize("L", [300, 5000])
def test_scores_of_any_magnitude(L, scale, N, dtype, size):
    """Scores that decide for one key give that key's value, with few rows and with many, keys in one piece or in several."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, L // 64 + 2, 1, 128, 64, [L])
    q = (queries(1, 8, N, 128, torch.float32, "heads").clamp(-5, 5) * size).to(dtype)
    out = ma.cached_attention_b200(q, cache, table, ints(L), scale=scale)[0].double().cpu()
    k, v = (held(c, s, table[0], L, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, clear = one_hot(q[0], k, v, L - N, scale)
    assert bool(clear.any()) and bool(out.isfinite().all())
    # the weight in f16, its sum in 32 bits and the rounding of the result
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -20 + HALF_STEP[dtype]) * want.abs() + SUBNORMAL[dtype])[clear].all())
    # what is not clear lies between the values
    most, least = v.amax((0, 1)), v.amin((0, 1))
    assert bool((out <= most + 2.0 ** -7 * most.abs()).all()) and bool((out >= least - 2.0 ** -7 * least.abs()).all())


@pytest.mark.parametrize("softcap", [1e5, 1e9, 1e30])
@pytest.mark.parametrize("N", [1, 20, 80])
def test_large_caps_of_large_scores(N, softcap):
    import monarch_attention_b200 as ma
    cache, table = filled(1, 6, 1, 128, 64, [300])
    q = (queries(1, 8, N, 128, BF, "heads").float() * softcap / 10).to(BF)
    out = ma.cached_attention_b200(q, cache, table, ints(300), scale=0.1, softcap=softcap)[0].double().cpu()
    k, v = (held(c, s, table[0], 300, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, clear = one_hot(q[0], k, v, 300 - N, 0.1, softcap)
    assert bool(clear.any()) and bool(out.isfinite().all())
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) * want.abs())[clear].all())


@pytest.mark.parametrize("exponent", [-20, -30, -39, 0, 50])
@pytest.mark.parametrize("N", [1, 3, 4, 20, 40])
@pytest.mark.parametrize("L", [300, 5000])
def test_zero_scales_beside_values_of_any_size(L, N, exponent):
    """Blocks of scale zero hold zeros; the others' values count in full beside them, however small they are."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, L // 64 + 2, 2, 64, 64, [L])
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.v_scale.fill_(2.0 ** exponent)
    cache.v_scale[torch.rand(cache.v_scale.shape, generator=g, device="cuda") < 0.5] = 0.0
    q = queries(1, 8, N, 64, BF, "heads")
    check(ma.cached_attention_b200(q, cache, table, ints(L)), q, cache, table, [L], None, 64)


@pytest.mark.parametrize("N,exponents", [(N, e) for N in (20, 40) for e in ((-40, -40), (60, 60), (-40, 60), (-30, -20), (10, 30))] +
                         [(N, e) for N in (1, 3, 4) for e in ((-14, -14), (15, 15), (-14, 15))])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("L", [300, 5000])
def test_large_scores_over_values_of_other_scales(L, size, N, exponents):
    """A value's scale is a part of its weight, however far beyond it the scores are: any scale with many rows, 2^-14 to 2^15 with few."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, L // 64 + 2, 1, 64, 64, [L])
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.v_scale.copy_(torch.exp2(torch.randint(exponents[0], exponents[1] + 1, cache.v_scale.shape, generator=g, device="cuda").float()))
    q = (queries(1, 8, N, 64, BF, "heads").float() * size).to(BF)
    out = ma.cached_attention_b200(q, cache, table, ints(L))[0].double().cpu()
    k, v = (held(c, s, table[0], L, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, clear = one_hot(q[0], k, v, L - N, 0.125)
    assert bool(clear.any()) and bool(out.isfinite().all())
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) * want.abs())[clear].all())


@pytest.mark.parametrize("N", [1, 3, 4, 20, 40])
@pytest.mark.parametrize("L", [200, 5000])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 20, 2.0 ** 30, 2.0 ** 100])
def test_equal_keys_share_the_weight_whatever_the_scores(size, L, N):
    """All keys are one and the same, so the result is the mean of the values, and the scales of the blocks are apart.

    Weights are equal, so each is as far off as another; 2^-11 of a weight in f16, L 2^-24 of the largest value, sums 2^-20."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, L // 64 + 2, 1, 64, 64, [L])
    cache.k_scale.fill_(0.25)
    cache.k.view(torch.uint8).fill_(0x38)
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.v_scale.copy_(torch.exp2(torch.randint(-6, 7, cache.v_scale.shape, generator=g, device="cuda").float()))
    q = torch.full((1, 4, N, 64), size, dtype=BF, device="cuda")
    q[:, 1] *= -1
    out = ma.cached_attention_b200(q, cache, table, ints(L), causal=False)[0]
    v = held(cache.v, cache.v_scale, table[0], L, 64)[0]
    bound = (2.0 ** -11 + 2.0 ** -20) * v.abs().mean(0) + 2.0 ** -24 * v.abs().amax()
    close(out, v.mean(0).expand(4, N, 64), bound + 2.0 ** -8 * (v.mean(0).abs() + bound))


@pytest.mark.parametrize("e", range(18, 28))
@pytest.mark.parametrize("delta", [8.0, 14.0, 15.0, 15.5, 16.0, 17.0, 24.0])
@pytest.mark.parametrize("N", [1, 3, 40])
def test_a_little_above_the_reference_at_large_scores(N, delta, e):
    """Later keys that are 2^delta above earlier ones, at scores of 2^e where the last bit of a 32-bit score is 2^(e - 23): weights stay in f16.

    In units of log2 all scores are off by that bit, so the earlier keys' share of 2^-delta by a factor of two to it; values are 1 and 2."""
    import monarch_attention_b200 as ma
    L, D = 512, 64
    cache = ma.PagedKV.allocate(8, 1, D, 64)
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    k[..., 0] = 0x38          # 1: 2^e to all
    k[4:, :, :, 1] = 0x38     # and delta to the later half
    v[:4], v[4:] = 0x38, 0x40
    q = torch.zeros(1, 4, N, D, dtype=BF, device="cuda")
    q[..., 0], q[..., 1] = 2.0 ** e, delta
    out = ma.cached_attention_b200(q, cache, torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8), ints(L), causal=False, scale=math.log(2.0))
    out = out.double().cpu()
    assert bool(out.isfinite().all())
    least, most = (2 - 1 / (1 + 2.0 ** x) for x in (delta - 2.0 ** (e - 22), delta + 2.0 ** (e - 22)))
    slack = 2.0 ** -8 * 2 + 2.0 ** -10
    assert bool((out >= least - slack).all()) and bool((out <= most + slack).all())


@pytest.mark.parametrize("size", [1e33, 1e35, 1e36])
@pytest.mark.parametrize("N", [1, 3, 4, 20, 40])
def test_queries_near_the_end_of_32_bits(N, size):
    """bf16 goes to 3e38: rows are brought to f16 by their own exponent whatever it is, as long as the scores are numbers of 32 bits."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, 6, 1, 128, 64, [300])
    q = (queries(1, 8, N, 128, BF, "heads").float() * size).to(BF)
    out = ma.cached_attention_b200(q, cache, table, ints(300))[0].double().cpu()
    k, v = (held(c, s, table[0], 300, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, clear = one_hot(q[0], k, v, 300 - N, 128 ** -0.5)
    assert bool(clear.any()) and bool(out.isfinite().all())
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) * want.abs())[clear].all())


def test_an_append_is_a_change_of_the_pool():
    """A backward pass that needs what the pool held before says so, as after any operation in place."""
    import monarch_attention_b200 as ma
    cache = ma.PagedKV.allocate(2, 1, 64, 16)
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    k = queries(1, 1, 1, 64, BF, "heads")
    w = torch.ones_like(cache.v_scale).requires_grad_(True)
    y = (w * cache.v_scale).sum()
    before = [t._version for t in cache]
    with torch.no_grad():
        ma.append_kv_b200(cache, k, k, table, ints(1))
    assert all(t._version > n for t, n in zip(cache, before))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        pool = ma.PagedKV.allocate(2, 1, 64, 16)
        ma.append_kv_b200(pool, k, k, table, ints(1))
    assert torch.equal(pool.k.view(torch.uint8), cache.k.view(torch.uint8)) and torch.equal(pool.k_scale, cache.k_scale)


@pytest.mark.parametrize("part", ["k_scale", "v_scale"])
def test_a_pool_that_requires_a_gradient_is_refused(part):
    import monarch_attention_b200 as ma
    cache = ma.PagedKV.allocate(2, 1, 64, 16)
    cache = cache._replace(**{part: getattr(cache, part).clone().requires_grad_(True)})
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    k = queries(1, 1, 1, 64, BF, "heads")
    for call in (lambda: ma.append_kv_b200(cache, k, k, table, ints(1)), lambda: ma.cached_attention_b200(k, cache, table, ints(1))):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("softcap", [1e-50, -1e-50, 1e-21, -1.0, 1e31, NAN])
def test_caps_that_would_be_none_in_32_bits_are_refused(softcap):
    import monarch_attention_b200 as ma
    cache, table = filled(1, 2, 1, 64, 16, [20])
    with pytest.raises(ValueError, match="softcap"):
        ma.cached_attention_b200(queries(1, 1, 1, 64, BF, "heads"), cache, table, ints(20), softcap=softcap)


@pytest.mark.parametrize("N,H", [(4, 4), (40, 4)])
def test_a_result_in_a_buffer_with_the_query(N, H):
    """In its place or beside it, row for row, it is taken; over rows that others still read it is refused, whatever the strides are."""
    import monarch_attention_b200 as ma
    L, D = 300, 64
    cache, table = filled(2, 6, 2, D, 64, [L, L])
    n = ints(L, L)
    whole = torch.zeros(2 * (N + 1) * 3 * H * D + N * D, dtype=BF, device="cuda")
    buffer = whole[:2 * (N + 1) * 3 * H * D].view(2, N + 1, 3, H, D)
    buffer[:, :N, 0] = queries(2, H, N, D, BF, "heads").transpose(1, 2)
    part = lambda i, first=0: buffer[:, first:first + N, i].transpose(1, 2)   # noqa: E731
    q = part(0)
    want = ma.cached_attention_b200(q, cache, table, n)
    for bad in (part(0, 1), part(0).transpose(1, 2) if N == H else part(0, 1), buffer.view(2, -1)[:, H * D // 2:].as_strided(q.shape, q.stride()),
                buffer.as_strided(q.shape, (q.stride(0), D, 3 * H * D + D, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ma.cached_attention_b200(q, cache, table, n, out=bad)
    with pytest.raises(ValueError, match="overlap"):   # rows of the result over one another
        ma.cached_attention_b200(q, cache, table, n, out=torch.zeros(2 * H * N * D, dtype=BF, device="cuda").as_strided(q.shape, (H * N * D // 2, N * D // 2, D // 2, 1)))
    for i in (1, 2, 0):
        assert torch.equal(ma.cached_attention_b200(q, cache, table, n, out=part(i)), want)
        assert not bool(buffer[:, N].any())
    assert torch.equal(part(1), want) and torch.equal(part(2), want)


def test_pools_whose_parts_are_over_one_another_are_not_written():
    import monarch_attention_b200 as ma
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    k = queries(1, 2, 20, 64, BF, "heads")
    good = ma.PagedKV.allocate(4, 2, 64, 32)
    byte, e4m3 = torch.uint8, torch.float8_e4m3fn
    for bad in (dict(v=good.k), dict(v_scale=good.k_scale), dict(k=good.k[:1].expand(4, 2, 32, 64)), dict(v=good.v[:, :1].expand(4, 2, 32, 64)),
                dict(k_scale=good.k_scale[:, :1].expand(4, 2, 2)), dict(k=good.k.view(byte).view(-1).as_strided((4, 2, 32, 64), (4096, 1024, 64, 1)).view(e4m3)),
                dict(k=good.k[:3], v=good.k[1:], k_scale=good.k_scale[:3], v_scale=good.v_scale[:3])):
        with pytest.raises(ValueError, match="overlap"):
            ma.append_kv_b200(good._replace(**bad), k, k, table, ints(20))
    # one buffer for keys and values, page by page or token by token, is a pool like any other; reading shared pages is, too
    ma.append_kv_b200(good, k, -k, table, ints(20))
    q = queries(1, 4, 1, 64, BF, "heads")
    want = ma.cached_attention_b200(q, good, table, ints(20))
    for codes, scales in ((torch.zeros(4, 2, 2, 32, 64, dtype=byte, device="cuda").view(e4m3).unbind(1), torch.zeros(4, 2, 2, 2, device="cuda").unbind(1)),
                          ([t.permute(0, 2, 1, 3) for t in torch.zeros(4, 32, 2, 2, 64, dtype=byte, device="cuda").view(e4m3).unbind(2)],
                           torch.zeros(2, 4, 2, 2, device="cuda").unbind(0))):
        pool = ma.PagedKV(*codes, *scales)
        ma.append_kv_b200(pool, k, -k, table, ints(20))
        assert torch.equal(ma.cached_attention_b200(q, pool, table, ints(20)), want)
    ma.cached_attention_b200(q, good._replace(v=good.k), table, ints(20))


@pytest.mark.parametrize("E,Hk,N,L,D", [(1, 2, 40, 300, 64), (2, 4, 100, 5000, 128), (40, 4, 300, 600, 64)])
def test_a_wait_that_runs_out_ends_the_call_and_is_reported(E, Hk, N, L, D):
    """Many rows, with keys in one piece and in several: the values of each block of threads' first step never arrive.  All end by themselves, the next call
    raises, and the one after is an ordinary call."""
    import ctypes as C

    from monarch_attention_b200 import _cabi
    import monarch_attention_b200 as ma
    lib, H, page = _cabi.load(), 4 * Hk, 64
    cache, table = filled(E, L // page + 1, Hk, D, page, [L] * E)
    q, n = queries(E, H, N, D, BF, "heads"), ints(*[L] * E)
    good = ma.cached_attention_b200(q, cache, table, n)
    out = torch.empty_like(q)
    p = _cabi.Attend(_cabi.ABI_VERSION, E, H, N, _cabi.BF16, 1, 0, D ** -0.5, 0.0)
    p.q, p.out = (_cabi.Tensor4(t.data_ptr(), *t.stride()[:3]) for t in (q, out))
    p.cache = _cabi.Cache(*(t.data_ptr() for t in cache), *cache.k.shape, *cache.k.stride()[:3], *cache.v.stride()[:3], *cache.k_scale.stride()[:2],
                          *cache.v_scale.stride()[:2])
    p.sequences = _cabi.Sequences(table.data_ptr(), table.stride(0), table.shape[1], n.data_ptr(), None)
    ws = torch.empty(lib.ma_b200_cache_attend_workspace_bytes(C.byref(p)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ma_b200_cache_attend(C.byref(p), ws.data_ptr(), ws.numel(), stream) == _cabi.OK
    assert torch.equal(out, good) and lib.ma_b200_poll_device_status(0) == _cabi.OK
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    assert lib.ma_b200_selftest_attend_wait_expiry(C.byref(p), ws.data_ptr(), ws.numel(), stream) == _cabi.OK
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 2000   # (waits of 4096 tries, a round of blocks after another)
    with pytest.raises(RuntimeError, match="gave up"):
        ma.cached_attention_b200(q, cache, table, n)
    assert lib.ma_b200_poll_device_status(0) == _cabi.OK
    assert torch.equal(ma.cached_attention_b200(q, cache, table, n), good)


def test_results_of_no_tokens():
    import monarch_attention_b200 as ma
    cache, table = filled(2, 2, 2, 64, 16, [20, 3])
    q = torch.empty_strided((2, 4, 0, 64), (0, 0, 0, 1), dtype=BF, device="cuda")
    out = ma.cached_attention_b200(q, cache, table, ints(20, 3), out=q)
    assert out.shape == q.shape and ma.append_kv_b200(cache, q[:, :2], q[:, :2], table, ints(20, 3)) is None


@pytest.mark.parametrize("exponents", [(-40, -40), (60, 60), (-40, 60), (-30, -20)])
@pytest.mark.parametrize("N", [1, 3, 4])
@pytest.mark.parametrize("size", [1e4, 1e5, 1e6, 1e7])
def test_few_rows_with_scores_below_their_limit_over_values_of_any_scale(size, N, exponents):
    import monarch_attention_b200 as ma
    cache, table = filled(1, 6, 1, 64, 64, [300])
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.v_scale.copy_(torch.exp2(torch.randint(exponents[0], exponents[1] + 1, cache.v_scale.shape, generator=g, device="cuda").float()))
    q = (queries(1, 8, N, 64, BF, "heads").float() * size).to(BF)
    out = ma.cached_attention_b200(q, cache, table, ints(300))[0].double().cpu()
    k, v = (held(c, s, table[0], 300, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, clear = one_hot(q[0], k, v, 300 - N, 0.125)
    assert bool(clear.any()) and bool(out.isfinite().all())
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) * want.abs())[clear].all())
