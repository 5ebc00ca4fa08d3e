"""Attention over the paged 8-bit cache against the definition in 64 bits."""
import pytest
import torch

from decoder_reference import HALF_STEP, SUBNORMAL, attention, close, held

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def filled(E, per, Hk, D, page, lengths, layout="heads", seed=0, spare=2):
    """A pool whose sequences have random tokens, and NaN in all else."""
    import monarch_attention_b200 as ma
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = E * per + spare
    table = torch.randperm(pages, generator=g, device="cuda")[:E * per].view(E, per).to(torch.int32)
    parts = []
    for _ in range(2):
        x = torch.randn(pages, Hk, page, D, generator=g, device="cuda") * 1.5 + 0.5 * torch.randn(1, Hk, 1, D, generator=g, device="cuda")
        x = x * 2.0 ** torch.randint(-2, 3, (pages, Hk, page // 16, 1, 1), generator=g, device="cuda").expand(-1, -1, -1, 16, -1).reshape(pages, Hk, page, 1)
        s = torch.exp2(torch.ceil(torch.log2(x.view(pages, Hk, page // 16, 16, D).abs().amax((-1, -2)) / 448)))
        codes = (x / s.repeat_interleave(16, -1)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        alive = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for e in range(E):
            p = torch.arange(int(lengths[e]), device="cuda")
            alive[table[e].long()[p // page], p % page] = True
        codes = torch.where(alive[:, None, :, None], codes, torch.full_like(codes, 0x7f))
        s = torch.where(alive.view(pages, 1, page // 16, 16).any(-1), s, torch.full_like(s, float("nan")))
        if layout == "tokens":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
        parts.append((codes.view(torch.float8_e4m3fn), s))
    return ma.PagedKV(parts[0][0], parts[1][0], parts[0][1], parts[1][1]), table


def queries(E, H, N, D, dtype, layout, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn((E, N, H, D) if layout == "tokens" else (E, H, N, D), generator=g, device="cuda").to(dtype)
    return t.permute(0, 2, 1, 3) if layout == "tokens" else t


def check(out, q, cache, table, lengths, counts, page, causal=True, scale=None, softcap=0.0, window=0):
    E, H, N, D = q.shape
    assert out.shape == q.shape and out.dtype == q.dtype
    for e in range(E):
        L, n = int(lengths[e]), N if counts is None else int(counts[e])
        assert not bool(out[e, :, n:].any()), "rows of padding are zero"
        if n == 0:
            continue
        k, v = held(cache.k, cache.k_scale, table[e], L, page), held(cache.v, cache.v_scale, table[e], L, page)
        want, bound = attention(q[e, :, :n], k, v, L - n, causal, D ** -0.5 if scale is None else scale, softcap, window)
        close(out[e, :, :n], want, bound + HALF_STEP[q.dtype] * (want.abs() + bound) + SUBNORMAL[q.dtype], f"sequence {e} of {L} tokens")


CASES = [  # E, H, Hk, N, D, page, lengths, counts
    (1, 1, 1, 1, 64, 16, [1], None), (1, 1, 1, 1, 128, 16, [2], None), (2, 4, 4, 1, 64, 16, [16, 17], None), (3, 8, 8, 1, 128, 32, [31, 32, 33], None),
    (5, 12, 12, 1, 64, 64, [1, 127, 128, 129, 500], None), (4, 8, 1, 1, 128, 64, [100, 1000, 7, 255], None), (3, 40, 8, 1, 128, 16, [257, 64, 300], None),
    (2, 12, 2, 3, 64, 32, [40, 333], None), (3, 4, 2, 5, 128, 128, [5, 600, 129], [5, 3, 0]), (2, 8, 2, 9, 64, 16, [9, 200], [2, 9]),
    (2, 6, 3, 40, 128, 64, [40, 170], [33, 40]), (1, 16, 2, 70, 64, 32, [100], None), (1, 3, 1, 128, 128, 16, [700], None),
    (150, 2, 1, 1, 64, 16, list(range(0, 150)), None), (1, 16, 2, 1, 128, 128, [9001], None), (1, 2, 2, 1, 64, 256, [20000], None),
    (2, 64, 1, 2, 128, 16, [50, 3], None), (1, 8, 8, 300, 64, 16, [300], None)]


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_matches_the_definition(case, causal, dtype, layout):
    import monarch_attention_b200 as ma
    E, H, Hk, N, D, page, lengths, counts = CASES[case]
    per = max(lengths) // page + 2
    cache, table = filled(E, per, Hk, D, page, lengths, layout, seed=case)
    q = queries(E, H, N, D, dtype, layout)
    dev = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts)]
    out = ma.cached_attention_b200(q, cache, table, *dev, causal=causal, token_major_output=layout == "tokens")
    assert out.transpose(1, 2).is_contiguous() if layout == "tokens" else out.is_contiguous()
    check(out, q, cache, table, lengths, counts, page, causal)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N,window,softcap,scale", [(1, 1, 0.0, None), (1, 100, 0.0, None), (1, 128, 20.0, 0.3), (7, 1, 0.0, None), (7, 33, 5.0, None), (1, 0, 30.0, 0.5),
                                                    (60, 40, 0.0, None), (60, 300, 15.0, None), (2, 10 ** 9, 0.0, -0.1)])
@pytest.mark.parametrize("Hk,D", [(2, 64), (4, 128)])
def test_windows_caps_and_scales(Hk, D, N, window, softcap, scale, dtype):
    import monarch_attention_b200 as ma
    lengths, page = [N, 333, 1025, 150], 32
    counts = [N, max(N - 3, 1), 0, N] if N > 1 else None
    cache, table = filled(4, 40, Hk, D, page, lengths)
    q = queries(4, 8, N, D, dtype, "tokens")
    dev = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts)]
    out = ma.cached_attention_b200(q, cache, table, *dev, scale=scale, softcap=softcap, window=window)
    check(out, q, cache, table, lengths, counts, page, True, scale, softcap, window)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("E,H,Hk,N,D,page,lengths,counts,causal,window,softcap,scale", [
    (1, 4, 1, 64, 128, 64, [5000], None, True, 0, 0.0, None), (2, 8, 2, 33, 64, 32, [3000, 40], [33, 5], True, 0, 0.0, None),
    (1, 2, 2, 130, 128, 128, [4100], None, False, 0, 10.0, None), (2, 6, 1, 90, 64, 16, [2500, 1], [90, 1], True, 700, 0.0, None),
    (1, 1, 1, 600, 128, 64, [600], None, True, 0, 0.0, None), (3, 5, 1, 257, 64, 64, [257, 2000, 300], [257, 0, 100], True, 0, 0.0, -0.2),
    (1, 8, 8, 1100, 64, 64, [1100], None, True, 33, 0.0, None), (1, 3, 1, 77, 128, 32, [1023], None, True, 0, 0.0, 0.0)])
def test_prompts(E, H, Hk, N, D, page, lengths, counts, causal, window, softcap, scale, dtype):
    """Many rows: one tile or two of them, keys in one piece or several, sequences of one token, without tokens, or shorter than the rest."""
    import monarch_attention_b200 as ma
    cache, table = filled(E, max(lengths) // page + 2, Hk, D, page, lengths, "tokens")
    q = queries(E, H, N, D, dtype, "tokens")
    dev = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts)]
    out = ma.cached_attention_b200(q, cache, table, *dev, causal=causal, window=window, softcap=softcap, scale=scale)
    check(out, q, cache, table, lengths, counts, page, causal, scale, softcap, window)


@pytest.mark.parametrize("N", [1, 20, 80])
def test_blocks_of_other_quantisers(N):
    """Scales that are no powers of two, and zero (with codes that are not): what counts is code * scale."""
    import monarch_attention_b200 as ma
    cache, table = filled(2, 6, 2, 128, 64, [300, 90 + N])
    g = torch.Generator(device="cuda").manual_seed(4)
    for s in (cache.k_scale, cache.v_scale):
        s.mul_(0.6 + torch.rand(s.shape, generator=g, device="cuda"))
        s[torch.rand(s.shape, generator=g, device="cuda") < 0.3] = 0.0
    q = queries(2, 8, N, 128, BF, "heads")
    lengths = [300, 90 + N]
    out = ma.cached_attention_b200(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check(out, q, cache, table, lengths, None, 64)


def test_more_queries_than_keys_leaves_the_first_rows_empty():
    """Tokens at positions before the sequence's first see nothing and are zero."""
    import monarch_attention_b200 as ma
    cache, table = filled(2, 2, 2, 64, 16, [3, 0])
    q = queries(2, 4, 5, 64, BF, "heads")
    out = ma.cached_attention_b200(q, cache, table, torch.tensor([3, 0], dtype=torch.int32, device="cuda"))
    assert not bool(out[0, :, :2].any()) and not bool(out[1].any())
    k, v = (held(c, s, table[0], 3, 16) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, bound = attention(q[0], k, v, -2, True, 64 ** -0.5)
    close(out[0, :, 2:], want[:, 2:], bound[:, 2:] + 2.0 ** -8 * (want[:, 2:].abs() + bound[:, 2:]))


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 3e4, 1e30])
def test_queries_of_any_magnitude(size):
    """bf16 rows are brought into the range of f16 by a power of two; scores that decide for one key are exact."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, 5, 1, 128, 64, [300])
    q = (queries(1, 8, 1, 128, BF, "heads").float() * size).to(BF)
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    out = ma.cached_attention_b200(q, cache, table, lengths)
    if size <= 1.0:
        check(out, q, cache, table, [300], None, 64)
        return
    k, v = (held(c, s, table[0], 300, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    best = (q[0, :, 0].double().cpu() @ k[0].T).argmax(-1)
    assert torch.equal(out[0, :, 0].cpu(), v[0][best].to(BF))


def test_blocks_whose_values_are_zero_or_far_apart():
    import monarch_attention_b200 as ma
    lengths = torch.tensor([64], dtype=torch.int32, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    for tops in ([0.0, 1.0, 0.0, 0.0], [0.0] * 4, [1e30, 1.0, 1e-10, 0.0], [2.0 ** -40, 2.0 ** 40, 1.0, 1.0]):
        cache = ma.PagedKV.allocate(4, 1, 64, 16)
        g = torch.Generator(device="cuda").manual_seed(1)
        k = torch.randn(1, 1, 64, 64, generator=g, device="cuda").to(BF)
        v = (torch.randn(1, 1, 64, 64, generator=g, device="cuda") * torch.tensor(tops, device="cuda").repeat_interleave(16)[:, None]).to(BF)
        ma.append_kv_b200(cache, k, v, table, lengths)
        q = queries(1, 1, 1, 64, BF, "heads")
        check(ma.cached_attention_b200(q, cache, table, lengths), q, cache, table, [64], None, 16)


def test_steps_of_a_decoder_agree_with_the_whole_at_once():
    """A prompt in pieces and tokens one at a time, through the module, give what one call over the whole gives, to rounding."""
    import monarch_attention_b200 as ma
    E, H, Hk, D, page, total = 3, 8, 2, 128, 32, 90
    rotary = ma.RotaryPositions(D, scaling="linear", factor=2.0)
    module = ma.CachedAttention(rotary)
    table = torch.randperm(3 * 4, generator=torch.Generator().manual_seed(0)).view(3, 4).to(torch.int32).cuda()
    q, k, v = (queries(E, h, total, D, BF, "tokens", seed=s) for s, h in ((1, H), (2, Hk), (3, Hk)))
    caches = [ma.PagedKV.allocate(12, Hk, D, page) for _ in range(2)]
    whole = module(q, k, v, caches[0], table, torch.full((E,), total, dtype=torch.int32, device="cuda"))
    at, parts = 0, []
    for n in [33, 16, 1, 1, 7] + [1] * 32:
        lengths = torch.full((E,), at + n, dtype=torch.int32, device="cuda")
        parts.append(module(q[:, :, at:at + n], k[:, :, at:at + n], v[:, :, at:at + n], caches[1], table, lengths))
        at += n
    assert at == total
    # codes of a block filled over several calls may differ in the subnormal range; both results are held to the same cache's definition
    turned = ma.rotary_b200(q, None, rotary)[0]
    for out, cache in ((whole, caches[0]), (parts[-1], caches[1])):
        n = out.shape[2]
        check(out, turned[:, :, total - n:], cache, table, [total] * E, None, page)
    assert torch.allclose(torch.cat(parts, 2).float(), whole.float(), atol=0.15)


def test_cross_attention_through_the_module():
    import monarch_attention_b200 as ma
    cache, table = filled(2, 4, 4, 64, 64, [200, 77])
    q = queries(2, 4, 3, 64, HF, "tokens")
    module = ma.CachedAttention(causal=False)
    module.token_major_output = True
    out = module(q, None, None, cache, table, torch.tensor([200, 77], dtype=torch.int32, device="cuda"))
    check(out, q, cache, table, [200, 77], None, 64, causal=False)
    assert out.transpose(1, 2).is_contiguous()
    with pytest.raises(ValueError):
        module(q, q, None, cache, table, torch.tensor([200, 77], dtype=torch.int32, device="cuda"))


def test_beams_share_a_prefix():
    """Sequences whose tables name the same pages read the same keys."""
    import monarch_attention_b200 as ma
    cache, table = filled(1, 5, 2, 64, 32, [150])
    q = queries(4, 4, 1, 64, BF, "heads")
    lengths = torch.full((4,), 150, dtype=torch.int32, device="cuda")
    out = ma.cached_attention_b200(q, cache, table.expand(4, -1), lengths)
    check(out, q, cache, table.expand(4, -1), [150] * 4, None, 32)


def test_out_aligned_views_and_unaligned_queries():
    import monarch_attention_b200 as ma
    cache, table = filled(2, 4, 2, 64, 64, [200, 77])
    lengths = torch.tensor([200, 77], dtype=torch.int32, device="cuda")
    q = queries(2, 4, 3, 64, BF, "heads")
    want = ma.cached_attention_b200(q, cache, table, lengths)
    wide = torch.zeros(2, 4, 3, 72, dtype=BF, device="cuda")
    got = ma.cached_attention_b200(q, cache, table, lengths, out=wide[..., :64])
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want) and not bool(wide[..., 64:].any())
    odd = torch.zeros(2, 4, 3, 67, dtype=BF, device="cuda")
    odd[..., 1:65] = q
    assert torch.equal(ma.cached_attention_b200(odd[..., 1:65], cache, table, lengths), want)
    assert torch.equal(ma.cached_attention_b200(q, cache, table, lengths, out=q.clone()), want)
    same = q.clone()   # in the place of the query
    assert torch.equal(ma.cached_attention_b200(same, cache, table, lengths, out=same), want)
    with pytest.raises(ValueError):
        ma.cached_attention_b200(q, cache, table, lengths, out=odd[..., 1:65])


def test_captured_steps_and_two_graphs_at_once():
    """A captured step replayed with other lengths; two graphs in flight on two streams, each with scratch of its own."""
    import monarch_attention_b200 as ma
    E, H, Hk, D, page = 2, 8, 2, 128, 64
    caches = [filled(E, 40, Hk, D, page, [2500, 2500], seed=s) for s in (1, 2)]
    lengths = [torch.tensor([2000, 5], dtype=torch.int32, device="cuda") for _ in caches]
    qs = [queries(E, H, 1, D, BF, "heads", seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for (cache, table), n, q in zip(caches, lengths, qs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ma.cached_attention_b200(q, cache, table, n))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for pair in ([2500, 1], [128, 129], [0, 2500]):
        for n in lengths:
            n.copy_(torch.tensor(pair, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (cache, table), q, out in zip(caches, qs, outs):
            check(out, q, cache, table, pair, None, page)
            assert torch.equal(out, ma.cached_attention_b200(q, cache, table, torch.tensor(pair, dtype=torch.int32, device="cuda")))


def test_calls_back_to_back_and_the_same_bits():
    import monarch_attention_b200 as ma
    cache, table = filled(3, 20, 4, 64, 64, [1200, 3, 700])
    lengths = torch.tensor([1200, 3, 700], dtype=torch.int32, device="cuda")
    qs = [queries(3, 8, 2, 64, HF, "tokens", seed=s) for s in range(3)]
    want = [ma.cached_attention_b200(q, cache, table, lengths) for q in qs]
    torch.cuda.synchronize()
    buffer = torch.empty_like(qs[0])
    for i in range(12):
        buffer.copy_(qs[i % 3])
        out = ma.cached_attention_b200(buffer, cache, table, lengths)
        buffer.zero_()
        assert torch.equal(out, want[i % 3])


def test_bad_pages_are_reported_and_the_others_unharmed():
    import monarch_attention_b200 as ma
    cache, table = filled(3, 4, 2, 64, 16, [60, 60, 60])
    q = queries(3, 4, 1, 64, BF, "heads")
    lengths = torch.tensor([60, 60, 60], dtype=torch.int32, device="cuda")
    want = ma.cached_attention_b200(q, cache, table, lengths)
    for page in (-1, 14, 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[1, 2] = page
        out = ma.cached_attention_b200(q, cache, bad, lengths)
        torch.cuda.synchronize()
        assert torch.equal(out[[0, 2]], want[[0, 2]])
        with pytest.raises(RuntimeError, match="page outside the cache"):
            ma.cached_attention_b200(q, cache, table, lengths)
    for length in (-1, 65, 2 ** 31 - 1):
        bad = lengths.clone()
        bad[1] = length
        ma.cached_attention_b200(q, cache, table, bad)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="length or count"):
            ma.cached_attention_b200(q, cache, table, lengths)
    assert torch.equal(ma.cached_attention_b200(q, cache, table, lengths), want)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: its last pages are read and written where they are."""
    import monarch_attention_b200 as ma
    pages, page = (2 ** 32 + 2 ** 26) // (64 * 128) // 4, 64
    cache = ma.PagedKV.allocate(pages, 4, 128, page)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([170], dtype=torch.int32, device="cuda")
    k, v, q = (queries(1, h, 170, 128, BF, "tokens", seed=s) for s, h in ((1, 4), (2, 4), (3, 8)))
    ma.append_kv_b200(cache, k, v, table, lengths)
    used = table[0].long()
    small = ma.PagedKV(*(t.view(torch.uint8)[used].view(t.dtype) if t.dtype == torch.float8_e4m3fn else t[used] for t in cache))
    out = ma.cached_attention_b200(q[:, :, -2:], cache, table, lengths)
    check(out, q[:, :, -2:], small, torch.arange(3)[None], [170], None, page)


def test_refusals():
    import monarch_attention_b200 as ma
    cache, table = filled(2, 4, 2, 64, 16, [60, 60])
    q, n = torch.zeros(2, 4, 1, 64, device="cuda", dtype=BF), torch.tensor([60, 60], dtype=torch.int32, device="cuda")
    wide = ma.PagedKV(*(torch.zeros(8, 2, 16, 32, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)), *cache[2:])
    for bad in [dict(query=q.float()), dict(query=q[0]), dict(query=q[:, :3]), dict(query=q[:1]), dict(query=q[..., :32]), dict(page_table=table.long()),
                dict(page_table=table[0]), dict(page_table=table[:, :0]), dict(page_table=table.cpu()), dict(lengths=n.long()), dict(lengths=n[:1]),
                dict(counts=n.long()), dict(counts=n[:1]), dict(window=-1), dict(window=5, causal=False), dict(softcap=-1.0), dict(softcap=float("inf")),
                dict(scale=float("nan")), dict(out=q.float()), dict(out=q[:1]), dict(cache=cache._replace(k=cache.k.view(torch.uint8))),
                dict(cache=cache._replace(k=cache.k.cpu())), dict(cache=cache._replace(k_scale=cache.k_scale.half())), dict(cache=wide),
                dict(cache=cache._replace(v=cache.v[:4])), dict(query=q.clone().requires_grad_(True))]:
        with pytest.raises(ValueError):
            ma.cached_attention_b200(**{**dict(query=q, cache=cache, page_table=table, lengths=n), **bad})
    k = torch.zeros(2, 2, 1, 64, device="cuda", dtype=BF)
    for bad in [dict(key=k.float()), dict(value=k.half()), dict(key=k[:, :1]), dict(value=k[:1]), dict(query=q[:1]), dict(query=q.half()),
                dict(rotary=ma.RotaryPositions(12)), dict(rotary=ma.RotaryPositions(128)), dict(key=k.clone().requires_grad_(True)),
                dict(lengths=n.long()), dict(page_table=table.t())]:
        with pytest.raises(ValueError):
            ma.append_kv_b200(**{**dict(cache=cache, key=k, value=k, page_table=table, lengths=n), **bad})
    with pytest.raises(TypeError):
        ma.append_kv_b200(cache, k, k, table, n, rotary=64)
    assert ma.cached_attention_b200(q[:0], cache, table[:0], n[:0]).shape == (0, 4, 1, 64)
    assert ma.cached_attention_b200(q[:, :, :0], cache, table, n).shape == (2, 4, 0, 64)
    assert ma.append_kv_b200(cache, k[:, :, :0], k[:, :, :0], table, n) is None


@pytest.mark.parametrize("N,G", [(4, 2), (40, 4)])
def test_windows_as_large_as_integers_go(N, G):
    """More tokens than the sequence is long, with windows whose arithmetic would leave 32 bits."""
    import monarch_attention_b200 as ma
    cache, table = filled(2, 4, 2, 64, 16, [3, 60])
    q = queries(2, 2 * G, N, 64, BF, "heads")
    lengths = torch.tensor([3, 60], dtype=torch.int32, device="cuda")
    want = ma.cached_attention_b200(q, cache, table, lengths)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30):
        assert torch.equal(ma.cached_attention_b200(q, cache, table, lengths, window=window), want)
    with pytest.raises(ValueError):
        ma.cached_attention_b200(q, cache, table, lengths, window=2 ** 31)


def test_prompts_and_appends_are_captured_and_replayed():
    import monarch_attention_b200 as ma
    rotary = ma.RotaryPositions(64, pairs="interleaved")
    module = ma.CachedAttention(rotary)
    cache = ma.PagedKV.allocate(40, 2, 64, 32)
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    lengths, counts = torch.tensor([100, 600], dtype=torch.int32, device="cuda"), torch.tensor([100, 50], dtype=torch.int32, device="cuda")
    q, k, v = (queries(2, h, 100, 64, BF, "tokens", seed=h) for h in (8, 2, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = module(q, k, v, cache, table, lengths, counts)
    for seed, pair, own in ((5, [100, 600], [100, 50]), (6, [640, 77], [3, 77]), (7, [0, 1], [0, 1])):
        for t in (q, k, v):
            t.copy_(queries(*t.shape, BF, "tokens", seed=seed))
        lengths.copy_(torch.tensor(pair, dtype=torch.int32)), counts.copy_(torch.tensor(own, dtype=torch.int32))
        before = [t.clone() if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8).clone() for t in cache]
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        other = ma.PagedKV(*(t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t for t in before))
        assert torch.equal(got, module(q, k, v, other, table, lengths, counts))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, other))


def test_first_calls_of_a_process_are_captured():
    """What a first call sets up (shared memory, the status word, attributes) does not invalidate a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, monarch_attention_b200 as ma
r = ma.RotaryPositions(128)
cache = ma.PagedKV.allocate(16, 2, 128, 64)
table = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
q, k, v = (torch.randn(1, h, 64, 128, device="cuda").to(torch.bfloat16) for h in (8, 2, 2))
n, many = torch.tensor([64], dtype=torch.int32, device="cuda"), torch.tensor([1000], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, b = ma.rotary_b200(q, k, r)
    c = ma.append_kv_b200(cache, k, v, table, n, query=q, rotary=r)
    d = ma.cached_attention_b200(c, cache, table, n)
    e = ma.cached_attention_b200(c[:, :, -1:], cache, table, many)
    f = ma.append_kv_b200(cache, k[:, :, :1], v[:, :, :1], table, many, query=q[:, :, :1], rotary=r)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(a, ma.rotary_b200(q, None, r)[0]) and torch.equal(d, ma.cached_attention_b200(c, cache, table, n))
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_calls_on_other_streams_and_from_threads():
    """Calls at once on streams of their own, with a cache for reading in common."""
    import threading

    import monarch_attention_b200 as ma
    cache, table = filled(2, 30, 2, 128, 64, [1800, 900])
    lengths = torch.tensor([1800, 900], dtype=torch.int32, device="cuda")
    qs = [queries(2, 8, n, 128, BF, "tokens", seed=n) for n in (1, 5, 80)]
    want = [ma.cached_attention_b200(q, cache, table, lengths) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for j in range(20):
                q = qs[(i + j) % 3]
                if not torch.equal(ma.cached_attention_b200(q, cache, table, lengths), want[(i + j) % 3]):
                    wrong.append((i, j))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_the_rows_of_out_do_not_overlap():
    import monarch_attention_b200 as ma
    cache, table = filled(2, 4, 2, 64, 16, [3, 60])
    q = queries(2, 4, 1, 64, BF, "heads")
    lengths = torch.tensor([3, 60], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ma.cached_attention_b200(q, cache, table, lengths, out=torch.zeros(1, 4, 1, 64, dtype=BF, device="cuda").expand(2, -1, -1, -1))
    with pytest.raises(ValueError):
        ma.cached_attention_b200(q, cache, table, lengths, softcap=1e-30)


@pytest.mark.parametrize("N", [1, 9, 40])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30])
def test_caps_far_above_the_scores(cap, N):
    """A cap that no score comes near leaves them as they are: its error is a part of the score, not of the cap.

    Scores of s lose s^3 / (3 cap^2), 10^-5 at most, and 2^-18 of themselves in the capping; the bound without a cap has D 2^-24 of the sum of
    magnitudes, which is more than that, twice."""
    import monarch_attention_b200 as ma
    lengths = [500, 40]
    cache, table = filled(2, 9, 2, 128, 64, lengths)
    q = queries(2, 8, N, 128, BF, "heads")
    out = ma.cached_attention_b200(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), softcap=cap)
    for e, L in enumerate(lengths):
        k, v = held(cache.k, cache.k_scale, table[e], L, 64), held(cache.v, cache.v_scale, table[e], L, 64)
        want, bound = attention(q[e], k, v, L - N, True, 128 ** -0.5)
        close(out[e], want, 2 * bound + 2.0 ** -8 * (want.abs() + 2 * bound), f"cap {cap}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-4, -1e-4])
def test_rows_of_zeros_over_keys_of_zeros(scale, D):
    """Many rows, some of zeros and some of padding, over blocks of keys of zeros (the smallest scale of all): a mask stays a mask."""
    import monarch_attention_b200 as ma
    lengths, counts, N, page = [200, 90], [40, 33], 40, 32
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts)]
    cache = ma.PagedKV.allocate(16, 2, D, page)
    k, v, q = (queries(2, h, n, D, BF, "heads", seed=s) for s, h, n in ((1, 2, 200), (2, 2, 200), (3, 8, N)))
    k[:, :, 16:100] = 0
    q[:, :, ::3] = 0
    ma.append_kv_b200(cache, k, v, table, dev[0], dev[0])
    out = ma.cached_attention_b200(q, cache, table, *dev, scale=scale)
    check(out, q, cache, table, lengths, counts, page, scale=scale)


@pytest.mark.parametrize("G,N,L", [(4, 1, 9000), (8, 6, 300), (4, 80, 3000)])
def test_the_result_in_the_querys_place(G, N, L):
    import monarch_attention_b200 as ma
    cache, table = filled(2, L // 64 + 1, 2, 64, 64, [L, L // 2])
    lengths = torch.tensor([L, L // 2], dtype=torch.int32, device="cuda")
    q = queries(2, 2 * G, N, 64, BF, "tokens")
    want = ma.cached_attention_b200(q, cache, table, lengths)
    buffer = torch.zeros(q.numel() + 64, device="cuda", dtype=BF)
    shifted = [buffer[i:i + q.numel()].view(2, 2 * G, N, 64) for i in (0, 64)]
    with pytest.raises(ValueError):  # rows would be overwritten before others read them
        ma.cached_attention_b200(shifted[0], cache, table, lengths, out=shifted[1])
    assert ma.cached_attention_b200(q, cache, table, lengths, out=q) is not None and torch.equal(q, want)


def test_a_result_over_what_a_backward_pass_needs_is_noticed():
    import monarch_attention_b200 as ma
    cache, table = filled(1, 2, 1, 64, 64, [100])
    q, w = queries(1, 1, 1, 64, BF, "heads"), torch.ones(1, 1, 1, 64, device="cuda", dtype=BF, requires_grad=True)
    saved = torch.zeros_like(q)
    y = (w * saved).sum()
    with torch.no_grad():
        ma.cached_attention_b200(q, cache, table, torch.tensor([100], dtype=torch.int32, device="cuda"), out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        ma.cached_attention_b200(q, cache, table, torch.tensor([100], dtype=torch.int32, device="cuda"), out=torch.zeros_like(q))


@pytest.mark.parametrize("E,H,Hk,N,D,dtype", [(12, 12, 12, 1, 64, BF), (16, 32, 8, 1, 128, HF), (18, 32, 8, 3, 128, BF), (70, 8, 2, 4, 64, HF)])
def test_heads_that_nearly_fill_the_device(E, H, Hk, N, D, dtype):
    """As many heads as SMs or fewer, of some thousand tokens at most: none is split, and a CTA has twelve warps' slices of several steps."""
    import monarch_attention_b200 as ma
    lengths = [(211 * e + 3) % 2100 + N for e in range(E)]
    cache, table = filled(E, 35, Hk, D, 64, lengths)
    q = queries(E, H, N, D, dtype, "heads")
    out = ma.cached_attention_b200(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check(out, q, cache, table, lengths, None, 64)


@pytest.mark.parametrize("N,L", [(3, 40), (3, 5000), (9, 700), (40, 300), (40, 5000), (150, 300)])
def test_rows_without_keys_are_zero_beside_nan(N, L):
    """A NaN among the values reaches the rows that see it; rows of padding and rows in front of the sequence's first token stay zero."""
    import monarch_attention_b200 as ma
    lengths, counts = [L, 2], [N - 1, N]
    cache, table = filled(2, L // 32 + 1, 2, 64, 32, lengths)
    for e, t in ((0, L // 2), (1, 1)):
        cache.v.view(torch.uint8)[int(table[e, t // 32]), :, t % 32, 5] = 0x7f
    q = queries(2, 8, N, 64, BF, "heads")
    out = ma.cached_attention_b200(q, cache, table, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts)))
    assert not bool(out[0, :, N - 1].any()) and not bool(out[1, :, :N - 2].any())
    assert bool(out[0, :, :N - 1, 5][:, -1].isnan().all()) and bool(out[1, :, -1, 5].isnan().all())
    assert bool(out[..., :5].isfinite().all()) and bool(out[..., 6:].isfinite().all())
