"""Accepted drafts and forked sequences: whole numbers and codes, equal to the definitions'; and a decoder's steps with both."""
import pytest
import torch

from decoder_reference import HALF_STEP, SUBNORMAL, attention, close, held
from drafts_reference import accepted, close_up, forked, trees
from test_kv_cache_gpu import heads

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def on_gpu(x, dtype=torch.int32):
    return None if x is None else torch.tensor(x, dtype=dtype, device="cuda")


def pools(layers, pages, Hk, D, page, layout="heads", seed=0, powers=True):
    """The caches of all layers, in one buffer each for keys and values, or (layout "both") in one for both; any codes, NaN among them."""
    import monarch_attention_b200 as ma
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, 2, pages, page, Hk, D) if layout == "tokens" else (layers, pages, 2, Hk, page, D) if layout == "both" else (layers, 2, pages, Hk, page, D)
    codes = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = 2.0 ** torch.randint(-5, 6, (layers, 2, pages, Hk, page // 16), generator=g, device="cuda").float()
    if not powers:
        scales = scales * (0.6 + torch.rand(scales.shape, generator=g, device="cuda"))
    if layout == "both":
        codes = codes.transpose(1, 2)
    elif layout == "tokens":
        codes = codes.transpose(3, 4)
    return [ma.PagedKV(codes[i, 0], codes[i, 1], scales[i, 0], scales[i, 1]) for i in range(layers)]


def cpu_copy(caches):
    return [[t.view(torch.uint8).cpu().clone() if t.dtype == torch.float8_e4m3fn else t.cpu().clone() for t in c] for c in caches]


def check_pools(caches, want):
    for i, (c, w) in enumerate(zip(cpu_copy(caches), want)):
        for name, a, b in zip(("k", "v", "k_scale", "v_scale"), c, w):
            if a.dtype == torch.uint8:  # (NaN has a sign that a conversion may lose)
                a, b = (torch.where(x & 0x7f == 0x7f, 0x7f, x) for x in (a, b))
            assert torch.equal(a, b), f"{name} of layer {i}: {int((a != b).sum())} differ"


# --- accepted drafts -------------------------------------------------------------------------------------------------------

ACCEPT = [  # layers, E, Hk, N, D, page, first (tokens in front of the call), counts, layout
    (1, 1, 1, 1, 64, 16, [0], None, "heads"), (2, 3, 2, 7, 128, 16, [0, 13, 100], None, "heads"), (3, 2, 12, 7, 64, 32, [9, 31], [5, 0], "tokens"), (1, 4, 1, 30, 128, 64, [60, 1, 16, 15], [30, 2, 1, 29], "both"),
    (2, 1, 3, 200, 64, 128, [77], None, "heads"), (1, 2, 1, 512, 128, 16, [5, 40], [512, 300], "tokens"), (40, 2, 1, 12, 64, 16, [20, 3], None, "heads"), (5, 70, 2, 10, 128, 32, list(range(70)), None, "heads")]


@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
@pytest.mark.parametrize("kind", ["random", "forest", "chain", "deep"])
@pytest.mark.parametrize("case", range(len(ACCEPT)))
def test_drafts_are_accepted(case, kind, ids):
    import monarch_attention_b200 as ma
    layers, E, Hk, N, D, page, first, counts, layout = ACCEPT[case]
    g = torch.Generator().manual_seed(case)
    caches = pools(layers, E * ((max(first) + N) // page + 1) + 3, Hk, D, page, layout, case)
    table = torch.randperm(caches[0].k.shape[0], generator=g)[:E * ((max(first) + N) // page + 1)].view(E, -1).to(torch.int32).cuda()
    parents = trees(E, N, "chain" if kind == "deep" else kind, case)
    if kind == "deep":   # two chains side by side: the second is right, and all of it moves
        parents = torch.arange(-2, N - 2).clamp_min(-1).expand(E, N).contiguous().to(torch.int32).cuda()
        parents[:, 1:2] = 0
        parents[:, 2:3] = 0
    # few different answers, so that several children fit and lines are long
    drafted, answers = (torch.randint(0, 2, (E, N), generator=g).to(ids) + (2 ** 33 if ids == torch.int64 else 0) for _ in range(2))
    if kind == "deep":
        drafted[:, 2::2], answers[:, 0], answers[:, 2::2] = 7, 7, 7
        drafted[:, 1::2] = 3
    count = counts or [N] * E
    lengths = [a + b for a, b in zip(first, count)]
    want, paths = cpu_copy(caches), []
    for e in range(E):
        paths.append(accepted(parents[e].tolist(), drafted[e].tolist(), answers[e].tolist(), count[e]))
        for w in want:
            close_up(w[0], w[2], table[e], first[e], paths[-1], page)
            close_up(w[1], w[3], table[e], first[e], paths[-1], page)
    sizes = on_gpu(lengths)
    got = ma.accept_drafts_b200(caches if layers > 1 else caches[0], table, sizes, on_gpu(counts), parents, drafted.cuda(), answers.cuda())
    assert got.path.tolist() == [p + [-1] * (N - len(p)) for p in paths]
    assert got.lengths.dtype == torch.int32 and got.lengths.tolist() == [a + len(p) for a, p in zip(first, paths)] and sizes.tolist() == lengths
    assert got.answer.dtype == ids and got.answer.tolist() == [int(answers[e, p[-1]]) if p else -1 for e, p in enumerate(paths)]
    check_pools(caches, want)


def test_scales_of_other_quantisers_cost_a_rounding():
    import monarch_attention_b200 as ma
    caches = pools(1, 4, 2, 64, 16, powers=False)
    codes = caches[0].k.view(torch.uint8)
    codes.copy_(torch.where(codes & 0x7f == 0x7f, 0, codes))
    table, parents = on_gpu([[0, 1, 2, 3]]), on_gpu([[-1, 0, 0, 2, 3]])
    before = held(caches[0].k, caches[0].k_scale, table[0], 20, 16)
    tokens = on_gpu([[1, 2, 3, 4, 5]])
    got = ma.accept_drafts_b200(caches, table, on_gpu([20]), on_gpu([5]), parents, tokens, on_gpu([[3, 0, 4, 5, 9]]))
    assert got.path.tolist() == [[0, 2, 3, 4, -1]] and got.lengths.tolist() == [19] and got.answer.tolist() == [9]
    after, scale = held(caches[0].k, caches[0].k_scale, table[0], 19, 16), caches[0].k_scale.double().cpu()
    for to, of in [(i, i) for i in range(16)] + [(16, 17), (17, 18), (18, 19)]:
        # half a step of the code, half a step of the smallest, and two roundings of 32 bits
        close(after[:, to], before[:, of], (2.0 ** -4 + 2.0 ** -22) * before[:, of].abs() + 2.0 ** -10 * scale[to // 16, :, 0:1], f"token {to}")


def test_bad_counts_and_pages_are_left_out_and_reported():
    import monarch_attention_b200 as ma
    caches = pools(2, 6, 1, 64, 16)
    table = on_gpu([[0, 1, -1], [2, 3, 99], [4, 5, 5]])
    parents = on_gpu([[-1, 0, 0, 2]] * 3)
    tokens, answers = on_gpu([[1, 2, 3, 4]] * 3), on_gpu([[3, 0, 4, 0]] * 3)
    want = cpu_copy(caches)
    for w in want:   # sequence 0 lies on its pages; the others' tokens are on no page, or their count is above the length
        close_up(w[0], w[2], table[0], 16, [0, 2, 3], 16)
        close_up(w[1], w[3], table[0], 16, [0, 2, 3], 16)
    got = ma.accept_drafts_b200(caches, table, on_gpu([20, 37, 2]), None, parents, tokens, answers)
    torch.cuda.synchronize()
    assert got.lengths.tolist() == [19, 36, 2] and got.path.tolist() == [[0, 2, 3, -1], [0, 2, 3, -1], [-1] * 4] and got.answer.tolist() == [0, 0, -1]
    check_pools(caches, want)
    with pytest.raises(RuntimeError):
        ma.accept_drafts_b200(caches, table, on_gpu([20, 37, 2]), None, parents, tokens, answers)


def test_nothing_to_accept():
    import monarch_attention_b200 as ma
    caches = pools(1, 4, 1, 64, 16)
    table, lengths = on_gpu([[0, 1], [2, 3]]), on_gpu([7, 20])
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    got = ma.accept_drafts_b200(caches, table, lengths, None, none, none, none)
    assert got.lengths.tolist() == [7, 20] and got.path.shape == (2, 0) and got.answer.tolist() == [-1, -1]
    got = ma.accept_drafts_b200(caches, table[:0], lengths[:0], None, none[:0], none[:0], none[:0])
    assert got.lengths.shape == (0,) and got.path.shape == (0, 0)


# --- forked sequences --------------------------------------------------------------------------------------------------------

def sequences(E, page, lengths, spare, P, pages, seed=0):
    """A table whose rows hold pages for their length and `spare` more, all of their own; and the pages' uses."""
    g = torch.Generator().manual_seed(seed)
    free = torch.randperm(pages, generator=g).tolist()
    table, uses = [], [0] * pages
    for e in range(E):
        n = min(P, -(-lengths[e] // page) + spare[e])
        row = [free.pop() for _ in range(n)]
        for p in row:
            uses[p] = 1
        table.append(row + [-1] * (P - n))
    return table, uses


def run_fork(caches, uses, table, lengths, source, room, page):
    """The call beside its definition; returns what is there afterwards."""
    import monarch_attention_b200 as ma
    want, E = cpu_copy(caches), len(table)
    new_uses, new_table, new_lengths, copies = forked(uses, table, lengths, source if source is not None else list(range(E)), room if isinstance(room, list) else [room] * E, page)
    for a, b, tokens in copies:
        blocks = -(-tokens // 16)
        for w in want:
            for j in (0, 1):
                w[j][b, :, :blocks * 16] = w[j][a, :, :blocks * 16]
                w[j + 2][b, :, :blocks] = w[j + 2][a, :, :blocks]
    got = [on_gpu(x) for x in (uses, table, lengths)]
    ma.fork_sequences_b200(caches, *got, on_gpu(source), on_gpu(room) if isinstance(room, list) else room)
    assert got[2].tolist() == new_lengths
    assert got[1].tolist() == new_table
    assert got[0].tolist() == new_uses
    check_pools(caches, want)
    return new_uses, new_table, new_lengths


FORKS = [  # layers, E, Hk, D, page, lengths, spare pages, source, room
    (1, 1, 1, 64, 16, [5], [0], [0], 1), (2, 2, 2, 128, 16, [5, 40], [0, 1], [1, 0], 3), (3, 4, 12, 64, 16, [37] * 4, [0] * 4, [2, 2, 2, 2], 1), (1, 4, 2, 128, 64, [64, 100, 0, 300], [0, 0, 1, 2], [0, 0, 3, 1], 0),
    (2, 5, 1, 64, 32, [10, 20, 33, 64, 65], [1, 0, 0, 3, 1], [-1, 4, 4, -1, 1], [100, 1, 0, 0, 31]), (1, 3, 1, 64, 16, [48, 16, 1], [2, 2, 2], None, [0, 40, 15]),
    (36, 3, 1, 128, 32, [50, 9, 70], [0, 0, 0], [2, 2, 0], 1), (1, 2, 4, 64, 256, [700, 5], [0, 0], [0, 0], 1000)]


@pytest.mark.parametrize("layout", ["heads", "tokens", "both"])
@pytest.mark.parametrize("case", range(len(FORKS)))
def test_sequences_fork(case, layout):
    layers, E, Hk, D, page, lengths, spare, source, room = FORKS[case]
    P = max(lengths) // page + max(spare) + 8
    pages = sum(-(-n // page) + s for n, s in zip(lengths, spare)) + 40
    caches = pools(layers, pages, Hk, D, page, layout, case)
    table, uses = sequences(E, page, lengths, spare, P, pages, case)
    state = run_fork(caches, uses, table, lengths, source, room, page)
    for _ in range(2):   # and again, of what is shared now
        state = run_fork(caches, *state, source, room, page)


@pytest.mark.parametrize("E,P,page,pages,most", [(1500, 9, 16, 14000, 100), (300, 40, 16, 9000, 400), (7, 3000, 16, 20000, 40000), (40, 5, 64, 150, 200), (2, 2, 16, 100000, 20), (64, 33, 32, 4096, 1000)])
def test_sequences_fork_at_random(E, P, page, pages, most):
    g = torch.Generator().manual_seed(E)
    caches = pools(1, pages, 1, 64, page)
    lengths = torch.randint(0, most, (E,), generator=g).tolist()
    budget = pages // 2
    for e in range(E):   # rows that the pool has no room for are empty
        need = -(-lengths[e] // page)
        lengths[e] = lengths[e] if need <= budget and need < P else 0
        budget -= -(-lengths[e] // page)
    table, uses = sequences(E, page, lengths, [0] * E, P, pages, 1)
    state = (uses, table, lengths)
    for i in range(4):
        source = torch.randint(-1, E, (E,), generator=g)
        source = torch.where(torch.rand(E, generator=g) < 0.5, torch.arange(E), source).tolist()
        room = torch.randint(0, 20, (E,), generator=g).tolist()
        # (what is in the rows may grow beyond the table: then the room is cut, and reported, which the next call would raise)
        room = [min(r, P * page - (state[2][s] if s >= 0 else 0)) for r, s in zip(room, source)]
        if forked(*state, source, room, page)[0].count(0) < 2 * E and pages > 2 * E:
            source = [-1 if e % 2 else s for e, s in enumerate(source)]
        state = run_fork(caches, *state, source, room, page)


def test_pages_that_two_rows_hold_are_copied_before_they_are_written():
    """A sequence that was cut back into what it shares gets a page of its own, and so does the other; the page that both read is not given out meanwhile."""
    caches = pools(2, 20, 2, 64, 16)
    table, uses = sequences(2, 16, [40, 0], [0, 0], 6, 20, 3)
    state = run_fork(caches, uses, table, [40, 0], [0, 0], 1, 16)
    assert state[1][0][:2] == state[1][1][:2] and state[1][0][2] != state[1][1][2]
    state = run_fork(caches, state[0], state[1], [20, 25], None, 8, 16)
    assert state[1][0][0] == state[1][1][0] and state[1][0][1] != state[1][1][1]
    assert max(state[0][p] for row in state[1] for p in row[1:] if p >= 0) == 1


def reported(caches, match):
    import monarch_attention_b200 as ma
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=match):
        ma.fork_sequences_b200(caches, on_gpu([0] * caches[0].k.shape[0]), on_gpu([[-1]]), on_gpu([0]))


def test_a_pool_without_free_pages_is_reported():
    caches = pools(1, 6, 1, 64, 16)
    table, uses = sequences(3, 16, [33, 20, 0], [0, 0, 0], 4, 6)
    run_fork(caches, uses, table, [33, 20, 0], [0, 0, 0], 1, 16)      # (row 1's own pages suffice for both copies)
    run_fork(caches, uses, table, [33, 20, 0], [0, 0, 0], 17, 16)     # five pages more, of three
    reported(caches, "free pages")
    _, _, lengths = run_fork(caches, uses, table, [33, 20, 0], [0, 0, 0], 60, 16)
    assert lengths == [33, 33, 32]
    reported(caches, None)


def test_bad_sources_lengths_and_pages_are_reported():
    caches = pools(1, 12, 1, 64, 16)
    table, uses = sequences(3, 16, [33, 20, 5], [0, 0, 0], 4, 12)
    run_fork(caches, uses, table, [33, 20, 5], [7, -2, 2], 1, 16)
    reported(caches, "source")
    run_fork(caches, uses, table, [33, 500, -5], None, 1, 16)     # more tokens than the row has pages for, less than none
    reported(caches, "length")
    run_fork(caches, uses, table, [33, 20, 5], None, [1, 1000, -4], 16)   # more room than the table has, less than none
    reported(caches, "length")
    table[0][1] = 99
    run_fork(caches, uses, table, [10, 20, 5], None, 1, 16)
    reported(caches, "page")


def test_refusals():
    import monarch_attention_b200 as ma
    caches = pools(2, 8, 2, 64, 16)
    table, uses = sequences(2, 16, [20, 5], [0, 0], 3, 8)
    table, uses, lengths, source = on_gpu(table), on_gpu(uses), on_gpu([20, 5]), on_gpu([0, 0])
    parents, tokens = on_gpu([[-1, 0]] * 2), on_gpu([[1, 2]] * 2)
    ma.fork_sequences_b200(caches, uses, table, lengths, source, 1)
    ma.accept_drafts_b200(caches, table, lengths, None, parents, tokens, tokens)
    other = ma.PagedKV.allocate(8, 2, 128, 16)
    smaller = ma.PagedKV.allocate(7, 2, 64, 16)
    overlapping = ma.PagedKV(caches[0].k[:1].expand(8, -1, -1, -1), *caches[0][1:])
    grad = ma.PagedKV(caches[0].k, caches[0].v, caches[0].k_scale.clone().requires_grad_(), caches[0].v_scale)
    for bad in ([caches[0], other], [caches[0], smaller], [caches[0], caches[0]], [caches[0], ma.PagedKV(caches[1].k, caches[0].v, *caches[1][2:])], [overlapping], [],
                [ma.PagedKV(caches[0].k, caches[0].k, *caches[0][2:])], [grad], [ma.PagedKV.allocate(8, 2, 64, 16, device="cpu")]):
        with pytest.raises(ValueError):
            ma.fork_sequences_b200(bad, uses, table, lengths, source, 1)
        with pytest.raises(ValueError):
            ma.accept_drafts_b200(bad, table, lengths, None, parents, tokens, tokens)
    for bad in (caches[0].k, [caches[0].k], [(1, 2, 3, 4)], 5):
        with pytest.raises(TypeError):
            ma.fork_sequences_b200(bad, uses, table, lengths, source, 1)
    for kw in (dict(page_uses=uses[:7]), dict(page_uses=uses.long()), dict(page_table=table.long()), dict(page_table=table[:1].expand(2, -1)), dict(lengths=lengths[:1]), dict(lengths=lengths.cpu()),
               dict(source=source.long()), dict(source=source[:1]), dict(room=on_gpu([1])), dict(room=-1), dict(source=lengths), dict(room=uses[:2]), dict(lengths=uses[2:4])):
        with pytest.raises(ValueError):
            ma.fork_sequences_b200(caches, **{**dict(page_uses=uses, page_table=table, lengths=lengths, source=source, room=1), **kw})
    with pytest.raises(TypeError):
        ma.fork_sequences_b200(caches, uses, table, lengths, source, "1")
    for kw in (dict(parents=parents[:, :1]), dict(drafted=tokens.long()), dict(drafted=tokens.float(), answers=tokens.float()), dict(answers=tokens[:1]), dict(counts=tokens), dict(answers=tokens.cpu()),
               dict(drafted=on_gpu([[1, 2, 3, 4]] * 2)[:, ::2])):
        with pytest.raises(ValueError):
            ma.accept_drafts_b200(caches, **{**dict(page_table=table, lengths=lengths, counts=None, parents=parents, drafted=tokens, answers=tokens), **kw})
    wide = torch.zeros(1, 513, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="512"):
        ma.accept_drafts_b200(caches, torch.zeros(1, 40, dtype=torch.int32, device="cuda"), on_gpu([600]), None, wide - 1, wide, wide)


# --- a decoder's steps ---------------------------------------------------------------------------------------------------------

def decoder(E=6, layers=3, H=8, Hk=2, D=64, page=32, N=9, P=12, pages=80):
    """Steps of a decoder in place: forks, a tree of drafts through all layers, its acceptance.  Returns the state and the step."""
    import monarch_attention_b200 as ma
    g = torch.Generator(device="cuda").manual_seed(0)
    rotary = ma.RotaryPositions(D)
    attn = ma.CachedAttention(rotary)
    s = dict(caches=[ma.PagedKV.allocate(pages, Hk, D, page) for _ in range(layers)], uses=on_gpu([0] * pages), table=on_gpu([[-1] * P] * E), lengths=on_gpu([0] * E),
             source=on_gpu(list(range(E))), room=on_gpu([N] * E), counts=on_gpu([N] * E), parents=trees(E, N, "random", 1), drafted=on_gpu([[0] * N] * E), answers=on_gpu([[0] * N] * E))
    s["x"] = [[(torch.randn(E, N, h, D, generator=g, device="cuda") * 1.5).to(BF).transpose(1, 2) for h in (H, Hk, Hk)] for _ in range(layers)]

    def step():
        ma.fork_sequences_b200(s["caches"], s["uses"], s["table"], s["lengths"], s["source"], s["room"])
        s["lengths"].add_(s["counts"])
        s["out"] = [attn(*x, c, s["table"], s["lengths"], s["counts"], s["parents"]) for x, c in zip(s["x"], s["caches"])]
        s["got"] = ma.accept_drafts_b200(s["caches"], s["table"], s["lengths"], s["counts"], s["parents"], s["drafted"], s["answers"])
        s["lengths"].copy_(s["got"].lengths)
    return s, step


def scripted(s, i):
    """The i-th step's inputs, written into the state's tensors."""
    g = torch.Generator().manual_seed(100 + i)
    E, N = s["drafted"].shape
    source = torch.arange(E)
    if i % 2:
        source = torch.where(torch.rand(E, generator=g) < 0.4, torch.randint(0, E, (E,), generator=g), source)
    if i == 4:
        source[3] = -1
    s["source"].copy_(source)
    s["counts"].copy_(torch.randint(1, N + 1, (E,), generator=g))
    s["parents"].copy_(trees(E, N, "random", i))
    for n in ("drafted", "answers"):
        s[n].copy_(torch.randint(0, 2, (E, N), generator=g))
    for x in s["x"]:
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g) * 1.5)


def everything(s):
    flat = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for c in s["caches"] for t in c]
    return [t.clone() for t in (*flat, *s["out"], *s["got"], s["uses"], s["table"], s["lengths"])]


def test_steps_of_a_decoder_keep_what_was_accepted():
    """What the sequences hold, followed on the CPU from the codes that each append wrote, through forks and acceptance; and attention over it."""
    import monarch_attention_b200 as ma
    page = 32
    s, step = decoder(page=page)
    E = 6
    truth = [[[torch.zeros(2, 0, 64, dtype=torch.float64) for _ in "kv"] for _ in range(E)] for _ in s["caches"]]
    for i in range(8):
        scripted(s, i)
        start_of = s["lengths"].tolist()
        step()
        source, counts = s["source"].tolist(), s["counts"].tolist()
        truth = [[[t.clone() for t in of[source[e]]] if source[e] >= 0 else [torch.zeros(2, 0, 64, dtype=torch.float64) for _ in "kv"] for e in range(E)] for of in truth]
        for layer, c in enumerate(s["caches"]):
            for e in range(E):
                path = [n for n in s["got"].path[e].tolist() if n >= 0]
                start = start_of[source[e]] if source[e] >= 0 else 0
                assert path == accepted(s["parents"][e].tolist(), s["drafted"][e].tolist(), s["answers"][e].tolist(), counts[e])
                assert int(s["lengths"][e]) == start + len(path) == truth[layer][e][0].shape[1] + len(path)
                for j, (codes, scale) in enumerate(((c.k, c.k_scale), (c.v, c.v_scale))):
                    now = held(codes, scale, s["table"][e], start + len(path), page)
                    steps = scale.cpu()[s["table"][e].clamp_min(0).long().cpu()].double().transpose(0, 1).flatten(1, 2).repeat_interleave(16, -1)[:, :start + len(path), None]
                    # older tokens are exact but for values that have become subnormal
                    close(now[:, :start], truth[layer][e][j], 2.0 ** -9 * steps[:, :start], f"step {i}, layer {layer}, sequence {e}")
                    x = s["x"][layer][1 + j][e][:, path].double().cpu()
                    if j == 1:
                        # half a step of the code, and twice (the append, the move) half of the smallest, of a scale under 2^-5: 14 = 448 * 2^-5 is 9 deviations
                        assert float(s["x"][layer][1 + j].abs().max()) < 14.0
                        close(now[:, start:], x, 2.0 ** -4 * x.abs() + 2.0 ** -9 * 2.0 ** -5, f"step {i}, layer {layer}, new values of {e}")
                    truth[layer][e][j] = now
        used = [0] * s["uses"].numel()
        for row in s["table"].tolist():
            for p in row:
                if p >= 0:
                    used[p] += 1
        assert used == s["uses"].tolist()
    # one more token of each, over all that was accepted
    ma.fork_sequences_b200(s["caches"], s["uses"], s["table"], s["lengths"], None, 1)
    q, k, v = (heads(E, h, 1, 64, BF, "tokens", 50 + h) for h in (8, 2, 2))
    s["lengths"].add_(1)
    c = s["caches"][1]
    ma.append_kv_b200(c, k, v, s["table"], s["lengths"])
    out = ma.cached_attention_b200(q, c, s["table"], s["lengths"])
    for e in range(E):
        L = int(s["lengths"][e])
        kk, vv = held(c.k, c.k_scale, s["table"][e], L, page), held(c.v, c.v_scale, s["table"][e], L, page)
        close(kk[:, :-1], truth[1][e][0], 2.0 ** -9 * c.k_scale.max().item() * torch.ones(1, dtype=torch.float64), "keys")
        want, bound = attention(q[e], kk, vv, L - 1, True, 64 ** -0.5)
        close(out[e], want, bound + HALF_STEP[BF] * (want.abs() + bound) + SUBNORMAL[BF], f"sequence {e}")


def test_steps_are_captured_and_replayed():
    """A captured step, replayed over other lengths, trees and forks, has the bits of the calls; two graphs in turn do not share scratch."""
    eager, step = decoder()
    first, capture_first = decoder()
    second, capture_second = decoder()
    graphs = []
    for s, fn in ((first, capture_first), (second, capture_second)):
        scripted(s, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        for t in (*[t for c in s["caches"] for t in c], s["uses"], s["lengths"]):
            t.view(torch.uint8).zero_()
        s["table"].fill_(-1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fn()
        graphs.append(graph)
    for i in range(6):
        for s in (eager, first, second):
            scripted(s, i)
        step()
        for g in graphs:
            g.replay()
        want = everything(eager)
        for s in (first, second):
            assert all(torch.equal(a, b) for a, b in zip(everything(s), want))


def test_steps_on_two_streams_do_not_meet():
    alone, step = decoder()
    pairs = [decoder() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in pairs]
    for i in range(5):
        scripted(alone, i)
        step()
        for s, _ in pairs:
            scripted(s, i)
        torch.cuda.synchronize()
        for stream, (_, fn) in zip(streams, pairs):
            with torch.cuda.stream(stream):
                fn()
        torch.cuda.synchronize()
        want = everything(alone)
        for s, _ in pairs:
            assert all(torch.equal(a, b) for a, b in zip(everything(s), want))
