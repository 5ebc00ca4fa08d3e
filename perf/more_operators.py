"""What a user of drafted continuations and of shared sequences has the paged cache do.

``listed()`` gives the representative calls, ``draw(rng)`` more of the same ranges.  ``run`` computes one call: with
``own`` through the library's entry points, else in elementary tensor operations in 32 bits (angles in 64).

Operators (``op`` of a case):

* ``tree``: attention of the tokens of a tree over the cache.  ``parents`` names each token's parent among the call's tokens (-1: none); a token
  sees what is cached in front of the call, its ancestors and itself, and stands at the position of its depth.
* ``place``: the append of such a tree, keys and queries rotated at the positions of their depth.
* ``accept``: which drafted tokens the model's answers confirm, and the cache of all layers closed up over them.
* ``fork``: sequences that go on from others (or end, or begin): pages shared and counted, half-filled ones copied in all layers, new ones given out.

Fields: ``E`` sequences, ``H`` query heads, ``Hk`` key/value heads, ``N`` drafted tokens, ``D`` head width, ``L`` most tokens of a sequence,
those of the call among them, ``page`` tokens of a page, ``layers``; ``ragged`` lengths; ``counts``: sequences bring fewer than N tokens;
``layout`` as projections have it (``tokens``: (E, H, N, D) views of (E, N, H, D)) or ``heads``; ``window`` and ``softcap`` (0: none) of the attention;
``beams`` sequences that descend from one another, ``ending`` the share of sequences that end (and are followed by new ones).
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
BASE = 10000.0
BLOCK = 16           # tokens that share a scale
MOST_TOKENS = 512    # of a tree
PEAK_KEYS = 16 * 8 * 8192 * 128            # most elements of the keys that an attention reads
PEAK_SCORES = 8 * 32 * 61 * 8192           # most scores of one
PEAK_POOL = 16 * 2048 * 8 * 64 * 128       # most elements of the keys of all layers' pools


def _tree(name, E, H, Hk, N, D, dtype, L, page, ragged=True, counts=False, window=0, softcap=0.0, layout="tokens"):
    return dict(name=name, op="tree", E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, ragged=ragged, counts=counts,
                window=window, softcap=softcap, layout=layout)


def _place(name, E, H, Hk, N, D, dtype, L, page, pairs="half", counts=False, layout="tokens"):
    return dict(name=name, op="place", E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, pairs=pairs, ragged=True, counts=counts, layout=layout)


def _accept(name, layers, E, Hk, N, D, L, page, counts=False):
    return dict(name=name, op="accept", layers=layers, E=E, Hk=Hk, N=N, D=D, L=L, page=page, ragged=True, counts=counts)


def _fork(name, layers, E, Hk, D, L, page, beams, ending=0.0):
    return dict(name=name, op="fork", layers=layers, E=E, Hk=Hk, D=D, L=L, page=page, beams=beams, ending=ending)


def listed():
    return [
        # a few guesses for one sequence: latency is all of it
        _tree("tree_one", 1, 12, 12, 7, 64, "f16", 500, 16, ragged=False),
        # small trees of a serving batch, grouped heads: the cache's bytes count
        _tree("tree_batch", 16, 16, 4, 8, 128, "bf16", 8192, 64, counts=True),
        # trees of many guesses, sliding window, capped scores, sequences with fewer guesses
        _tree("tree_window", 32, 12, 12, 25, 64, "f16", 4096, 32, counts=True, window=1024, softcap=30.0, layout="heads"),
        # wide trees of a serving batch
        _tree("tree_wide", 8, 32, 8, 61, 128, "bf16", 8192, 64),
        # one wide tree behind one long context
        _tree("tree_long", 1, 16, 2, 33, 128, "bf16", 131071, 128, ragged=False),
        # a few guesses of a few sequences into the cache
        _place("place_few", 8, 12, 12, 7, 64, "bf16", 700, 16),
        # wide trees of a serving batch
        _place("place_wide", 64, 32, 8, 61, 128, "bf16", 600, 64, "interleaved", counts=True),
        # one sequence: which guesses were right, twelve layers closed up
        _accept("accept_one", 12, 1, 12, 7, 64, 300, 16),
        # a serving batch
        _accept("accept_batch", 16, 64, 8, 61, 128, 400, 64, counts=True),
        # four beams of one sentence
        _fork("fork_beams", 12, 4, 12, 64, 500, 16, 4),
        # a serving batch of groups of samples, some of which end and make room for others
        _fork("fork_batch", 16, 128, 8, 128, 1000, 64, 8, ending=0.1),
        # a few long contexts in small pages: their tables are what there is to do
        _fork("fork_long", 2, 8, 2, 64, 60000, 16, 4),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "place", "accept", "accept", "fork", "fork"])
    D = rng.choice([64, 128])
    group = rng.choice([1, 1, 2, 4, 4, 5, 8])
    Hk = rng.choice([1, 2, 4, 8, 12] if group < 8 else [1, 2, 4, 8])
    H, page = Hk * group, rng.choice([16, 32, 64, 128])
    layout, dtype = rng.choice(["tokens", "tokens", "heads"]), rng.choice(["bf16", "bf16", "f16"])
    N = rng.choice([1, rng.randint(2, 9), rng.randint(2, 9), _log_int(rng, 10, 64), _log_int(rng, 10, MOST_TOKENS)])
    if op == "tree":
        most = min(131071, PEAK_SCORES // (N * H), PEAK_KEYS // (Hk * D))
        L = N + _log_int(rng, 1, max(1, most - N))
        E = _log_int(rng, 1, max(1, min(64, PEAK_SCORES // (N * H * L), PEAK_KEYS // (Hk * D * L))))
        return dict(op=op, E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, ragged=rng.random() < 0.7, counts=N > 1 and rng.random() < 0.5,
                    window=rng.choice([0, 0, 0, rng.randint(1, L)]), softcap=rng.choice([0.0, 0.0, 20.0]), layout=layout)
    if op == "place":
        L = N + _log_int(rng, 1, 2000)
        E = _log_int(rng, 1, max(1, min(128, PEAK_POOL // (8 * L * Hk * D), PEAK_POOL // (16 * N * H * D))))
        return dict(op=op, E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, pairs=rng.choice(["half", "interleaved"]), ragged=True,
                    counts=N > 1 and rng.random() < 0.5, layout=layout)
    layers = _log_int(rng, 1, 24)
    if op == "accept":
        L = N + _log_int(rng, 1, 1000)
        E = _log_int(rng, 1, max(1, min(128, PEAK_POOL // (2 * layers * (L + 2 * page) * Hk * D))))
        return dict(op=op, layers=layers, E=E, Hk=Hk, N=N, D=D, L=L, page=page, ragged=True, counts=N > 1 and rng.random() < 0.5)
    L = _log_int(rng, 2, min(60000, PEAK_POOL // (4 * layers * Hk * D)))
    E = _log_int(rng, 2, max(2, min(256, PEAK_POOL // (2 * layers * (L + 2 * page) * Hk * D))))
    return dict(op=op, layers=layers, E=E, Hk=Hk, D=D, L=L, page=page, beams=rng.choice([1, 2, 4, 8]), ending=rng.choice([0.0, 0.1, 0.3]))


def _pool(g, dev, layers, pages, Hk, page, D):
    """Codes and scales of the keys (or values) of all layers: random magnitudes of a spread and an offset of each channel."""
    codes = torch.empty(layers, pages, Hk, page, D, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(layers, pages, Hk, page // BLOCK, device=dev)
    step = max(1, (1 << 26) // (Hk * page * D))
    for layer in range(layers):
        offset = 0.3 * torch.randn(1, Hk, 1, D, generator=g, device=dev)
        for i in range(0, pages, step):
            x = torch.randn(codes[layer, i:i + step].shape, generator=g, device=dev).mul_(1.5).add_(offset)
            x = x.view(-1, Hk, page // BLOCK, BLOCK, D)
            s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448.0)))
            codes[layer, i:i + step] = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(-1, Hk, page, D)
            scales[layer, i:i + step] = s
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    E, Hk, D, L, page = (case[x] for x in ("E", "Hk", "D", "L", "page"))
    if case["op"] == "fork":
        return _prepare_fork(case, g, dev)
    N = case["N"]
    state = dict(case=case)
    counts = torch.randint(1, N + 1, (E,), generator=g, device=dev) if case["counts"] else torch.full((E,), N, device=dev)
    lengths = torch.randint(N, L + 1, (E,), generator=g, device=dev) if case["ragged"] else torch.full((E,), L, device=dev)
    per = (L + 2 * BLOCK + page - 1) // page
    state["page_table"] = torch.randperm(E * per, generator=g, device=dev).view(E, per).to(torch.int32)
    state["lengths"], state["counts"] = lengths.to(torch.int32), counts.to(torch.int32) if case["counts"] else None
    # a token's parent is any earlier one: trees of a depth of some ln N
    n = torch.arange(N, device=dev)
    state["parents"] = torch.minimum((torch.rand(E, N, generator=g, device=dev) * n).floor().long(), n - 1).to(torch.int32)
    layers = case.get("layers", 1)
    for name in ("k", "v"):
        state[name + "_cache"], state[name + "_scale"] = _pool(g, dev, layers, E * per, Hk, page, D)
    if case["op"] == "accept":
        # the model answers each token with one of its drafted continuations four times in five
        state["drafted"] = torch.randint(0, 50265, (E, N), generator=g, device=dev)
        right = torch.rand(E, N, generator=g, device=dev) < 0.8
        child = torch.full((E, N), -1, device=dev).scatter_reduce(
            1, state["parents"].long().clamp_min(0), torch.where((state["parents"] >= 0) & right, n, -1), "amax")
        answers = torch.randint(0, 50265, (E, N), generator=g, device=dev)
        state["answers"] = torch.where(child >= 0, state["drafted"].gather(1, child.clamp_min(0)), answers)
        return state

    def heads(h, std):
        # projected hidden states: a spread and an offset of each channel of a head
        shape = (E, h, N, D) if case["layout"] == "heads" else (E, N, h, D)
        t = torch.randn(shape, generator=g, device=dev)
        t = t if case["layout"] == "heads" else t.permute(0, 2, 1, 3)
        t.mul_(std).add_(0.3 * torch.randn(1, h, 1, D, generator=g, device=dev))
        return t.to(DTYPES[case["dtype"]])

    state["q"] = heads(case["H"], 1.5)
    if case["op"] == "place":
        state["k"], state["v"] = heads(Hk, 1.5), heads(Hk, 1.5)
        state["frequencies"] = torch.tensor([BASE ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device=dev)
    return state


def _prepare_fork(case, g, dev):
    """Rows of pages of their own, in groups of ``beams``; a row goes on from one of its group's survivors (its own where it survives), or ends."""
    E, Hk, D, L, page, beams = (case[x] for x in ("E", "Hk", "D", "L", "page", "beams"))
    lengths = torch.randint(1, L + 1, (E,), generator=g, device=dev)
    lengths = lengths[torch.arange(E, device=dev) // beams * beams]     # those of a group are as long as one another
    per = (L + page - 1) // page + 1
    used = (lengths + page - 1) // page
    pages = E * per + 7
    column = torch.arange(per, device=dev)
    table = torch.randperm(pages, generator=g, device=dev)[:E * per].view(E, per)
    table = torch.where(column < used[:, None], table, -1).to(torch.int32)
    uses = torch.zeros(pages, dtype=torch.int32, device=dev)
    uses[table[table >= 0].long()] = 1
    row = torch.arange(E, device=dev)
    first = row // beams * beams
    size = torch.minimum(first + beams, torch.tensor(E, device=dev)) - first
    stays = torch.rand(E, generator=g, device=dev) < 0.4
    stays |= row == first
    picked = first + (torch.rand(E, generator=g, device=dev) * size).floor().long()
    source = torch.where(stays, row, torch.where(stays[picked], picked, first))
    ends = torch.rand(E, generator=g, device=dev) < case["ending"]
    ends &= ~torch.isin(row, source[source != row])                      # nothing goes on from one that ends
    source = torch.where(ends, -1, source)
    room = torch.where(ends, torch.randint(1, L + 1, (E,), generator=g, device=dev), 1)
    state = dict(case=case, page_uses=uses, page_table=table, lengths=lengths.to(torch.int32), source=source.to(torch.int32), room=room.to(torch.int32))
    for name in ("k", "v"):
        state[name + "_cache"], state[name + "_scale"] = _pool(g, dev, case["layers"], pages, Hk, page, D)
    return state


# --- the library's calls -------------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=64)
def _handle(dim, pairs):
    from monarch_attention_b200 import RotaryPositions
    return RotaryPositions(dim, base=BASE, pairs=pairs)


def _caches(s):
    """The layers' caches, as a program keeps them from its start."""
    if "caches" not in s:
        from monarch_attention_b200 import PagedKV
        s["caches"] = [PagedKV(*parts) for parts in zip(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])]
    return s["caches"]


def _run_own(s):
    import monarch_attention_b200 as ma
    c, caches = s["case"], _caches(s)
    if c["op"] == "tree":
        return ma.cached_attention_b200(s["q"], caches[0], s["page_table"], s["lengths"], s["counts"], softcap=c["softcap"], window=c["window"],
                                        parents=s["parents"], token_major_output=c["layout"] == "tokens")
    held = {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if c["op"] == "place":
        q = ma.append_kv_b200(caches[0], s["k"], s["v"], s["page_table"], s["lengths"], s["counts"], query=s["q"], rotary=_handle(c["D"], c["pairs"]),
                              parents=s["parents"])
        return {"q": q, **held}
    if c["op"] == "accept":
        a = ma.accept_drafts_b200(caches, s["page_table"], s["lengths"], s["counts"], s["parents"], s["drafted"], s["answers"])
        return {"lengths": a.lengths, "path": a.path, "answer": a.answer, **held}
    ma.fork_sequences_b200(caches, s["page_uses"], s["page_table"], s["lengths"], s["source"], s["room"])
    return {n: s[n] for n in ("page_uses", "page_table", "lengths", *held)}


# --- plain forms -----------------------------------------------------------------------------------------------------------

def _counts(s):
    return s["counts"].long() if s["counts"] is not None else torch.full_like(s["lengths"], s["case"]["N"], dtype=torch.long)


def _descent(parents):
    """(E, N, N): whether token m is token n or an ancestor of it."""
    N = parents.shape[1]
    n = torch.arange(N, device=parents.device)
    reach = ((parents[..., None] == n) | (n[:, None] == n)).float()
    for _ in range(max(1, (N - 1).bit_length())):   # paths of 1, 2, 4 .. steps
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _run_plain_tree(s):
    c = s["case"]
    E, H, Hk, N, D, L, page = (c[x] for x in ("E", "H", "Hk", "N", "D", "L", "page"))
    per = s["page_table"].shape[1]
    table = s["page_table"].long()

    def rows(codes, scales):
        x = codes[0].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x = x.view(E, per, Hk, page // BLOCK, BLOCK, D) * scales[0][table][..., None, None]
        return x.view(E, per, Hk, page, D).transpose(1, 2).reshape(E, Hk, per * page, D)[:, :, :L]

    q = s["q"].float().reshape(E, Hk, H // Hk, N, D).flatten(2, 3)
    score = torch.matmul(q, rows(s["k_cache"], s["k_scale"]).transpose(-1, -2)).view(E, Hk, H // Hk, N, L) * D ** -0.5
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    count = _counts(s)
    start = (s["lengths"].long() - count)[:, None]
    reach = _descent(s["parents"])
    position = start + reach.sum(-1) - 1                                  # of the call's tokens
    at = torch.arange(L, device=q.device).expand(E, L)
    m = (at - start).clamp(0, N - 1)
    cached = at < start
    seen = torch.where(cached[:, None], True, reach.gather(2, m[:, None].expand(-1, N, -1)) & (at - start < count[:, None])[:, None])
    if c["window"]:
        seen = seen & (torch.where(cached, at, position.gather(1, m))[:, None] > position[..., None] - c["window"])
    seen = (seen & (torch.arange(N, device=q.device) < count[:, None])[..., None])[:, None, None]
    score = score.masked_fill(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p.flatten(2, 3), rows(s["v_cache"], s["v_scale"])).view(E, H, N, D).to(s["q"].dtype)
    return out.transpose(1, 2).contiguous().transpose(1, 2) if c["layout"] == "tokens" else out


def _turned(x, cos, sin, pairs):
    """x's rows rotated, in 32 bits."""
    x = x.float()
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if pairs == "half" else (x[..., 0::2], x[..., 1::2])
    y = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat(y, -1) if pairs == "half" else torch.stack(y, -1).flatten(-2)


def _held(amax):
    """The smallest power of two, from 2^-40 to 2^60, of which 448 hold the largest magnitude of a block."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8).clamp(-40, 60))


def _blocks_at(s, start, moved):
    """Slots of the blocks from ``start`` on that N tokens can touch: (position, page, slot in the page); ``moved(position)``: which are in use.
    The others stand for the last block of a sequence's pages, which is not in use and gets back what it had."""
    N, page = s["case"]["N"], s["case"]["page"]
    blocks = (N + BLOCK - 2) // BLOCK + 1
    at = (start // BLOCK * BLOCK)[:, None] + torch.arange(blocks * BLOCK, device=start.device)
    there = torch.where(moved(at), at, s["page_table"].shape[1] * page - BLOCK + at % BLOCK)
    return at, s["page_table"].long().gather(1, there // page), there % page


def _run_plain_place(s):
    c = s["case"]
    E, N, D, Hk = c["E"], c["N"], c["D"], c["Hk"]
    dev = s["k"].device
    end, count = s["lengths"].long(), _counts(s)
    start = end - count
    depth = _descent(s["parents"]).sum(-1) - 1
    angle = (start[:, None] + depth).double()[:, None, :, None] * s["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    k = _turned(s["k"], cos, sin, c["pairs"])
    q = _turned(s["q"], cos, sin, c["pairs"]).to(s["q"].dtype)
    q = torch.where((torch.arange(N, device=dev) < count[:, None])[:, None, :, None], q, torch.zeros((), dtype=q.dtype, device=dev))
    at, pages, slot = _blocks_at(s, start, lambda p: p < end[:, None])
    held, new = at < start[:, None], (at >= start[:, None]) & (at < end[:, None])
    blocks = at.shape[1] // BLOCK
    source = (at - start[:, None]).clamp(0, N - 1)[:, None, :, None].expand(-1, Hk, -1, D)

    def write(codes, scales, x):
        x = x.float().gather(2, source).view(E, Hk, blocks, BLOCK, D)
        is_new, is_held = (m.view(E, 1, blocks, BLOCK, 1) for m in (new, held))
        raw = codes.view(torch.uint8)
        before = raw[pages, :, slot].permute(0, 2, 1, 3).reshape(E, Hk, blocks, BLOCK, D)
        old = scales[pages, :, slot // BLOCK].permute(0, 2, 1).reshape(E, Hk, blocks, BLOCK)[..., 0]
        fresh = _held(torch.where(is_new, x.abs(), 0.0).amax((-1, -2)))
        any_new, any_held = new.view(E, 1, blocks, BLOCK).any(-1), held.view(E, 1, blocks, BLOCK).any(-1)
        scale = torch.where(any_held, torch.where(any_new, torch.maximum(fresh, old), old), fresh)
        kept = before.view(torch.float8_e4m3fn).float() * (old / scale)[..., None, None]
        value = torch.where(is_new, (x / scale[..., None, None]).clamp(-448.0, 448.0), kept).to(torch.float8_e4m3fn).view(torch.uint8)
        value = torch.where(is_new | is_held, value, before)
        raw[pages, :, slot] = value.view(E, Hk, -1, D).permute(0, 2, 1, 3)
        scale = torch.where(any_new | any_held, scale, old)
        scales[pages[:, ::BLOCK], :, slot[:, ::BLOCK] // BLOCK] = scale.permute(0, 2, 1)

    write(s["k_cache"][0], s["k_scale"][0], k)
    write(s["v_cache"][0], s["v_scale"][0], s["v"])
    return {"q": q, **{n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _accepted(s):
    """(E, N) tokens that stand, and how many."""
    N = s["case"]["N"]
    n = torch.arange(N, device=s["drafted"].device)
    parent = s["parents"].long()
    fits = (parent >= 0) & (s["drafted"] == s["answers"].gather(1, parent.clamp_min(0)))
    fits[:, 0] = True
    fits &= n < _counts(s)[:, None]
    beaten = (fits[:, None] & (parent[:, :, None] == parent[:, None]) & (n < n[:, None])).any(-1)   # by an earlier one of the same parent
    fits = fits & ~beaten
    stands = ~(_descent(s["parents"]) & ~fits[:, None]).any(-1)
    return stands, stands.sum(-1)


def _run_plain_accept(s):
    c = s["case"]
    E, N, D, Hk, layers, page = (c[x] for x in ("E", "N", "D", "Hk", "layers", "page"))
    dev = s["drafted"].device
    start = s["lengths"].long() - _counts(s)
    stands, taken = _accepted(s)
    n = torch.arange(N, device=dev)
    path = torch.where(stands, n, N).sort(-1).values
    answer = s["answers"].gather(1, path.gather(1, (taken - 1).clamp_min(0)[:, None]).clamp_max(N - 1))[:, 0]
    answer = torch.where(taken > 0, answer, -1)
    in_place = (path == n).sum(-1)                                       # so many of them are where they belong
    lo, hi = (start + in_place)[:, None], (start + taken)[:, None]
    touched = (lo < hi)
    at, pages, slot = _blocks_at(s, torch.where(touched[:, 0], start + in_place, start), lambda p: touched & (p < hi))
    moved, stays = (at >= lo) & (at < hi), touched & (at < lo)
    blocks = at.shape[1] // BLOCK
    origin = start[:, None] + path.gather(1, (at - start[:, None]).clamp(0, N - 1)).clamp_max(N - 1)
    origin = torch.where(moved, origin, s["page_table"].shape[1] * page - BLOCK)
    from_page, from_slot = s["page_table"].long().gather(1, origin // page), origin % page

    def write(codes, scales):
        raw = codes.view(torch.uint8)

        def look(p, i):                                                  # (layers, Hk, E, blocks, BLOCK, D) codes and their scales
            x = raw[:, p, :, i].permute(2, 3, 0, 1, 4).reshape(layers, Hk, E, blocks, BLOCK, D)
            return x, scales[:, p, :, i // BLOCK].permute(2, 3, 0, 1).reshape(layers, Hk, E, blocks, BLOCK)

        before, old = look(pages, slot)
        x, xs = look(from_page, from_slot)
        x = x.view(torch.float8_e4m3fn).float() * xs[..., None]
        is_moved, is_stay = (m.view(E, blocks, BLOCK, 1) for m in (moved, stays))
        old = old[..., 0]
        need = _held(torch.where(is_moved, x.abs(), 0.0).amax((-1, -2)))
        any_moved, any_stay = (m.view(E, blocks, BLOCK).any(-1) for m in (moved, stays))
        scale = torch.where(any_moved, torch.where(any_stay, torch.maximum(need, old), need), old)
        kept = before.view(torch.float8_e4m3fn).float() * (old / scale)[..., None, None]
        value = torch.where(is_moved, x / scale[..., None, None], kept).to(torch.float8_e4m3fn).view(torch.uint8)
        value = torch.where(is_moved | (is_stay & any_moved[..., None, None]), value, before)
        raw[:, pages, :, slot] = value.view(layers, Hk, E, -1, D).permute(2, 3, 0, 1, 4)
        scales[:, pages[:, ::BLOCK], :, slot[:, ::BLOCK] // BLOCK] = scale.permute(2, 3, 0, 1)

    write(s["k_cache"], s["k_scale"])
    write(s["v_cache"], s["v_scale"])
    return {"lengths": (start + taken).to(torch.int32), "path": torch.where(path < N, path, -1).to(torch.int32), "answer": answer,
            **{x: s[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _run_plain_fork(s):
    c, page = s["case"], s["case"]["page"]
    table, uses, lengths = s["page_table"].long(), s["page_uses"].long(), s["lengths"].long()
    E, P = table.shape
    pages = uses.numel()
    dev = table.device
    row, column = torch.arange(E, device=dev), torch.arange(P, device=dev)
    source, room = s["source"].long(), s["room"].long()
    holds = (table >= 0).long().cumprod(1) > 0
    goes_on = source >= 0
    of = source.clamp_min(0)
    length = torch.where(goes_on, lengths[of], 0)
    full, need = length // page, (length + room + page - 1) // page
    # the row that keeps the pages behind the full ones: the row itself where it goes on from itself, else the first that goes on from it
    claim = torch.where(source == row, -1, row)
    keeper = torch.full((E + 1,), E, device=dev).scatter_reduce(0, torch.where(goes_on, of, E), claim, "amin")
    keeps = goes_on & (keeper[of] == claim)
    theirs = table[of]
    shared = goes_on[:, None] & (column < full[:, None])
    behind = keeps[:, None] & holds[of] & (column < need[:, None]) & (uses[theirs.clamp_min(0)] == 1)
    kept = (shared | behind | (column < full[:, None])).long().cumprod(1).bool() & (shared | behind)

    def count(entries, which):
        return torch.zeros(pages + 1, dtype=torch.long, device=dev).scatter_add(
            0, torch.where(which, entries, pages).flatten(), torch.ones(E * P, dtype=torch.long, device=dev))[:pages]

    uses = uses - count(table, holds) + count(theirs, kept)
    wanted = (column < need[:, None]) & ~kept
    # a page that is partly filled and stays with another row is copied, and not given out in this call
    at = full.clamp_max(P - 1)[:, None]
    tokens = length - full * page
    copies = goes_on & (tokens > 0) & ~kept.gather(1, at)[:, 0]
    read = count(theirs.gather(1, at).expand(E, P), copies[:, None] & (column == 0))
    free = torch.sort((uses + read != 0).to(torch.uint8), stable=True).indices   # free pages, the lowest first
    given = free[(wanted.flatten().long().cumsum(0) - 1).clamp(0, pages - 1)].view(E, P)
    new = torch.where(kept, theirs, torch.where(wanted, given, -1))
    uses = uses + count(given, wanted)
    src, dst = theirs.gather(1, at)[:, 0][copies], new.gather(1, at)[:, 0][copies]
    slot = torch.arange(page, device=dev)
    block = (slot < ((tokens[copies] + BLOCK - 1) // BLOCK * BLOCK)[:, None]).view(1, -1, 1, page, 1)
    for name in ("k", "v"):
        raw, scales = s[name + "_cache"].view(torch.uint8), s[name + "_scale"]
        raw[:, dst] = torch.where(block, raw[:, src], raw[:, dst])
        scales[:, dst] = torch.where(block[:, :, :, ::BLOCK, 0], scales[:, src], scales[:, dst])
    s["page_table"].copy_(new)
    s["page_uses"].copy_(uses)
    s["lengths"].copy_(length)
    return {n: s[n] for n in ("page_uses", "page_table", "lengths", "k_cache", "v_cache", "k_scale", "v_scale")}


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _run_plain_tree, "place": _run_plain_place, "accept": _run_plain_accept, "fork": _run_plain_fork}[state["case"]["op"]](state)


def work(case):
    E, Hk, D, L, page = (case[x] for x in ("E", "Hk", "D", "L", "page"))
    if case["op"] == "fork":
        # tables and counts in and out; the rows that neither stay nor end copy half a page as a mean
        P, layers = (L + page - 1) // page + 1, case["layers"]
        copied = 0.6 * E * (1 - 1 / case["beams"]) * (1 - case["ending"]) * page / 2
        return {"bytes": 4 * (2 * E * P + 2 * (E * P + 7) + 4 * E) + 4 * copied * layers * Hk * (D + 4 / BLOCK), "flops": 0}
    N = case["N"]
    real = 0.5 if case["counts"] else 1.0   # of the call's tokens, as a mean
    if case["op"] == "accept":
        # tokens of a tree of depth ln N of which some stand, but for the first, read and written in all layers
        moved = E * max(0.1, min(2.0, 0.5 * math.log(max(1.1, real * N))))
        return {"bytes": 4 * moved * case["layers"] * Hk * (D + 4 / BLOCK) + E * N * (4 + 16 + 4), "flops": 0}
    H = case["H"]
    if case["op"] == "place":
        fresh = real * E * N * D * Hk
        return {"bytes": 2 * (real * E * N * D * H + E * N * D * H + 2 * fresh) + 2 * fresh, "flops": 3 * real * E * N * D * (H + 2 * Hk)}
    tokens = (N + L) / 2 if case["ragged"] else L
    seen = min(tokens, case["window"] + real * N) if case["window"] else tokens
    return {"bytes": 2 * E * seen * Hk * (D + 4 / BLOCK) + 2 * (1 + real) * E * N * H * D, "flops": 4 * real * E * N * H * D * seen}


# --- the definitions in 64 bits, a sequence at a time --------------------------------------------------------------------

def _chain(parents, n):
    """Token n and its ancestors, the nearest first."""
    chain = []
    while n >= 0:
        chain.append(n)
        n = parents[n]
    return chain


def _sequence(s, e):
    length = int(s["lengths"][e])
    count = s["case"]["N"] if s["counts"] is None else int(s["counts"][e])
    return length - count, count


def _exact_tree(s):
    c, page = s["case"], s["case"]["page"]
    group = c["H"] // c["Hk"]
    out = torch.zeros(c["E"], c["H"], c["N"], c["D"], dtype=torch.float64, device=s["q"].device)
    for e in range(c["E"]):
        start, count = _sequence(s, e)
        length = start + count
        parents = s["parents"][e].tolist()
        sees = torch.ones(count, length, dtype=torch.bool)
        sees[:, start:] = False
        for n in range(count):
            chain = _chain(parents, n)
            if c["window"]:
                sees[n, :max(0, min(start, start + len(chain) - c["window"]))] = False
                chain = chain[:c["window"]]
            sees[n, [start + m for m in chain]] = True
        sees = sees.to(out.device)
        used = s["page_table"][e, :(length + page - 1) // page].long()
        for h in range(c["Hk"]):
            k, v = ((s[n + "_cache"][0].view(torch.uint8)[used, h].view(torch.float8_e4m3fn).double()
                     * s[n + "_scale"][0][used, h].double().repeat_interleave(BLOCK, -1)[..., None]).reshape(-1, c["D"])[:length] for n in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                w = s["q"][e, j, :count].double() @ k.T / math.sqrt(c["D"])
                if c["softcap"]:
                    w = c["softcap"] * torch.tanh(w / c["softcap"])
                out[e, j, :count] = torch.softmax(w.masked_fill(~sees, -math.inf), -1) @ v
    return out


def _exact_turn(x, position, f, pairs):
    """x (heads, N, D) in 64 bits as complex numbers turned by position * f."""
    turn = torch.polar(torch.ones(position.numel(), len(f), dtype=torch.float64, device=x.device), torch.outer(position.double(), f))
    first = torch.arange(len(f), device=x.device) * (1 if pairs == "half" else 2)
    second = first + (len(f) if pairs == "half" else 1)
    y = x.double().clone()
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_step(most):
    """The scale that 448 of hold ``most`` in 64 bits."""
    step = torch.exp2(torch.ceil(torch.log2(most.clamp_min(1e-300) / 448.0)).clamp(-39, 60))
    return torch.where(most <= 224.0 * step, step / 2, step)   # where the logarithm of a power of two came out above it


def _exact_place(s):
    """The held values before their rounding to 8 bits: what is stored is these to within half a step."""
    c, page = s["case"], s["case"]["page"]
    q = torch.zeros_like(s["q"], dtype=torch.float64)
    held = {n: s[n + "_cache"].double() for n in ("k", "v")}
    scale = {n: s[n + "_scale"].double().clone() for n in ("k", "v")}
    for e in range(c["E"]):
        start, count = _sequence(s, e)
        parents = s["parents"][e].tolist()
        position = torch.tensor([start + len(_chain(parents, n)) - 1 for n in range(count)], device=q.device)
        new = {"k": _exact_turn(s["k"][e, :, :count], position, s["frequencies"], c["pairs"]), "v": s["v"][e, :, :count].double()}
        q[e, :, :count] = _exact_turn(s["q"][e, :, :count], position, s["frequencies"], c["pairs"])
        for block in range(start // BLOCK, (start + count - 1) // BLOCK + 1):
            lo, hi = max(start, block * BLOCK), min(start + count, (block + 1) * BLOCK)
            at, row = int(s["page_table"][e, block * BLOCK // page]), block * BLOCK % page
            for n in ("k", "v"):
                x = new[n][:, lo - start:hi - start]
                step, older = _exact_step(x.abs().amax((-1, -2))), lo - block * BLOCK
                if older:
                    before = scale[n][0, at, :, row // BLOCK].clone()
                    step = torch.maximum(step, before)
                    held[n][0, at, :, row:row + older] *= (before / step)[:, None, None]
                held[n][0, at, :, row + older:row + hi - block * BLOCK] = x / step[:, None, None]
                scale[n][0, at, :, row // BLOCK] = step
    return {"q": q, "k_cache": held["k"], "v_cache": held["v"], "k_scale": scale["k"], "v_scale": scale["v"]}


def _exact_accept(s):
    """The closed-up caches before any rounding of codes that change their scale."""
    c, page = s["case"], s["case"]["page"]
    held = {n: s[n + "_cache"].double() for n in ("k", "v")}
    scale = {n: s[n + "_scale"].double().clone() for n in ("k", "v")}
    table = s["page_table"].tolist()
    drafted, answers, parents = (s[n].tolist() for n in ("drafted", "answers", "parents"))
    for e in range(c["E"]):
        start, count = _sequence(s, e)
        path = [0] if count else []
        while path:
            fit = [n for n in range(count) if parents[e][n] == path[-1] and drafted[e][n] == answers[e][path[-1]]]
            if not fit:
                break
            path.append(fit[0])
        ahead = [i for i, n in enumerate(path) if n != i]
        if not ahead:
            continue
        place = lambda p: (table[e][p // page], p % page)  # noqa: E731
        for n in ("k", "v"):
            values = {}
            for i in ahead:
                at, row = place(start + path[i])
                values[start + i] = held[n][:, at, :, row] * scale[n][:, at, :, row // BLOCK, None]
            for block in range((start + ahead[0]) // BLOCK, (start + len(path) - 1) // BLOCK + 1):
                at, row = place(block * BLOCK)
                here = [p for p in range(block * BLOCK, (block + 1) * BLOCK) if p in values]
                step, stay = _exact_step(torch.stack([values[p] for p in here]).abs().amax((0, -1))), here[0] - block * BLOCK
                before = scale[n][:, at, :, row // BLOCK].clone()
                if stay:
                    step = torch.maximum(step, before)
                    held[n][:, at, :, row:row + stay] *= (before / step)[..., None, None]
                for p in here:
                    held[n][:, at, :, row + p - block * BLOCK] = values[p] / step[..., None]
                scale[n][:, at, :, row // BLOCK] = step
    return {"lengths": None, "path": None, "answer": None, "k_cache": held["k"], "v_cache": held["v"], "k_scale": scale["k"], "v_scale": scale["v"]}


def exact(case, seed):
    if case["op"] == "fork":   # whole numbers and copies: nothing is computed
        return None
    s = prepare(case, seed)
    return {"tree": _exact_tree, "place": _exact_place, "accept": _exact_accept}[case["op"]](s)
