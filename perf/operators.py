"""What a user of the rotary positions, the paged 8-bit key/value cache and the attention over it has them do.

``listed()`` gives the representative calls, ``draw(rng)`` more of the same ranges.  ``run`` computes one call: with
``own`` through the library's entry points, else in elementary tensor operations in 32 bits (angles in 64).

Fields of a case: ``op`` (``rotary``, ``append``, ``attend``), ``E`` batch, ``H`` query heads, ``Hk`` key/value heads,
``N`` new tokens of a sequence, ``D`` head width, ``dtype``, ``layout`` (``heads``: contiguous (E, H, N, D) tensors;
``tokens``: (E, H, N, D) views of (E, N, H, D) projections).  Rotation: ``dim`` (0: none), ``pairs`` (``half`` or
``interleaved``), ``scaling``, ``factor``; ``train`` adds the backward pass; ``where`` says how positions come
(``range``: 0..N-1, ``given``: a tensor, from a far offset).  Cache: ``L`` most tokens of a sequence, those of the call
among them, ``page`` tokens of a page, ``ragged`` lengths; ``counts``: sequences bring fewer than N tokens; ``causal``,
``softcap`` and ``window`` (0: none) of the attention.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BASE = 10000.0
SCALED_FROM = 4096   # length that scaled positions were trained for
BLOCK = 16           # tokens that share a scale
PEAK_ELEMENTS = 65536 * 20 * 128          # most elements of a rotation
PEAK_CACHE = 32 * 8 * 8192 * 128          # most elements of the keys that an attention reads
PEAK_SCORES = 2 * 16 * 1024 * 16384       # most scores of one


def _rotary(name, E, H, Hk, N, D, dtype, dim, pairs, scaling="none", factor=1.0, train=False, where="range", layout="tokens"):
    return dict(name=name, op="rotary", E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, dim=dim, pairs=pairs, scaling=scaling,
                factor=factor, train=train, where=where, layout=layout)


def _append(name, E, H, Hk, N, D, dtype, L, page, dim, pairs="half", scaling="none", factor=1.0, ragged=True, counts=False, layout="tokens"):
    return dict(name=name, op="append", E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, dim=dim, pairs=pairs,
                scaling=scaling, factor=factor, ragged=ragged, counts=counts, layout=layout)


def _attend(name, E, H, Hk, N, D, dtype, L, page, ragged=True, counts=False, causal=True, softcap=0.0, window=0, layout="tokens"):
    return dict(name=name, op="attend", E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, ragged=ragged,
                counts=counts, causal=causal, softcap=softcap, window=window, layout=layout)


def listed():
    return [
        # one sentence through an encoder layer with rotary positions: latency is all of it
        _rotary("rotary_sentence", 1, 12, 12, 33, 64, "f16", 64, "half"),
        # fine-tuning at 1024 tokens in full precision, half of each head rotated: forward and backward
        _rotary("rotary_train_1024", 4, 12, 12, 1024, 64, "f32", 32, "interleaved", train=True),
        # long documents far beyond the trained length, at explicit positions
        _rotary("rotary_documents_7683", 4, 12, 12, 7683, 64, "f16", 64, "half", "ntk", 4.0, where="given"),
        # the longest sequence, grouped heads, scaled by parts
        _rotary("rotary_65536", 1, 16, 4, 65536, 128, "bf16", 128, "interleaved", "yarn", 16.0),
        # one token of a few sequences: the append of an interactive decoder
        _append("append_token", 8, 12, 12, 1, 64, "bf16", 700, 16, 64),
        # one token of a serving batch, grouped heads
        _append("append_token_batch", 256, 32, 8, 1, 128, "bf16", 512, 64, 128),
        # prompts of a serving batch, padded behind to the longest
        _append("append_prompts", 8, 16, 4, 1999, 128, "bf16", 2100, 64, 128, "interleaved", counts=True),
        # one token of one sequence: latency
        _attend("attend_token", 1, 12, 12, 1, 64, "f16", 500, 16, ragged=False),
        # one token of a serving batch of ragged lengths
        _attend("attend_batch", 32, 32, 8, 1, 128, "bf16", 8192, 64),
        # one token of one long context: few heads, the length has to be split
        _attend("attend_long", 1, 16, 2, 1, 128, "bf16", 131071, 128, ragged=False),
        # a few proposed tokens verified at once, capped scores, sliding window, sequences with fewer proposals
        _attend("attend_verify", 16, 16, 4, 5, 128, "f16", 4096, 32, counts=True, softcap=30.0, window=1024),
        # a piece of a prompt against what is already cached
        _attend("attend_prompt", 2, 16, 4, 1024, 128, "bf16", 16384, 64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "attend", "attend", "attend"])
    D = rng.choice([64, 64, 128, 128, 128])
    group = rng.choice([1, 1, 2, 4, 4, 5, 8])
    Hk = rng.choice([1, 2, 4, 8, 12] if group < 8 else [1, 2, 4, 8])
    H = Hk * group
    layout = rng.choice(["tokens", "tokens", "heads"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "rotary":
        D = rng.choice([32, 64, 64, 72, 80, 128])     # the models' widths
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        train = rng.random() < 0.4
        room = PEAK_ELEMENTS // (4 if train or dtype == "f32" else 1)
        N = _log_int(rng, 1, min(65536, room // ((H + Hk) * D)))
        E = _log_int(rng, 1, max(1, min(64, room // ((H + Hk) * D * N))))
        scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
        return dict(op=op, E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, dim=rng.choice([D, D, D // 2]), pairs=rng.choice(["half", "interleaved"]),
                    scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]), train=train,
                    where=rng.choice(["range", "given"]), layout=layout)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        N = rng.choice([1, 1, rng.randint(2, 40), _log_int(rng, 41, 4000)])
        L = N + _log_int(rng, 1, 4000)
        E = _log_int(rng, 1, max(1, min(256, PEAK_CACHE // (4 * L * Hk * D), PEAK_CACHE // (4 * N * H * D))))
        scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
        return dict(op=op, E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, dim=rng.choice([D, D, D // 2, 0]),
                    pairs=rng.choice(["half", "interleaved"]), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0]),
                    ragged=True, counts=rng.random() < 0.5, layout=layout)
    N = rng.choice([1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 1024)])
    L = N + _log_int(rng, 1, min(131071, PEAK_SCORES // (4 * N * H), PEAK_CACHE // (2 * Hk * D)) - N)
    E = _log_int(rng, 1, max(1, min(64, PEAK_SCORES // (4 * N * H * L), PEAK_CACHE // (2 * Hk * D * L))))
    causal = rng.random() < 0.8
    return dict(op=op, E=E, H=H, Hk=Hk, N=N, D=D, dtype=dtype, L=L, page=page, ragged=rng.random() < 0.7, counts=N > 1 and rng.random() < 0.5,
                causal=causal, softcap=rng.choice([0.0, 0.0, 20.0]), window=rng.choice([0, 0, rng.randint(1, L)]) if causal else 0, layout=layout)


def frequencies(case):
    """Radians per position of each pair, in 64 bits, and what sine and cosine are multiplied by."""
    dim, factor = case["dim"], case["factor"]
    base = BASE * factor ** (dim / (dim - 2)) if case["scaling"] == "ntk" else BASE
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if case["scaling"] == "linear":
        f = [x / factor for x in f]
    if case["scaling"] == "yarn":   # by parts: pairs of under 1 turn in the trained length interpolated, of over 32 left as they are
        kept = [min(1.0, max(0.0, (SCALED_FROM * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
        f = [x * (g + (1 - g) / factor) for x, g in zip(f, kept)]
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    E, H, Hk, N, D, dtype = (case[x] for x in ("E", "H", "Hk", "N", "D", "dtype"))
    dtype = DTYPES[dtype]

    def heads(h, std):
        # projected hidden states: a spread and an offset of each channel of a head
        shape = (E, h, N, D) if case["layout"] == "heads" else (E, N, h, D)
        t = torch.randn(shape, generator=g, device=dev)
        t = t if case["layout"] == "heads" else t.permute(0, 2, 1, 3)
        t.mul_(std).add_(0.3 * torch.randn(1, h, 1, D, generator=g, device=dev))
        return t.to(dtype)

    state = dict(case=case, q=heads(H, 1.5))
    if case.get("dim"):
        f, state["magnitude"] = frequencies(case)
        state["frequencies"] = torch.tensor(f, dtype=torch.float64, device=dev)
    if case["op"] == "rotary":
        state["k"], state["positions"] = heads(Hk, 1.5), None
        if case["where"] == "given":
            first = torch.randint(0, 1000000, (E, 1), generator=g, device=dev)
            state["positions"] = first + torch.arange(N, device=dev)
        if case["train"]:
            state["grads"] = (heads(H, 1.0), heads(Hk, 1.0))
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
        return state
    L, page = case["L"], case["page"]
    counts = torch.full((E,), N, device=dev)
    if case["counts"]:
        counts = torch.randint(0, N + 1, (E,), generator=g, device=dev)
    lengths = torch.full((E,), L, device=dev)
    if case["ragged"]:
        lengths = torch.randint(N, L + 1, (E,), generator=g, device=dev)
    per = (L + 2 * BLOCK + page - 1) // page
    pages = E * per
    state["page_table"] = torch.randperm(pages, generator=g, device=dev).view(E, per).to(torch.int32)
    state["lengths"] = lengths.to(torch.int32)
    state["counts"] = counts.to(torch.int32) if case["counts"] else None
    for name in ("k", "v"):   # pages in use, rows behind a sequence's end hold what was there before
        codes = torch.empty(pages, Hk, page, D, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty(pages, Hk, page // BLOCK, device=dev)
        offset = 0.3 * torch.randn(1, Hk, 1, D, generator=g, device=dev)
        step = max(1, (1 << 27) // (Hk * page * D))
        for i in range(0, pages, step):
            x = torch.randn(codes[i:i + step].shape, generator=g, device=dev).mul_(1.5).add_(offset)
            x = x.view(-1, Hk, page // BLOCK, BLOCK, D)
            s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448.0)))
            codes[i:i + step] = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(-1, Hk, page, D)
            scales[i:i + step] = s
        state[name + "_cache"], state[name + "_scale"] = codes, scales
    if case["op"] == "append":
        state["k"], state["v"] = heads(Hk, 1.5), heads(Hk, 1.5)
    return state


@functools.lru_cache(maxsize=64)
def _handle(dim, pairs, scaling, factor):
    from monarch_attention_b200 import RotaryPositions
    return RotaryPositions(dim, base=BASE, pairs=pairs, scaling=None if scaling == "none" else scaling, factor=factor,
                           trained_length=SCALED_FROM)


def _run_own(s):
    from monarch_attention_b200 import PagedKV, append_kv_b200, cached_attention_b200, rotary_b200
    c = s["case"]
    rotary = _handle(c["dim"], c["pairs"], c["scaling"], c["factor"]) if c.get("dim") else None
    if c["op"] == "rotary":
        q, k = rotary_b200(s["q"], s["k"], rotary, s["positions"])
        if c["train"]:
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), s["grads"])
            return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
        return {"q": q, "k": k}
    cache = PagedKV(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if c["op"] == "append":
        q = append_kv_b200(cache, s["k"], s["v"], s["page_table"], s["lengths"], s["counts"], query=s["q"], rotary=rotary)
        return {"q": q, "k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    return cached_attention_b200(s["q"], cache, s["page_table"], s["lengths"], s["counts"], causal=c["causal"],
                                 softcap=c["softcap"], window=c["window"], token_major_output=c["layout"] == "tokens")


def _turned(x, cos, sin, dim, pairs):
    """The first ``dim`` features of x's rows rotated, the others as they are, in 32 bits."""
    x = x.float()
    a, b = (x[..., :dim // 2], x[..., dim // 2:dim]) if pairs == "half" else (x[..., 0:dim:2], x[..., 1:dim:2])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.cat(y, -1) if pairs == "half" else torch.stack(y, -1).flatten(-2)
    return torch.cat((y, x[..., dim:]), -1)


def _run_plain_rotary(s):
    c = s["case"]
    p = s["positions"] if s["positions"] is not None else torch.arange(c["N"], device=s["q"].device)[None]
    angle = p.double()[:, None, :, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    q, k = (_turned(s[n], cos, sin, c["dim"], c["pairs"]).to(s[n].dtype) for n in ("q", "k"))
    if c["train"]:
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), s["grads"])
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    return {"q": q, "k": k}


def _held(amax):
    """The smallest power of two, from 2^-40 to 2^60, of which 448 hold the largest magnitude of a block."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8).clamp(-40, 60))


def _run_plain_append(s):
    c = s["case"]
    E, N, D, page = c["E"], c["N"], c["D"], c["page"]
    dev = s["k"].device
    end = s["lengths"].long()
    start = end - (s["counts"].long() if s["counts"] is not None else N)
    rows = torch.arange(N, device=dev)
    q, k = s["q"], s["k"].float()
    if c["dim"]:
        angle = (start[:, None] + rows).double()[:, None, :, None] * s["frequencies"]
        cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
        k = _turned(k, cos, sin, c["dim"], c["pairs"])
        q = _turned(q, cos, sin, c["dim"], c["pairs"]).to(q.dtype)
    if s["counts"] is not None:   # rows of padding give zeros
        q = torch.where((rows < s["counts"][:, None])[:, None, :, None], q, torch.zeros((), dtype=q.dtype, device=dev))
    blocks = (N + BLOCK - 2) // BLOCK + 1
    at = (start // BLOCK * BLOCK)[:, None] + torch.arange(blocks * BLOCK, device=dev)
    held, new = at < start[:, None], (at >= start[:, None]) & (at < end[:, None])
    # slots that hold nothing stand for the last block of the sequence's pages, which is not in use and gets back what it had
    at = torch.where(held | new, at, s["page_table"].shape[1] * page - BLOCK + at % BLOCK)
    pages = s["page_table"].long().gather(1, at // page)
    slot = at % page
    source = (at - start[:, None]).clamp(0, N - 1)[:, None, :, None].expand(-1, c["Hk"], -1, D)

    def write(codes, scales, x):
        x = x.float().gather(2, source).view(E, c["Hk"], blocks, BLOCK, D)
        is_new, is_held = (m.view(E, 1, blocks, BLOCK, 1) for m in (new, held))
        raw = codes.view(torch.uint8)
        before = raw[pages, :, slot].permute(0, 2, 1, 3).reshape(E, c["Hk"], blocks, BLOCK, D)
        old = scales[pages, :, slot // BLOCK].permute(0, 2, 1).reshape(E, c["Hk"], blocks, BLOCK)[..., 0]
        fresh = _held(torch.where(is_new, x.abs(), 0.0).amax((-1, -2)))
        any_new, any_held = new.view(E, 1, blocks, BLOCK).any(-1), held.view(E, 1, blocks, BLOCK).any(-1)
        scale = torch.where(any_held, torch.where(any_new, torch.maximum(fresh, old), old), fresh)
        kept = before.view(torch.float8_e4m3fn).float() * (old / scale)[..., None, None]
        value = torch.where(is_new, (x / scale[..., None, None]).clamp(-448.0, 448.0), kept).to(torch.float8_e4m3fn).view(torch.uint8)
        value = torch.where(is_new | is_held, value, before)
        raw[pages, :, slot] = value.view(E, c["Hk"], -1, D).permute(0, 2, 1, 3)
        scale = torch.where(any_new | any_held, scale, old)
        scales[pages[:, ::BLOCK], :, slot[:, ::BLOCK] // BLOCK] = scale.permute(0, 2, 1)

    write(s["k_cache"], s["k_scale"], k)
    write(s["v_cache"], s["v_scale"], s["v"])
    return {"q": q, "k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _run_plain_attend(s):
    c = s["case"]
    E, H, Hk, N, D, page = (c[x] for x in ("E", "H", "Hk", "N", "D", "page"))
    per = s["page_table"].shape[1]
    table = s["page_table"].long()

    def rows(codes, scales):
        x = codes.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x = x.view(E, per, Hk, page // BLOCK, BLOCK, D) * scales[table][..., None, None]
        return x.view(E, per, Hk, page, D).transpose(1, 2).reshape(E, Hk, per * page, D)[:, :, :c["L"]]

    q = s["q"].float().reshape(E, Hk, H // Hk, N, D).flatten(2, 3)
    score = torch.matmul(q, rows(s["k_cache"], s["k_scale"]).transpose(-1, -2)).view(E, Hk, H // Hk, N, c["L"]) * D ** -0.5
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    n, at = torch.arange(N, device=q.device), torch.arange(c["L"], device=q.device)
    counts = s["counts"].long() if s["counts"] is not None else torch.full((E,), N, device=q.device)
    last = s["lengths"].long()[:, None] - 1
    if c["causal"]:
        last = last - counts[:, None] + 1 + n
    last = last.expand(E, N)[..., None]
    seen = (at <= last) & (n < counts[:, None])[..., None]
    if c["window"]:
        seen = seen & (at > last - c["window"])
    seen = seen[:, None, None]
    score = score.masked_fill(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p.flatten(2, 3), rows(s["v_cache"], s["v_scale"])).view(E, H, N, D).to(s["q"].dtype)
    return out.transpose(1, 2).contiguous().transpose(1, 2) if c["layout"] == "tokens" else out


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return (_run_plain_rotary if op == "rotary" else _run_plain_append if op == "append" else _run_plain_attend)(state)


def work(case):
    E, H, Hk, N, D = (case[x] for x in ("E", "H", "Hk", "N", "D"))
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        passes = 2 if case["train"] else 1
        elements = E * N * D * (H + Hk)
        return {"bytes": passes * (2 * size * elements + (8 * E * N if case["where"] == "given" else 0)), "flops": passes * 3 * elements}
    real = 0.5 if case["counts"] else 1.0   # of the new tokens, as a mean
    if case["op"] == "append":
        fresh = real * E * N * D * Hk
        return {"bytes": real * E * N * D * H * size + E * N * D * H * size + 2 * fresh * (size + 1), "flops": 3 * real * E * N * D * (H + 2 * Hk)}
    L = (N + case["L"]) / 2 if case["ragged"] else case["L"]
    keys = min(L, case["window"] + real * N) if case["window"] else L
    seen = min(L, case["window"]) if case["window"] else L - (real * N / 2 if case["causal"] else 0)
    return {"bytes": 2 * E * keys * Hk * (D + 4 / BLOCK) + (1 + real) * E * N * H * D * size, "flops": 4 * real * E * N * H * D * seen}


# --- the definitions in 64 bits, a sequence and a head at a time -------------------------------------------------------

def _exact_rotation(x, position, f, magnitude, pairs):
    """x (heads, N, D) in 64 bits as complex numbers turned by position * f."""
    half = len(f)
    turn = torch.polar(torch.full((position.numel(), half), magnitude, dtype=torch.float64, device=x.device),
                       torch.outer(position.double(), f))
    y = x.double().clone()
    first = torch.arange(half, device=x.device) * (1 if pairs == "half" else 2)
    second = first + (half if pairs == "half" else 1)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_append(s):
    """The held values before their rounding to 8 bits: what is stored is these to within half a step."""
    c, page = s["case"], s["case"]["page"]
    q, out = torch.zeros_like(s["q"], dtype=torch.float64), {}
    held = {n: s[n + "_cache"].double() for n in ("k", "v")}
    scale = {n: s[n + "_scale"].double().clone() for n in ("k", "v")}
    for e in range(c["E"]):
        end = int(s["lengths"][e])
        count = c["N"] if s["counts"] is None else int(s["counts"][e])
        start = end - count
        if not count:
            continue
        position = torch.arange(start, end, device=q.device)
        new = {"k": s["k"][e, :, :count].double(), "v": s["v"][e, :, :count].double()}
        q[e, :, :count] = s["q"][e, :, :count].double()
        if c["dim"]:
            new["k"] = _exact_rotation(new["k"], position, s["frequencies"], s["magnitude"], c["pairs"])
            q[e, :, :count] = _exact_rotation(q[e, :, :count], position, s["frequencies"], s["magnitude"], c["pairs"])
        for block in range(start // BLOCK, (end - 1) // BLOCK + 1):
            lo, hi = max(start, block * BLOCK), min(end, (block + 1) * BLOCK)
            at, row = int(s["page_table"][e, block * BLOCK // page]), block * BLOCK % page
            for n in ("k", "v"):
                x = new[n][:, lo - start:hi - start]
                most = x.abs().amax((-1, -2))
                step = torch.exp2(torch.ceil(torch.log2(most.clamp_min(1e-300) / 448.0)).clamp(-39, 60))
                step = torch.where(most <= 224.0 * step, step / 2, step)   # where the logarithm of a power of two came out above it
                older = lo - block * BLOCK
                if older:
                    before = scale[n][at, :, row // BLOCK].clone()
                    step = torch.maximum(step, before)
                    held[n][at, :, row:row + older] *= (before / step)[:, None, None]
                held[n][at, :, row + older:row + hi - block * BLOCK] = x / step[:, None, None]
                scale[n][at, :, row // BLOCK] = step
    for n in ("k", "v"):
        out[n], out[n + "_scale"] = held[n], scale[n]
    return {"q": q, **out}


def _exact_attend(s):
    c, page = s["case"], s["case"]["page"]
    group = c["H"] // c["Hk"]
    out = torch.zeros(c["E"], c["H"], c["N"], c["D"], dtype=torch.float64, device=s["q"].device)
    for e in range(c["E"]):
        length = int(s["lengths"][e])
        count = c["N"] if s["counts"] is None else int(s["counts"][e])
        if not length or not count:
            continue
        used = s["page_table"][e, :(length + page - 1) // page].long()
        for h in range(c["Hk"]):
            k, v = ((s[n + "_cache"].view(torch.uint8)[used, h].view(torch.float8_e4m3fn).double()
                     * s[n + "_scale"][used, h].double().repeat_interleave(BLOCK, -1)[..., None]).reshape(-1, c["D"])[:length] for n in ("k", "v"))
            at = torch.arange(length, device=k.device)
            for j in range(group):
                w = s["q"][e, h * group + j, :count].double() @ k.T / math.sqrt(c["D"])
                if c["softcap"]:
                    w = c["softcap"] * torch.tanh(w / c["softcap"])
                if c["causal"]:
                    own_place = torch.arange(length - count, length, device=k.device)[:, None]
                    w = w.masked_fill(at > own_place, -math.inf)
                    if c["window"]:
                        w = w.masked_fill(at <= own_place - c["window"], -math.inf)
                out[e, h * group + j, :count] = torch.softmax(w, -1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    f, m = s["frequencies"], s["magnitude"]
    p = s["positions"] if s["positions"] is not None else torch.arange(case["N"], device=f.device).expand(case["E"], -1)
    out = {}
    with torch.no_grad():
        for n in ("q", "k"):
            out[n] = torch.stack([_exact_rotation(s[n][e], p[e], f, m, case["pairs"]) for e in range(case["E"])])
            if case["train"]:   # the transpose of a rotation turns back
                g = s["grads"]["qk".index(n)]
                out["d" + n] = torch.stack([_exact_rotation(g[e], -p[e], f, m, case["pairs"]) for e in range(case["E"])])
    return out
