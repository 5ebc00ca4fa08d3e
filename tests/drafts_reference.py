"""Definitions of drafted trees over the paged cache, of their acceptance and of forked sequences, token by token on the CPU."""
from __future__ import annotations

import math

import torch

from decoder_reference import attention

BLOCK = 16


def line(parents, n):
    """Token n and its ancestors, the nearest first; a parent that is no earlier token is none."""
    out = []
    while n >= 0:
        out.append(n)
        n = parents[n] if -1 <= parents[n] < n else -1
    return out


def trees(E, N, kind, seed=0):
    """(E, N) int32 parents on the GPU."""
    g = torch.Generator().manual_seed(seed)
    n = torch.arange(N).expand(E, N)
    if kind == "chain":
        p = n - 1
    elif kind == "star":      # no parents at all
        p = torch.full((E, N), -1)
    elif kind == "wide":      # all children of the first
        p = torch.where(n > 0, 0, -1)
    else:                     # any earlier token, or (forests) none
        p = torch.minimum((torch.rand(E, N, generator=g) * n).floor().long(), n - 1)
        if kind == "forest":
            p = torch.where(torch.rand(E, N, generator=g) < 0.2, -1, p)
    return p.to(torch.int32).cuda()


def seen_by_tree(parents, length, count, window):
    """(count, length): which keys the tokens of a tree see."""
    start = length - count
    seen = torch.zeros(count, length, dtype=torch.bool)
    for n in range(count):
        chain = line(parents, n)
        place = start + len(chain) - 1
        if start > 0:
            seen[n, max(0, max(place, 0) - window + 1) if window else 0:start] = True
        for m in chain[:window] if window else chain:
            if start + m >= 0:
                seen[n, start + m] = True
        if start + n < 0:
            seen[n] = False
    return seen


def tree_attention(q, k, v, seen, scale, softcap=0.0):
    """q (H, n, D) over k, v (Hk, L, D) where `seen` (n, L), in 64 bits: result and bound, a row at a time as attention without a mask over what it sees."""
    H, n, D = q.shape
    out, bound = torch.zeros(H, n, D, dtype=torch.float64), torch.zeros(H, n, D, dtype=torch.float64)
    most = v.abs().amax() if v.numel() else torch.zeros(())
    for r in range(n):
        at = seen[r].nonzero()[:, 0]
        if at.numel():
            o, b = attention(q[:, r:r + 1], k[:, at], v[:, at], 0, False, scale, softcap)
            # (weights below the f16 range count for all keys of the sequence, as in attention())
            out[:, r], bound[:, r] = o[:, 0], b[:, 0] + seen.shape[1] * 2.0 ** -24 * most
    return out, bound


def power_for(most):
    """The smallest power of two from 2^-40 to 2^60 of which 448 hold `most`."""
    if most == 0.0:
        return 2.0 ** -40
    m, e = math.frexp(most)
    return 2.0 ** min(max(e - 9 if m <= 0.875 else e - 8, -40), 60)


def accepted(parents, drafted, answers, count):
    path = [0] if count else []
    while path:
        fit = [n for n in range(path[-1] + 1, count) if (parents[n] if -1 <= parents[n] < n else -1) == path[-1] and drafted[n] == answers[path[-1]]]
        if not fit:
            return path
        path.append(fit[0])
    return path


def close_up(raw, scale, table, start, path, page):
    """raw (pages, heads, page, D) uint8 codes and scale (pages, heads, page / 16), changed in place."""
    ahead = [i for i, n in enumerate(path) if n != i]
    if not ahead:
        return
    where = lambda p: (int(table[p // page]), p % page)  # noqa: E731
    as_value = lambda c: c.view(torch.float8_e4m3fn).double()  # noqa: E731
    values = {}
    for i in ahead:
        at, row = where(start + path[i])
        values[start + i] = as_value(raw[at, :, row].contiguous()) * scale[at, :, row // BLOCK, None].double()
    for block in range((start + ahead[0]) // BLOCK, (start + len(path) - 1) // BLOCK + 1):
        at, row = where(block * BLOCK)
        here = [p for p in range(block * BLOCK, (block + 1) * BLOCK) if p in values]
        stay = here[0] - block * BLOCK
        for h in range(raw.shape[1]):
            most = max(float(torch.nan_to_num(values[p][h].abs(), nan=0.0).amax()) for p in here)
            step, before = power_for(most), float(scale[at, h, row // BLOCK])
            if stay:
                step = max(step, before)
                if step != before:
                    old = raw[at, h, row:row + stay]
                    raw[at, h, row:row + stay] = (as_value(old.contiguous()) * (before / step)).float().to(torch.float8_e4m3fn).view(torch.uint8)
            for p in here:
                raw[at, h, row + p - block * BLOCK] = (values[p][h] / step).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8)
            scale[at, h, row // BLOCK] = step


def forked(uses, table, lengths, source, room, page):
    """Lists of what fork_sequences_b200 leaves: uses, table, lengths, and the copies (from, to, tokens)."""
    E, P, pages = len(table), len(table[0]), len(uses)
    held = []
    for row in table:
        n = 0
        while n < P and 0 <= row[n] < pages:
            n += 1
        held.append(row[:n])
    source = [s if -1 <= s < E else e for e, s in enumerate(source)]
    keeper = {}
    for e, s in enumerate(source):
        if s >= 0 and (s not in keeper or s == e):
            keeper[s] = e if s == e or s not in keeper else keeper[s]
    rows, out = [], list(uses)
    for e, s in enumerate(source):
        length = min(max(lengths[s], 0), len(held[s]) * page) if s >= 0 else 0
        full, need = length // page, min(-(-(length + max(room[e], 0)) // page), P)
        kept = held[s][:full] if s >= 0 else []
        if s >= 0 and keeper[s] == e:
            for p in held[s][full:need]:
                if uses[p] != 1:
                    break
                kept = kept + [p]
        copied = held[s][full] if length % page and len(kept) == full else None
        rows.append([length, kept, need, copied])
    for e in range(E):
        for p in held[e]:
            out[p] -= 1
    for _, kept, _, _ in rows:
        for p in kept:
            out[p] += 1
    read = {r[3] for r in rows}
    free = [p for p in range(pages) if out[p] == 0 and p not in read]
    new_table, new_lengths, copies = [], [], []
    for length, kept, need, copied in rows:
        got = [free.pop(0) if free else None for _ in range(need - len(kept))]
        got = [p for p in got if p is not None]
        for p in got:
            out[p] += 1
        new_lengths.append(min(length, (len(kept) + len(got)) * page))
        new_table.append(kept + got + [-1] * (P - len(kept) - len(got)))
        if copied is not None and got:
            copies.append((copied, got[0], length % page))
    return out, new_table, new_lengths, copies
