"""Definitions in 64 bits of the rotary positions, the paged 8-bit cache and the attention over it, and error bounds by arithmetic.

Half a step of rounding: bf16 2^-8, f16 2^-11, f32 2^-24, e4m3 2^-4 of the value (2^-10 of the scale for subnormal codes).
"""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Below a type's smallest normal number 2^m the steps stay at eps * 2^m, so a value there is off by up to eps / 2 * 2^m whatever its size: for f16
# 2^-11 * 2^-14 = 2^-25, which half a step of 2^-11 of the value does not cover (a result of 2^-16 may be off by 2^-25 = 2^-9 of it).
SUBNORMAL = {t: h * torch.finfo(t).smallest_normal for t, h in HALF_STEP.items()}


def pair_index(dim, pairs):
    i = torch.arange(dim // 2)
    return (i, i + dim // 2) if pairs == "half" else (2 * i, 2 * i + 1)


def rotate(x, positions, rotary, inverse=False):
    """x (..., N, D) rotated at positions (broadcastable to (..., N)), in 64 bits; and the sum of magnitudes that enter each element."""
    x = x.double().cpu()
    a, b = pair_index(rotary.dim, rotary.pairs)
    f = torch.tensor(rotary.frequencies, dtype=torch.float64)
    angle = positions.double().cpu()[..., None] * f
    if inverse:
        angle = -angle
    cos, sin = rotary.magnitude * angle.cos(), rotary.magnitude * angle.sin()
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    both = rotary.magnitude * (x[..., a].abs() + x[..., b].abs())
    size[..., a], size[..., b] = both, both
    return y, size


def rotation_bound(want, size, dtype):
    """One rounding to the type; before it sines within 2^-22 (2 units in the last place, and the angle to 2^-25 turns) and three 32-bit roundings."""
    return HALF_STEP[dtype] * want.abs() + 8 * 2.0 ** -24 * size + SUBNORMAL[dtype]


def held(codes, scales, table, length, page):
    """(heads, length, D) in 64 bits: what a sequence's cached tokens stand for."""
    used = table[:(length + page - 1) // page].long().cpu()
    x = codes.cpu().view(torch.uint8)[used].view(torch.float8_e4m3fn).double()
    s = scales.cpu()[used].double().repeat_interleave(16, -1)[..., None]
    return (x * s).transpose(0, 1).flatten(1, 2)[:, :length]


def attention(q, k, v, first, causal, scale, softcap=0.0, window=0):
    """q (H, n, D) at positions first.. over k, v (Hk, L, D), in 64 bits: result and the bound of the kernel's error.

    Scores: products in 32-bit sums, so (D + 8) 2^-24 of the sum of magnitudes (D 2^-25 of it more where bf16 rows are brought to f16), and
    2^-22 of a cap.  A weight is off by as much, by 2^-11 (f16) and 2^-20 (exponentials, scales, order of sums); weights under the f16 range
    by 2^-25 of the largest, times a code of at most twice the largest value's: length * 2^-24 of that.
    """
    q, k, v = q.double().cpu(), k.double(), v.double()
    H, n, D = q.shape
    L = k.shape[1]
    k, v = (t.repeat_interleave(H // t.shape[0], 0) for t in (k, v))
    s = q @ k.mT * scale
    size = (q.abs() @ k.abs().mT) * abs(scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    at, place = torch.arange(L), first + torch.arange(n)[:, None]
    seen = torch.ones(n, L, dtype=torch.bool)
    if causal:
        seen = at <= place
        if window:
            seen = seen & (at > place - window)
    s = s.masked_fill(~seen, -math.inf)
    w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    out = w @ v
    off = (size * (1.5 * D + 8) * 2.0 ** -24 + abs(softcap) * 2.0 ** -22).masked_fill(~seen, 0.0).amax(-1, keepdim=True) if L else torch.zeros(H, n, 1)
    most = v.abs().amax() if v.numel() else 0.0
    bound = (2.0 ** -11 + 2.0 ** -20 + 2 * off) * (w @ v.abs()) + L * 2.0 ** -24 * most
    return out, bound


def close(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() - bound)
    assert bool((over <= 0).all()), f"{what}: off by {float((got - want).abs().max()):.3e}, {float((over > 0).double().mean()):.2e} of the elements over the bound"
