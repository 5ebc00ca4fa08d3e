"""Rotary positions of queries and keys.

Pair ``i`` of a head at position ``p`` is turned by the angle ``p * f_i``, ``f_i = base ** (-2 i / dim)``.  The rotation runs
in the library (``ma_b200_rotary_apply``), forward and backward; angles are exact at any position, because a frequency is
kept as a 64-bit fixed-point fraction of a turn and ``p * f_i`` taken modulo one turn in integers.  There is no table of
positions and so no longest position.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

Tensor = torch.Tensor

HALF, INTERLEAVED = 0, 1
_PAIRS = {"half": HALF, "interleaved": INTERLEAVED}
# pi to 50 digits: a turn is 2 pi radians, and 64 bits of a fraction of one are wanted
_PI = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)


class RotaryPositions:
    """The rotation of a model's heads: which features form pairs, and how fast each pair turns.

    ``dim``: rotated features of a head, even, at most 256; those behind stay as they are.  ``pairs``: ``"half"``, feature ``i`` with
    ``i + dim / 2``, or ``"interleaved"``, ``2 i`` with ``2 i + 1``.  ``scaling``, for contexts ``factor`` times as long as the
    ``trained_length``:

    * ``None``: none;
    * ``"linear"``: all frequencies divided by ``factor`` (positions are interpolated);
    * ``"ntk"``: ``base`` multiplied by ``factor ** (dim / (dim - 2))``: the slowest pair is divided by ``factor``, the fastest kept;
    * ``"yarn"``: by parts: pairs of more than 32 turns in ``trained_length`` kept, of less than one divided by ``factor``, those
      between mixed linearly in their number of turns; sines and cosines multiplied by ``0.1 ln(factor) + 1``; ``factor`` from 1 on.  (Some
      checkpoints were trained with a mixture that is linear in the pair's number between two borders; that is another rotation.)

    The object holds no device memory: it is made once and serves any device, stream and position.
    """

    def __init__(self, dim: int, base: float = 10000.0, pairs: str = "half", scaling: str | None = None, factor: float = 1.0,
                 trained_length: int | None = None):
        if dim <= 0 or dim % 2 or dim > 256:
            raise ValueError(f"dim must be even, positive and at most 256, got {dim}")
        if pairs not in _PAIRS:
            raise ValueError(f"pairs must be 'half' or 'interleaved', got {pairs!r}")
        if not (base > 0.0 and math.isfinite(base)):
            raise ValueError("base must be positive")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"unknown scaling {scaling!r}")
        if scaling is not None and not (factor > 0.0 and math.isfinite(factor)):
            raise ValueError("factor must be positive")
        if scaling == "yarn" and factor < 1.0:
            raise ValueError("the 'yarn' scaling needs a factor of at least 1")
        if scaling == "ntk" and dim == 2:
            raise ValueError("the 'ntk' scaling needs more than one pair")
        self.dim, self.base, self.pairs, self.scaling, self.factor = int(dim), float(base), pairs, scaling, float(factor)
        self.trained_length = trained_length
        self.magnitude = 1.0
        try:
            b = self.base * self.factor ** (dim / (dim - 2)) if scaling == "ntk" else self.base
            f = [b ** (-2.0 * i / dim) for i in range(dim // 2)]
            if scaling == "linear":
                f = [x / self.factor for x in f]
            elif scaling == "yarn":
                if not trained_length or trained_length <= 0:
                    raise ValueError("the 'yarn' scaling needs trained_length")
                kept = [min(1.0, max(0.0, (trained_length * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
                f = [x * (g + (1.0 - g) / self.factor) for x, g in zip(f, kept)]
                self.magnitude = 0.1 * math.log(self.factor) + 1.0
        except (OverflowError, ZeroDivisionError):
            b, f = math.inf, []
        if not all(math.isfinite(x) for x in (b, *f)):
            raise ValueError("the frequencies are no finite numbers")
        #: radians per position of each pair
        self.frequencies = tuple(f)
        turns = [round(Fraction(x) / (2 * _PI) * 2 ** 64) % 2 ** 64 for x in f]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64)
        self._native = (self.turns, self.dim, _PAIRS[pairs], self.magnitude)

    def __repr__(self) -> str:
        extra = "" if self.scaling is None else f", scaling={self.scaling!r}, factor={self.factor}, trained_length={self.trained_length}"
        return f"RotaryPositions({self.dim}, base={self.base}, pairs={self.pairs!r}{extra})"


_rotary = None


def _load():
    global _rotary
    from .monarch_attention import native_module
    _rotary = native_module().rotary
    return _rotary


def rotary_b200(query: Tensor, key: Tensor | None, rotary: RotaryPositions, positions: Tensor | None = None, *,
                inverse: bool = False) -> tuple[Tensor, Tensor | None]:
    """Rotated copies of ``query`` (E, H, N, D) and ``key`` (E, Hk, N, D; or None), in one launch.

    ``positions``: int32 or int64 of shape (N) or (E, N) on the same device, negative ones allowed; None: 0 .. N-1.  ``inverse`` turns
    back (the transpose: a magnitude other than one is multiplied once more).  float32, bfloat16 and float16, any strides (an inner
    stride other than one costs a copy); results keep the order of their input's strides.  Arithmetic is in 32 bits, rounded
    once.  Differentiable in both, any number of times, in reverse and
    in forward mode.
    """
    if not isinstance(rotary, RotaryPositions):
        raise TypeError("rotary must be a RotaryPositions")
    return (_rotary or _load())(query, key, *rotary._native, positions, inverse)
