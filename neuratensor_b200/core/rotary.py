"""Frequencies of rotary positions, plain and scaled for contexts longer than trained.

``RotaryEmbedding`` (model.py:88-116) has the plain ones; ``rotary_frequencies``
adds the scaled forms for ``native.rotary``, which takes any frequencies and a
factor on the rotated pairs.
"""
from __future__ import annotations

import math
from typing import Tuple

import torch
from torch import Tensor


class Seen:
    """A buffer as it was: held, so that no other tensor can take its place unnoticed, with its version."""

    def __init__(self, t: Tensor) -> None:
        self.tensor, self.version = t, self._version(t)

    @staticmethod
    def _version(t: Tensor) -> int:
        return 0 if t.is_inference() else t._version

    def still(self, t: Tensor) -> bool:
        """Whether `t` is the buffer, unwritten since."""
        return t is self.tensor and self._version(t) == self.version


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained_len: int = 2048, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> Tuple[Tensor, float]:
    """(float32 frequencies [dim / 2], factor on the rotated pairs) for ``native.rotary``.

    F_i = base^(-2i / dim), and with ``factor`` s > 1:

    * "linear": F_i / s, every position s times nearer;
    * "base": base * s^(dim / (dim - 2)) for base, which keeps the fastest frequency and
      divides the slowest by s;
    * "by_parts": F_i where it turns at least ``fast`` times within ``trained_len`` tokens,
      F_i / s where it turns at most ``slow`` times, and in between a mean weighted by
      the turns; pairs are multiplied by 1 + 0.1 ln s, which sharpens the scores of long
      contexts."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2, got {dim}")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling not in ("none", "linear", "base", "by_parts"):
        raise ValueError(f"scaling must be none, linear, base or by_parts, got {scaling!r}")
    mscale = 1.0
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        if not 0 < slow < fast:
            raise ValueError(f"0 < slow < fast, got {slow} and {fast}")
        turns = trained_len * f / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        mscale = 1.0 + 0.1 * math.log(factor)
    return f.float().to(device), mscale
