"""Rotary positions: features of queries and keys turned by angles that grow with the position.

No counterpart in the reference."""
import math

import torch

ops = torch.ops.torch_butterfly


def rotary(x, positions, frequencies, interleaved=False, magnitude=1.0):
    """``x`` (*, heads, features) with pair ``p`` of every head's first ``2 * len(frequencies)`` features turned by the angle
    ``positions * frequencies[p]`` and scaled by ``magnitude``: ``(a, b) -> magnitude * (a cos - b sin, a sin + b cos)``.
    A pair is features ``p`` and ``p + len(frequencies)``, or ``2 p`` and ``2 p + 1`` (``interleaved``).  Further
    features stay as they are.

    ``x`` float32 or bfloat16 with any strides, ``positions`` (*) int64, ``frequencies`` float64 (``rotary_frequencies``
    makes them).  Angles are formed in 64 bits, whatever the position.  Gradients of any order exist (no forward mode)."""
    if x.is_cuda:
        return ops.rotary(x, positions, frequencies, interleaved, magnitude)
    pairs = frequencies.shape[0]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    angles = (positions.to(torch.float64).unsqueeze(-1) * frequencies).unsqueeze(-2)
    cosine, sine = ((magnitude * f(angles)).to(wide) for f in (torch.cos, torch.sin))
    part = x[..., :2 * pairs].to(wide)
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :pairs], part[..., pairs:])
    turned = (a * cosine - b * sine, a * sine + b * cosine)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * pairs:]), -1)


def rotary_frequencies(rotated, base=10000.0, scaling=None, factor=1.0, context=None, fast=32.0, slow=1.0, device=None):
    """``(frequencies, magnitude)`` for ``rotary``: ``base ** (-2 p / rotated)`` for the pairs of ``rotated`` features, as
    they are or for contexts ``factor`` times as long:

    * ``"linear"``: all divided by ``factor`` (positions interpolated);
    * ``"base"``: a larger base, with which the slowest frequency is divided by ``factor`` and the fastest stays;
    * ``"parts"``: pairs that turn at least ``fast`` times within ``context`` tokens (the original length) stay, those that
      turn at most ``slow`` times are divided by ``factor``, a linear ramp in the number of turns between;
      magnitude ``0.1 log(factor) + 1``."""
    if rotated <= 0 or rotated % 2:
        raise ValueError(f"rotated must be positive and even, got {rotated}")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
    if not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "base" and rotated > 2:
        base *= factor ** (rotated / (rotated - 2))
    frequencies = base ** (-torch.arange(rotated // 2, dtype=torch.float64) * 2 / rotated)
    magnitude = 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "parts":
        if context is None:
            raise ValueError("scaling 'parts' needs the original context")
        if not fast > slow:
            raise ValueError("fast must be above slow")
        turns = frequencies * context / (2 * math.pi)
        stay = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        frequencies = frequencies * stay + frequencies / factor * (1.0 - stay)
        magnitude = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device), magnitude
