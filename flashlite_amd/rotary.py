"""Frequencies of the rotary operators (``forward_rotary``, ``rotary_to_cache``,
``forward_norm_rotary``) and the axes of their pairs."""

from __future__ import annotations

import math

import torch


def rotary_frequencies(rot_dim: int, base: float = 10000.0, method: str | None = None,
                       factor: float = 1.0, trained: int = 0, fast: float = 32.0,
                       slow: float = 1.0, device=None):
    """(freqs, scale) of a rotary over the first ``rot_dim`` columns of a head:
    radians a position of each pair (float64 [rot_dim / 2]) and the factor on
    the rotated columns.

    Pair j turns by ``base ** (-2 j / rot_dim)`` a position.  ``method`` scales
    that for contexts ``factor`` times longer than the ``trained`` one:

    - None: not scaled;
    - "linear": every frequency divided by ``factor`` (positions interpolated);
    - "ntk": a larger base, with which the slowest pair is divided by
      ``factor`` and the fastest kept;
    - "yarn": pairs that turn more than ``fast`` times over ``trained``
      positions are kept, those that turn less than ``slow`` times divided by
      ``factor``, with a linear ramp over the pairs between; scale is
      0.1 ln(factor) + 1.
    """
    if rot_dim < 0 or rot_dim % 2 != 0:
        raise ValueError(f"rot_dim must be even and not negative (got {rot_dim})")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"base must be finite and above 1 (got {base})")
    if method not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown method {method!r} (None, 'linear', 'ntk' or 'yarn')")
    if method is not None and not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"factor must be finite and at least 1 (got {factor})")
    j = torch.arange(rot_dim // 2, dtype=torch.float64)
    scale = 1.0
    if method == "ntk" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freqs = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * j / max(rot_dim, 1))
    if method == "linear":
        freqs = freqs / factor
    elif method == "yarn":
        if trained < 1 or not fast > slow > 0:
            raise ValueError("yarn needs trained >= 1 and fast > slow > 0")

        def pair(turns):  # the (fractional) pair that turns so often over `trained` positions
            return rot_dim * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))

        # (the ramp may end past the last pair, which then is not divided in full)
        lo = max(math.floor(pair(fast)), 0)
        hi = min(math.ceil(pair(slow)), rot_dim - 1)
        ramp = ((j - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        freqs = freqs * (1.0 - ramp) + freqs / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    return freqs.to(device) if device is not None else freqs, scale


def rotary_axes(sections, interleaved: bool = False, device=None):
    """The axis of each pair (int32 [sum(sections)]) where ``sections[a]`` pairs
    turn by a token's position on axis a.

    The sections follow one another, or with ``interleaved`` the axes take
    turns, pair after pair, until their sections are used up (every axis then
    has fast and slow pairs); what is left of the longer ones follows.
    """
    sections = [int(s) for s in sections]
    if not sections or min(sections) < 0:
        raise ValueError(f"sections must be counts of pairs, not negative (got {sections})")
    if not interleaved:
        axes = [a for a, count in enumerate(sections) for _ in range(count)]
    else:
        axes = [a for turn in range(max(sections)) for a, count in enumerate(sections)
                if turn < count]
    return torch.tensor(axes, dtype=torch.int32, device=device)
