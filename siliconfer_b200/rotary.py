"""Rotary positions on the GPU: half and interleaved layouts, the whole head or its first part, scaled tables.

The angles come from a table of cosines and sines, built once on the host in
64 bits, so that a position of a million turns as exactly as the first one.
siliconfer applies its positions through MLX (siliconfer/model/layers.py).
The kernel is in libsf_q4.so (``sf_rotary``); there is no CPU fallback, and no
gradient: outputs are detached from inputs that require one.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from . import _lib


def rotary_frequencies(rot: int, base: float = 10000.0, scaling=None, factor: float = 1.0, original_max: int = 4096,
                       beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(radians a position for each of the rot / 2 pairs, factor of the table's values), in 64 bits.

    scaling None: base^(-2j / rot).  ``"linear"``: positions divided by
    ``factor``.  ``"ntk"``: base raised so that the slowest pair turns
    ``factor`` times slower and the fastest as before.  ``"yarn"``: pairs that
    make more than ``beta_fast`` turns within ``original_max`` positions keep
    their speed, those with fewer than ``beta_slow`` are slowed by ``factor``,
    a ramp in between, and the values are scaled by 0.1 ln(factor) + 1."""
    if rot < 2 or rot % 2:
        raise RuntimeError("rot must be a positive even number")
    if factor < 1.0:
        raise RuntimeError("factor must be at least 1")
    j = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2)) if rot > 2 else base
    freq = base ** (-2.0 * j / rot)
    if scaling in (None, "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling != "yarn":
        raise RuntimeError(f"unknown rotary scaling {scaling!r} (linear, ntk, yarn)")

    def pair_of(turns):
        return rot * math.log(original_max / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo = max(math.floor(pair_of(beta_fast)), 0)
    hi = min(math.ceil(pair_of(beta_slow)), rot - 1)
    slow = np.clip((j - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
    return freq * (1 - slow) + freq / factor * slow, 0.1 * math.log(factor) + 1.0


def rotary_table(max_pos: int, rot: int, base: float = 10000.0, scaling=None, factor: float = 1.0,
                 original_max: int = 4096, device=None, **ramp) -> torch.Tensor:
    """fp32 [max_pos, rot]: row p holds the rot / 2 cosines, then the sines, of position p (see ``rotary_frequencies``)."""
    if max_pos < 1:
        raise RuntimeError("max_pos must be positive")
    freq, gain = rotary_frequencies(rot, base, scaling, factor, original_max, **ramp)
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * freq
    table = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32) * np.float32(gain))
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else "cpu"
    return table.to(device)


def apply_rotary(x, positions, table, interleaved: bool = False, out=None):
    """x [T, heads, head_dim] turned by its tokens' positions [T] (int32 or int64).

    The first table.shape[1] elements of a head are turned, in pairs (j, rot / 2 + j),
    or (2j, 2j + 1) when ``interleaved``; the others are copied.  ``out`` may be x."""
    return _lib.ext().rotary(x, positions, table, interleaved, out)


__all__ = ["rotary_frequencies", "rotary_table", "apply_rotary"]
