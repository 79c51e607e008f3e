"""Rotary positions, and the append of keys and values to a paged cache.

One launch rotates a step's (or a prompt's) queries and keys and writes the
keys and values to their slots of the paged cache (num_blocks, kv_heads,
block_size, head_dim) through the block table.  Tables of cosines and sines
come from :func:`rotary_tables`, once per model.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib


def rotary_tables(rotary_dim: int, max_positions: int, theta: float = 10000.0, *, scaling: Optional[Dict] = None,
                  device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), each (max_positions, rotary_dim / 2) float32, of angle position * theta^(-2 i / rotary_dim).

    Angles are computed in 64 bits, so positions of any size keep their fraction of a turn.  ``scaling``
    stretches a model trained on short contexts over long ones:

    * ``{"type": "linear", "factor": f}``: positions divided by f;
    * ``{"type": "ntk", "factor": f}``: theta grows so that the slowest pair is divided by f and the fastest kept;
    * ``{"type": "yarn", "factor": f, "original": n, "beta_fast": 32, "beta_slow": 1, "magnitude": m}``: pairs that
      turn more than beta_fast times within the original context n are kept, those below beta_slow turns are
      divided by f, linearly between in the pair's index; cosines and sines are multiplied by m
      (default 0.1 ln f + 1);
    * ``{"type": "bands", "factor": f, "original": n, "low": 1, "high": 4}``: pairs with a wavelength below
      n / high are kept, above n / low divided by f, and blended linearly in n / wavelength between.
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim ({rotary_dim}) must be even and not negative")
    if max_positions < 1:
        raise ValueError(f"max_positions ({max_positions}) must be positive")
    if not theta > 0:
        raise ValueError(f"theta ({theta}) must be positive")
    index = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    magnitude = 1.0
    s = dict(scaling or {})
    kind, factor = s.pop("type", None), float(s.pop("factor", 1.0))
    if not factor > 0:
        raise ValueError(f"scaling factor ({factor}) must be positive")
    if kind == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inverse = theta ** (-index / max(rotary_dim, 1))
    if kind == "linear":
        inverse = inverse / factor
    elif kind == "yarn":
        n, fast, slow = float(s.pop("original")), float(s.pop("beta_fast", 32)), float(s.pop("beta_slow", 1))
        magnitude = float(s.pop("magnitude", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))

        def pair_of(turns):
            return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low = max(math.floor(pair_of(fast)), 0)
        high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
        ramp = ((index / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        inverse = inverse / factor * ramp + inverse * (1 - ramp)
    elif kind == "bands":
        n, low, high = float(s.pop("original")), float(s.pop("low", 1)), float(s.pop("high", 4))
        kept = ((n * inverse / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        inverse = inverse * kept + inverse / factor * (1 - kept)
    elif kind not in (None, "ntk"):
        raise ValueError(f"unknown scaling type {kind!r}; expected linear, ntk, yarn or bands")
    if s:
        raise ValueError(f"unknown scaling keys for {kind!r}: {sorted(s)}")
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * inverse
    return (angle.cos() * magnitude).float().to(device), (angle.sin() * magnitude).float().to(device)


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                     interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """Rotary embedding of x (tokens, heads, head_dim) at ``positions`` (tokens,).

    The first 2 * cos.shape[1] columns turn, in pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    ``interleaved``; the rest are copied.  ``inverse`` turns back: the transposed map, which is also the
    gradient with respect to x of the forward one.
    """
    return _lib.require_binding().rotary(x, None, None, positions, cos, sin, None, None, None, None, interleaved,
                                         inverse, 1.0, 1.0, False)


def rotary_append_paged(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                        cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], k_cache: torch.Tensor,
                        v_cache: torch.Tensor, block_tables: torch.Tensor, *, seq_ids: Optional[torch.Tensor] = None,
                        interleaved: bool = False, k_scale: float = 1.0, v_scale: float = 1.0,
                        return_keys: bool = False):
    """Rotate q and k and append k and v to the paged cache, in one launch.

    q (tokens, q_heads, head_dim), k and v (tokens, kv_heads, head_dim), strided views allowed; token t
    sits at ``positions[t]`` of sequence ``seq_ids[t]`` (default: token t belongs to sequence t; a
    negative id appends nothing).  ``cos`` / ``sin`` as in :func:`rotary_embedding`; None appends without
    rotating (positions given by a bias instead).  float8_e4m3fn caches hold round(k (1 / k_scale)), saturated.
    Returns the rotated q, or (q, k) with ``return_keys``; q None gives None.

    A position outside the tables or the block table, or a page outside the cache, appends nothing and
    sets the device's status word (:func:`check_status`).
    """
    return _lib.require_binding().rotary(q, k, v, positions, cos, sin, k_cache, v_cache, block_tables, seq_ids,
                                         interleaved, False, k_scale, v_scale, return_keys)
