"""Rotation tables for :func:`native.qk_norm_rope` and :func:`native.paged_append`.

The reference takes post-RoPE Q/K from its model (teacher/chunked_extract.py:164-172); a serving program that feeds
the selector and the attention itself needs the angles.  They are formed in 64 bits and rounded once: at position
131072 an fp32 angle product is off by up to 7e-3 rad.  Frequency scaling for contexts longer than the trained one
only changes the table, so it costs the kernels nothing.
"""
from __future__ import annotations

import math

import torch

SCALINGS = ("linear", "ntk", "yarn", "banded")


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """float64 angles per position ``[rotary_dim / 2]`` and the factor cos and sin are multiplied by.

    ``scaling`` has a ``type``, a ``factor`` >= 1 and, by type:

    * ``linear``: every frequency divided by the factor (position interpolation);
    * ``ntk``: the base raised to ``base * factor ** (d / (d - 2))``, which leaves the fastest pair and divides the slowest by
      the factor;
    * ``yarn`` (Peng et al. 2023): pairs that turn more than ``beta_fast`` (32) times over ``original_positions``
      are kept, those under ``beta_slow`` (1) divided by the factor, a linear ramp between; cos and sin times
      ``attention_factor`` (0.1 ln(factor) + 1);
    * ``banded``: wavelengths under ``original_positions / high_freq_factor`` are kept, over ``original_positions /
      low_freq_factor`` divided by the factor, and mixed between in the wave number.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if base <= 1:
        raise ValueError(f"base must be above 1, got {base}")

    def plain(b):
        return b ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)

    freq = plain(float(base))
    if scaling is None:
        return freq, 1.0
    kind = scaling.get("type")
    if kind not in SCALINGS:
        raise ValueError(f"scaling type must be one of {SCALINGS}, got {kind!r}")
    factor = float(scaling["factor"])
    if factor < 1:
        raise ValueError(f"scaling factor must be at least 1, got {factor}")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of at least 4")
        return plain(float(base) * factor ** (rotary_dim / (rotary_dim - 2))), 1.0
    original = float(scaling["original_positions"])
    if kind == "yarn":
        def pair_of(turns):  # the (fractional) pair that turns so often over the original positions
            return rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(math.floor(pair_of(float(scaling.get("beta_fast", 32)))), 0)
        high = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        mult = scaling.get("attention_factor")
        return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1 if mult is None else float(mult)
    low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
    if high <= low:
        raise ValueError("high_freq_factor must be above low_freq_factor")
    turns = original * freq / (2 * math.pi)  # over the original positions
    mix = ((turns - low) / (high - low)).clamp(0, 1)
    return freq * mix + freq / factor * (1 - mix), 1.0


def rope_table(rotary_dim: int, positions: int, base: float = 10000.0, scaling: dict | None = None,
               device="cuda") -> torch.Tensor:
    """fp32 ``[positions, rotary_dim]``: cos of each position's angles, then their sin."""
    if positions < 1:
        raise ValueError(f"positions must be positive, got {positions}")
    freq, mult = rope_frequencies(rotary_dim, base, scaling)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return torch.cat([angles.cos() * mult, angles.sin() * mult], dim=1).float()
