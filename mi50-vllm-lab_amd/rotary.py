"""Rotary tables for rotary_cache_write: cosines and sines of position x frequency, formed in 64 bits and laid out once.

Frequency of pair i of rotary_dim / 2: base^(-2 i / rotary_dim). For contexts beyond the trained one the frequencies are
scaled (`scaling`):
  linear  all frequencies divided by `factor` (positions interpolated).
  ntk     the base raised to base * factor^(rotary_dim / (rotary_dim - 2)): the lowest frequency is divided by factor, the
          highest stays.
  yarn    Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models" (2023): pairs that turn more than
          beta_fast times over the original context keep their frequency, those that turn less than
          beta_slow times are divided by factor, linearly blended in between over the pair number (whose ends, rounded outwards,
          are kept within 0 and rotary_dim - 1); the cosines and sines are multiplied by 0.1 ln(factor) + 1 (or by attention_factor).
"""
from __future__ import annotations

import math

import torch


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """The frequencies of the rotary_dim / 2 pairs (float64) and the factor of the cosines and sines."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    pairs = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    freq = float(base) ** -pairs
    if scaling is None:
        return freq, 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            return freq, 1.0
        return (float(base) * factor ** (rotary_dim / (rotary_dim - 2))) ** -pairs, 1.0
    if kind == "yarn":
        original = float(scaling["original_max_position"])
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

        def pair_of(turns: float) -> float:  # the pair number that turns so often over the original context
            return rotary_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        # (hi may lie beyond the last pair: if that still turns more than beta_slow times, the ramp ends behind it)
        lo, hi = max(0, math.floor(pair_of(fast))), min(rotary_dim - 1, math.ceil(pair_of(slow)))
        number = torch.arange(rotary_dim // 2, dtype=torch.float64)
        slowed = ((number - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        mult = scaling.get("attention_factor")
        mult = float(mult) if mult is not None else (0.1 * math.log(factor) + 1.0)
        return freq * (1.0 - slowed) + freq / factor * slowed, mult
    raise ValueError(f"unknown rotary scaling {kind!r}: linear, ntk or yarn")


def rotary_table(rotary_dim: int, max_positions: int, base: float = 10000.0, scaling: dict | None = None,
                 device="cpu") -> torch.Tensor:
    """cos_sin [max_positions, rotary_dim] (fp32) of rotary_cache_write: the cosines of the rotary_dim / 2 angles, then the
    sines. scaling: None or {"type": "linear" | "ntk" | "yarn", "factor": .., ...} (see the module)."""
    if max_positions < 0:
        raise ValueError("max_positions must not be negative")
    freq, mult = rotary_frequencies(rotary_dim, base, scaling)
    # a position x frequency that is correct to 64 bits over any context, a slab of positions at a time
    out = torch.empty((max_positions, rotary_dim), dtype=torch.float32, device=device)
    freq = freq.to(device)
    for p in range(0, max_positions, 1 << 16):
        angle = torch.arange(p, min(max_positions, p + (1 << 16)), dtype=torch.float64, device=device)[:, None] * freq
        out[p:p + (1 << 16), :rotary_dim // 2] = angle.cos() * mult
        out[p:p + (1 << 16), rotary_dim // 2:] = angle.sin() * mult
    return out
