"""Rotary positions, head norms and cache appends in 64 bits, element by element from their definitions (CPU)."""

from __future__ import annotations

import math

import torch


def angles(rotary_dim: int, base: float, scaling: dict | None = None) -> tuple[list[float], float]:
    """Each pair's angle per position, and the factor on cosines and sines, pair by pair."""
    s = scaling or {}
    kind, factor, trained = s.get("rope_type", "default"), s.get("factor", 1.0), s.get("original_max_position_embeddings")
    out = []
    for i in range(rotary_dim // 2):
        w = base ** (-2.0 * i / rotary_dim)
        if kind == "linear":
            w /= factor
        elif kind == "ntk":
            w = (base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * i / rotary_dim)
        elif kind == "llama3":
            low, high = s.get("low_freq_factor", 1.0), s.get("high_freq_factor", 4.0)
            length = 2 * math.pi / w
            if length > trained / low:
                w /= factor
            elif length >= trained / high:
                blend = (trained / length - low) / (high - low)
                w = (1 - blend) * w / factor + blend * w
        elif kind == "yarn":
            def edge(turns):  # where base ** (-2 x / r) makes `turns` turns over the trained length, in halves of x
                return rotary_dim / 2 * math.log(trained / (turns * 2 * math.pi), base)

            down, up = (math.floor, math.ceil) if s.get("truncate", True) else (float, float)
            lo = max(down(edge(s.get("beta_fast", 32))), 0)
            hi = min(up(edge(s.get("beta_slow", 1))), rotary_dim - 1)
            share = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
            w = w / factor * share + w * (1 - share)
        out.append(w)
    if kind != "yarn":
        return out, 1.0
    if "attention_factor" in s:
        return out, s["attention_factor"]
    ln = math.log(factor)
    if "mscale" in s and "mscale_all_dim" in s:
        return out, (0.1 * s["mscale"] * ln + 1) / (0.1 * s["mscale_all_dim"] * ln + 1)
    return out, 0.1 * ln + 1


def rotate(x, positions, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, interleaved: bool = False,
           weight=None, eps: float = 1e-6):
    """``(y, size)`` in float64 for ``x`` ``[T, H, D]``: the normed and rotated heads, and the sum of the magnitudes that
    went into each element (what a rounding inside is relative to)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    ws, amp = angles(rotary_dim, base, scaling)
    y, size = x.clone(), x.abs()
    for i, w in enumerate(ws):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
        th = positions.double().clamp(min=0)[:, None] * w
        c, s = amp * th.cos(), amp * th.sin()
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = amp * (x[..., a].abs() + x[..., b].abs())
    return y, size
