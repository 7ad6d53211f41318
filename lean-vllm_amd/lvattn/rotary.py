"""Rotary positions of queries and keys, after an RMS norm of each head where a model has one, on the GPU.

What a layer does between its q/k/v projection and ``store_kvcache`` / ``forward``, in one launch (``lv_rotary``):
``norm_rotary`` norms and rotates, ``apply_rotary`` only rotates; ``MI355XAttention.append_kvcache`` does either on the
way into the paged cache. ``Packer.pack`` returns the ``positions`` they read. ``rotary_table`` lays out the cosines and
sines once, for the plain frequencies or ones scaled to contexts longer than the trained ones.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from . import _capi, checks


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[np.ndarray, float]:
    """Angle per position of each of the ``rotary_dim / 2`` pairs (float64), and the factor on cosines and sines.

    ``scaling`` (None: ``base ** (-2 i / rotary_dim)``) names a ``rope_type``, as checkpoints' configurations do:

    - ``linear``: positions divided by ``factor``;
    - ``ntk``: the base raised by ``factor ** (r / (r - 2))``, so that the slowest pair is slowed by ``factor``;
    - ``llama3``: pairs of fewer than ``low_freq_factor`` (1) turns over ``original_max_position_embeddings`` slowed by
      ``factor``, of more than ``high_freq_factor`` (4) kept, a linear blend between;
    - ``yarn`` (Peng et al., "YaRN", 2023): the blend linear over the pairs' indices, from ``beta_fast`` (32) turns to
      ``beta_slow`` (1), at whole indices unless ``truncate`` is False, and cosines and sines times ``attention_factor``:
      by default ``a(1)`` with ``a(m) = 0.1 m ln(factor) + 1``, or ``a(mscale) / a(mscale_all_dim)`` where both are given.

    Other keys are refused: one that is ignored would give other angles than the checkpoint's.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: the rotary width {rotary_dim} is not a positive even number")
    if not base > 1:
        raise ValueError(f"rotary_frequencies: base {base} is not above 1")
    r, s = rotary_dim, dict(scaling or {})
    kind = s.pop("rope_type", None) or s.pop("type", None) or "default"
    keys = {"default": (), "linear": ("factor",), "ntk": ("factor",),
            "llama3": ("factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"),
            "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate",
                     "attention_factor", "mscale", "mscale_all_dim")}
    if kind not in keys:
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} is not one of {', '.join(keys)}")
    other = sorted(set(s) - set(keys[kind]))
    if other:
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} takes no {', '.join(other)}")
    exponents = np.arange(0, r, 2, dtype=np.float64) / r
    inv = float(base) ** -exponents
    if kind == "default":
        return inv, 1.0
    factor = float(s.get("factor", 0.0))
    if not factor >= 1.0:
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} needs a factor of at least 1, got {s.get('factor')}")
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "ntk":
        if r == 2:
            raise ValueError("rotary_frequencies: ntk scaling needs a rotary width above 2")
        return (float(base) * factor ** (r / (r - 2))) ** -exponents, 1.0
    trained = s.get("original_max_position_embeddings")
    if not trained or trained <= 0:
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} needs original_max_position_embeddings")
    if kind == "llama3":
        low, high = float(s.get("low_freq_factor", 1.0)), float(s.get("high_freq_factor", 4.0))
        if not 0 < low < high:
            raise ValueError(f"rotary_frequencies: low_freq_factor {low} and high_freq_factor {high}")
        kept = np.clip((trained * inv / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        return inv * (kept + (1.0 - kept) / factor), 1.0

    def pair_of(turns: float) -> float:  # twice the index of the pair that makes so many turns over the trained length
        return r * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))

    fast, slow = float(s.get("beta_fast") or 32.0), float(s.get("beta_slow") or 1.0)
    if not 0 < slow < fast:
        raise ValueError(f"rotary_frequencies: beta_fast {fast} and beta_slow {slow}")
    lo, hi = pair_of(fast), pair_of(slow)
    if s.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, r - 1)
    slowed = np.clip((np.arange(r // 2) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)

    def a(m: float) -> float:
        return 0.1 * m * math.log(factor) + 1.0

    amp = s.get("attention_factor")
    if amp is None:
        both = s.get("mscale") and s.get("mscale_all_dim")
        amp = a(float(s["mscale"])) / a(float(s["mscale_all_dim"])) if both else a(1.0)
    return inv * (1.0 - slowed + slowed / factor), float(amp)


def rotary_table(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: dict | None = None,
                 device="cuda") -> torch.Tensor:
    """fp32 ``[max_position, rotary_dim]``: each position's ``rotary_dim / 2`` cosines, then its sines. Angles are taken
    in 64 bits (an fp32 angle at position 10^5 is off by up to 4e-3) and only the table is rounded."""
    if max_position < 1:
        raise ValueError(f"rotary_table: {max_position} positions")
    inv, amp = rotary_frequencies(rotary_dim, base, scaling)
    inv = torch.from_numpy(inv).to(device)
    table = torch.empty(max_position, rotary_dim, dtype=torch.float32, device=device)
    half, step = rotary_dim // 2, 1 << 16
    for at in range(0, max_position, step):  # the 64-bit angles of 65536 positions at a time
        angles = torch.arange(at, min(at + step, max_position), dtype=torch.float64, device=device)[:, None] * inv
        table[at:at + step, :half] = angles.cos().mul_(amp)
        table[at:at + step, half:] = angles.sin_().mul_(amp)
    return table


def head_args(what: str, name: str, t, tokens: int, dim: int, dtype, device: int) -> tuple:
    """Pointer, token stride, head stride and heads of ``t`` ``[T, H, D]`` for the C call (None: no heads). Raises
    ``ValueError`` unless it has ``tokens``, ``dim``, ``dtype``, a unit dim stride and lies on GPU ``device``."""
    if t is None:
        return None, 0, 0, 0
    shape, stride = t.shape, t.stride()
    if (len(shape) != 3 or shape[0] != tokens or shape[2] != dim or stride[2] != 1 or t.dtype is not dtype
            or t.get_device() != device):
        raise ValueError(f"{what}: {name} is {t.dtype} {tuple(shape)} of strides {stride} on {t.device}, not {dtype} "
                         f"[{tokens}, H, {dim}] of unit dim stride beside the other heads")
    return t.data_ptr(), stride[0], stride[1], shape[1]


def rotary_args(what: str, positions, table, q_weight, k_weight, tokens: int, dim: int, dtype, device: int) -> tuple:
    """The C call's positions, table and weights. Raises ``ValueError`` unless ``positions`` is contiguous int64 ``[T]``,
    ``table`` contiguous fp32 ``[P, r]`` with r even and at most D, the weights contiguous ``[D]`` of the heads' dtype, and
    all on GPU ``device``."""
    if positions.dtype is not torch.int64 or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"{what}: positions must be contiguous int64 [{tokens}], got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    shape = table.shape
    if (len(shape) != 2 or table.dtype is not torch.float32 or shape[0] < 1 or shape[1] < 2 or shape[1] % 2
            or shape[1] > dim or not table.is_contiguous()):
        raise ValueError(f"{what}: the table must be contiguous fp32 [positions, r] with r even and at most the head "
                         f"width {dim}, got {table.dtype} {tuple(shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (dim,) or w.dtype is not dtype or not w.is_contiguous()
                              or w.get_device() != device):
            raise ValueError(f"{what}: {name} must be contiguous {dtype} [{dim}] beside the heads, got {w.dtype} "
                             f"{tuple(w.shape)} on {w.device}")
    if device < 0 or positions.get_device() != device or table.get_device() != device:
        raise ValueError(f"{what}: positions on {positions.device}, table on {table.device}, heads on GPU {device}; all "
                         "must be on one GPU")
    if checks.ENABLED:
        checks.check_positions(positions, shape[0])
    return positions.data_ptr(), table.data_ptr(), shape[0], shape[1], _capi.ptr(q_weight), _capi.ptr(k_weight)


def first_heads(what: str, t) -> tuple:
    """Tokens, width, dtype and GPU of the heads that the others have to match."""
    if t.dim() != 3 or t.dtype not in _capi.DTYPES:
        raise ValueError(f"{what}: heads are bf16 or fp16 [T, H, D], got {t.dtype} {tuple(t.shape)}")
    tokens, _, dim = t.shape
    return tokens, dim, t.dtype, t.get_device()


def output_heads(what: str, name: str, x, out, like: tuple):
    """``out``, checked against its input ``x`` ``[T, H, D]``, or a new tensor; and its arguments for the C call."""
    if out is None:
        if x is None:
            return None, (None, 0, 0)
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        return out, (out.data_ptr(), x.size(1) * like[1], like[1])
    if x is None or out.shape != x.shape:
        raise ValueError(f"{what}: {name} is {tuple(out.shape)}, its input "
                         f"{'missing' if x is None else tuple(x.shape)}")
    if (out.stride(0) == 0 and out.size(0) > 1) or (out.stride(1) == 0 and out.size(1) > 1):
        raise ValueError(f"{what}: {name} of strides {out.stride()} holds one row for several heads or tokens")
    return out, head_args(what, name, out, *like)[:3]


def apply_rotary(q, k, positions, table, interleaved: bool = False, out_q=None, out_k=None):
    """Rotary positions on ``q`` ``[T, Hq, D]`` and ``k`` ``[T, Hkv, D]`` (either may be None), any token and head strides:
    views of a fused projection, or of a part of each head, will do. ``positions`` int64 ``[T]``; ``table`` as
    ``rotary_table`` makes it, of r <= D: the first r dims of each head turn in pairs ``(i, i + r / 2)``, or
    ``(2 i, 2 i + 1)`` if ``interleaved``, the others are copied. Returns ``(q', k')``: new tensors, or ``out_q`` /
    ``out_k``, each of which may be its input itself (in place) and must not overlap it otherwise. In fp32, rounded once.
    A negative position rotates as position 0 (padding); one past the table gives NaN."""
    return _rotate("apply_rotary", q, k, None, None, positions, table, 0.0, interleaved, out_q, out_k)


def norm_rotary(q, k, q_weight, k_weight, positions, table, eps: float = 1e-6, interleaved: bool = False, out_q=None,
                out_k=None):
    """``apply_rotary`` on ``x * rsqrt(mean(x^2) + eps) * weight`` of every head, ``q_weight`` / ``k_weight`` ``[D]`` of the
    heads' dtype (None: those heads are not normed), in the same pass and rounded only once."""
    return _rotate("norm_rotary", q, k, q_weight, k_weight, positions, table, eps, interleaved, out_q, out_k)


def _rotate(what, q, k, q_weight, k_weight, positions, table, eps, interleaved, out_q, out_k):
    if q is None and k is None:
        raise ValueError(f"{what}: no heads to rotate")
    like = first_heads(what, q if q is not None else k)
    tokens, dim, dtype, device = like
    *q_args, heads = head_args(what, "q", q, *like)
    *k_args, kv_heads = head_args(what, "k", k, *like)
    pos, tab, positions_held, width, qw, kw = rotary_args(what, positions, table, q_weight, k_weight, *like)
    out_q, oq_args = output_heads(what, "out_q", q, out_q, like)
    out_k, ok_args = output_heads(what, "out_k", k, out_k, like)
    _capi.call_on(device, "lv_rotary", *q_args, *k_args, pos, tab, positions_held, width, int(interleaved), qw, kw, eps,
                  tokens, heads, kv_heads, dim, *oq_args, *ok_args, _capi.DTYPES[dtype])
    return out_q, out_k
