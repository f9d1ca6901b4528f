"""Rotary positions of queries and keys (no counterpart in the reference,
whose models rotate before they hand their keys to the cache)."""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native

def rotary_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None,
                       factor: float = 1.0, original_len: int = 0, slow_turns: float = 1.0,
                       fast_turns: float = 32.0, device="cuda"):
    """Frequencies of rotary positions: (inv_freq, amplitude) for ``apply_rotary``
    and the paged cache; computed once and kept.

    inv_freq is (rot_dim / 2,) float64, radians per position of each pair:
    base^(-2 p / rot_dim), changed for contexts longer than the trained one by
      'linear'  every pair slowed by ``factor``
      'ntk'     the base raised so that the slowest pair slows by ``factor``
      'yarn'    pairs that make fewer than ``slow_turns`` turns in
                ``original_len`` positions slow by ``factor``, those with more
                than ``fast_turns`` stay, and between them the share that stays
                grows linearly with the number of turns; the amplitude is
                0.1 ln(factor) + 1 (as printed in Peng et al., 2023)

    Many checkpoints with YaRN were trained with another ramp under that name,
    linear in the pair's index, that is in the logarithm of the turns: in the
    pairs between, its frequencies differ from these by up to 56 % (128 elements,
    base 10000, 4096 positions, factor 8).  For such a model compute its own
    vector; every call takes any (rot / 2,) float64 tensor as ``inv_freq``.
    """
    if rot_dim < 8 or rot_dim % 8:
        raise ValueError(f"rotary_frequencies: rot_dim {rot_dim} is not a multiple of 8")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("rotary_frequencies: scaling must be None, 'linear', 'ntk' or 'yarn', "
                         f"got {scaling!r}")
    if not base > 0 or not factor > 0:
        raise ValueError("rotary_frequencies: base and factor must be positive")
    amplitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = float(base) ** -(torch.arange(0, rot_dim, 2, dtype=torch.float64, device="cpu") / rot_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if original_len <= 0 or not fast_turns > slow_turns:
            raise ValueError("rotary_frequencies: 'yarn' needs original_len > 0 and "
                             "fast_turns > slow_turns")
        turns = f * original_len / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return f.to(device), amplitude


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 inv_freq: torch.Tensor, *, interleaved: bool = False, amplitude: float = 1.0,
                 inverse: bool = False, out=None):
    """Turn q and k by their tokens' positions, in one launch.

    q (B, Hq, S, D) and k (B, Hk, S, D) with positions (B, S) or (S,), or
    packed rows q (T, Hq, D) and k (T, Hk, D) with positions (T,); fp16 or
    bf16, any strides; k may be None.  positions int32 or int64 (negative ones
    turn back).  The first 2 * len(inv_freq) elements of a head are turned, as
    pairs (p, p + half) or, ``interleaved``, (2p, 2p + 1), and scaled by
    ``amplitude``; the rest passes through.  ``inverse`` turns by the negative
    angles.  Angles are reduced to one turn in 64 bits, so far positions lose
    nothing.  Returns (q, k), or q alone without k: new tensors, or ``out``
    (a tensor or pair of them, which may be the inputs themselves; one that
    shares memory with an input otherwise, or with itself, is refused).
    """
    qo, ko = (out, None) if out is None or isinstance(out, torch.Tensor) else out
    if out is not None and (qo is None or (ko is None) != (k is None)):
        raise ValueError("apply_rotary: out must match (q, k)")
    return _native.ops().rotary(q, k, positions, inv_freq, interleaved, amplitude, inverse, qo, ko)
