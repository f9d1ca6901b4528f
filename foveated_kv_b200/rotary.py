"""Rotary positions of queries and keys (no counterpart in the reference,
whose models rotate before they hand their keys to the cache)."""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _native

_F16 = torch.float16
_BF16 = torch.bfloat16


def refuse_grad(who: str, *tensors) -> None:
    """These operators serve; they carry no gradient."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{who}: inputs that require a gradient are not supported "
                                 "(call it under torch.no_grad())")


def rows16(who: str, name: str, t: torch.Tensor, dtype, index: int):
    """(t, strides of its sequence, token and head) as 16-bit rows that the
    kernels can address: contiguous heads, 8-byte aligned, strides of a
    multiple of 4 elements; t is copied where it is not so.  t is
    (B, H, S, D) or (tokens, H, D)."""
    if t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{who}: {name} is {t.dtype} on {t.device}, expected {dtype} on cuda:{index}")
    st = t.stride()
    if len(st) == 3:
        a, h, d = st
        s, b = a, 0
    else:
        b, h, s, d = st
    if d != 1 or (b | s | h) & 3 or t.data_ptr() & 7:
        return rows16(who, name, t.clone(memory_format=torch.contiguous_format), dtype, index)
    return t, (b, s, h)


def out16(who: str, name: str, t: torch.Tensor, like: torch.Tensor, index: int):
    """The same of a tensor that is written: it must be so already."""
    if t.shape != like.shape:
        raise ValueError(f"{who}: {name} is {tuple(t.shape)}, expected {tuple(like.shape)}")
    r, st = rows16(who, name, t, like.dtype, index)
    if r is not t or any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{who}: {name} must be 8-byte aligned rows that do not overlap, with strides of a "
                         "multiple of 4 elements")
    return r, st


def on_device(index: int, fn, *args) -> int:
    """fn(*args, the device's current stream), with that device current."""
    if torch._C._cuda_getDevice() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def check_frequencies(who: str, inv_freq: torch.Tensor, index: int) -> None:
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or inv_freq.get_device() != index \
            or not inv_freq.is_contiguous():
        raise ValueError(f"{who}: inv_freq must be a contiguous float64 vector on cuda:{index}")


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
                than ``fast_turns`` stay, the others in between; the amplitude
                is 0.1 ln(factor) + 1 (Peng et al., 2023)
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
    f = float(base) ** -(torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
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
    (a tensor or pair of them, which may be the inputs themselves).
    """
    who = "apply_rotary"
    dt, index, shape = q.dtype, q.get_device(), q.shape
    if index < 0:
        raise ValueError(f"{who}: q must be a CUDA tensor")
    if dt is not _F16 and dt is not _BF16:
        raise ValueError(f"{who}: q is {dt}, expected float16 or bfloat16")
    refuse_grad(who, q, k)
    ps = positions.shape
    if len(shape) == 4:
        B, Hq, S, D = shape
        fits = ps == (B, S) or ps == (S,)
    elif len(shape) == 3:
        S, Hq, D = shape
        B = 1
        fits = ps == (S,)
    else:
        raise ValueError(f"{who}: q must be (B, H, S, D) or (T, H, D), got {tuple(shape)}")
    pd = positions.dtype
    if not fits or (pd is not torch.int64 and pd is not torch.int32) or positions.get_device() != index:
        raise ValueError(f"{who}: positions {tuple(ps)} {pd} do not go with q {tuple(shape)}: int32 or int64 "
                         "(B, S), (S,) or, packed, (T,), on q's device")
    check_frequencies(who, inv_freq, index)
    pst = positions.stride()
    if len(pst) == 1:
        pst = (0, pst[0])
    qo = ko = None
    if out is not None:
        qo, ko = (out, None) if isinstance(out, torch.Tensor) else out
        if qo is None or (ko is None) != (k is None):
            raise ValueError(f"{who}: out must match (q, k)")
    q, q_st = rows16(who, "q", q, dt, index)
    qo, qo_st = rows16(who, "out", torch.empty_like(q), dt, index) if qo is None else out16(who, "out", qo, q, index)
    Hk, k_ptr, ko_ptr, k_st, ko_st = 0, None, None, (0, 0, 0), (0, 0, 0)
    if k is not None:
        kshape = k.shape
        if len(kshape) != len(shape) or kshape[-1] != D or kshape[0] != shape[0] \
                or (len(shape) == 4 and kshape[2] != S):
            raise ValueError(f"{who}: k {tuple(kshape)} does not go with q {tuple(shape)}")
        Hk = kshape[1]
        k, k_st = rows16(who, "k", k, dt, index)
        ko, ko_st = rows16(who, "out", torch.empty_like(k), dt, index) if ko is None else \
            out16(who, "out", ko, k, index)
        k_ptr, ko_ptr = k.data_ptr(), ko.data_ptr()
    sh = _native.RotaryShape(B, S, Hq, Hk, D, 2 * inv_freq.numel(), dt is _BF16, interleaved, inverse,
                             pd is torch.int64, amplitude, 0, *pst, *q_st, *qo_st, *k_st, *ko_st)
    _native.check(on_device(index, _native.load().fkv_rotary, C.byref(sh), q.data_ptr(), k_ptr,
                            positions.data_ptr(), inv_freq.data_ptr(), qo.data_ptr(), ko_ptr), "fkv_rotary")
    return qo if k is None else (qo, ko)
