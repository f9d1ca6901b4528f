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


def rows16(who: str, name: str, t: torch.Tensor, dtype, device) -> torch.Tensor:
    """t as 16-bit rows the kernels can address: contiguous heads, 8-byte
    aligned, strides of a multiple of 4 elements; copied where it is not."""
    if t.dtype is not dtype or t.device != device:
        raise ValueError(f"{who}: {name} is {t.dtype} on {t.device}, expected {dtype} on {device}")
    st = t.stride()
    if st[-1] != 1 or t.data_ptr() & 7 or any(s & 3 for s in st[:-1]):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def on_device(device: torch.device, fn, *args) -> int:
    """fn(*args, the device's current stream), with that device current."""
    i = device.index
    if torch.cuda.current_device() == i:
        return fn(*args, torch._C._cuda_getCurrentRawStream(i))
    with torch.cuda.device(i):
        return fn(*args, torch._C._cuda_getCurrentRawStream(i))


def check_frequencies(who: str, inv_freq: torch.Tensor, device) -> None:
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or inv_freq.device != device \
            or not inv_freq.is_contiguous():
        raise ValueError(f"{who}: inv_freq must be a contiguous float64 vector on {device}")


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
    if not q.is_cuda:
        raise ValueError(f"{who}: q must be a CUDA tensor")
    dev, dt = q.device, q.dtype
    if dt is not _F16 and dt is not _BF16:
        raise ValueError(f"{who}: q is {dt}, expected float16 or bfloat16")
    nd = q.dim()
    if nd not in (3, 4):
        raise ValueError(f"{who}: q must be (B, H, S, D) or (T, H, D), got {tuple(q.shape)}")
    refuse_grad(who, q, k)
    shape = q.shape
    if nd == 4:
        B, Hq, S, D = shape
    else:
        B, (S, Hq, D) = 1, shape
    Hk = 0
    if k is not None:
        want = (B, k.shape[1], S, D) if nd == 4 else (S, k.shape[1], D)
        if tuple(k.shape) != want:
            raise ValueError(f"{who}: k {tuple(k.shape)} does not go with q {tuple(shape)}")
        Hk = k.shape[1]
    if positions.device != dev or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: positions must be int32 or int64 on {dev}")
    if tuple(positions.shape) not in (((B, S), (S,)) if nd == 4 else ((S,),)):
        raise ValueError(f"{who}: positions {tuple(positions.shape)} do not go with q {tuple(shape)}")
    check_frequencies(who, inv_freq, dev)

    outs = (None, None) if out is None else (out, None) if isinstance(out, torch.Tensor) else tuple(out)
    if out is not None and (len(outs) != 2 or (outs[1] is None) != (k is None)):
        raise ValueError(f"{who}: out must match (q, k)")
    sh = _native.RotaryShape(B, S, Hq, Hk, D, 2 * inv_freq.numel(), dt is _BF16, interleaved, inverse,
                             positions.dtype is torch.int64, amplitude)
    sh.pos_stride[:] = positions.stride() if positions.dim() == 2 else (0, positions.stride(0) if S else 0)
    ptrs, res = [], []
    for name, x, o, fin, fout in (("q", q, outs[0], sh.q_stride, sh.q_out_stride),
                                  ("k", k, outs[1], sh.k_stride, sh.k_out_stride)):
        if x is None:
            ptrs += [None, None]
            continue
        x = rows16(who, name, x, dt, dev)
        if o is None:
            o = torch.empty(x.shape, dtype=dt, device=dev)
        elif o.shape != x.shape or rows16(who, "out", o, dt, dev) is not o \
                or any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
            raise ValueError(f"{who}: out for {name} has another shape, or is not 8-byte aligned "
                             "rows with strides of a multiple of 4 elements")
        for t, f in ((x, fin), (o, fout)):
            st = t.stride()
            f[:] = (st[0], st[2], st[1]) if nd == 4 else (0, st[0], st[1])
        ptrs += [x.data_ptr(), o.data_ptr()]
        res.append(o)
    _native.check(on_device(dev, _native.load().fkv_rotary, C.byref(sh), ptrs[0], ptrs[2], positions.data_ptr(),
                            inv_freq.data_ptr(), ptrs[1], ptrs[3]), "fkv_rotary")
    return res[0] if k is None else tuple(res)
