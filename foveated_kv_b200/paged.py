"""Paged key-value cache: sequences of any lengths in one pool of pages, next
to the tiered cache, which wants one length for a whole batch (no counterpart
in the reference).

``paged_append`` writes new tokens (rotating and quantising them on the way),
``paged_attend`` attends one new token per sequence over its pages, and
``paged_read`` gives a sequence back as dense keys and values, for instance
for ``compress_layer``.  ``PagedKVCache`` keeps the pages, the page table and
the free list of all layers.

Tensors shared by the three functions, P pages of ``page`` tokens:
  k_pages, v_pages  (P, Hk, page, D) float16, bfloat16 or float8_e4m3fn; D 64,
                    128 or 256, page a power of two from 8 to 256
  k_scale, v_scale  (P, Hk, page) float32, for float8 pages: a stored row is
                    its codes times this
  table             (B, W) int32: page of tokens [j * page, (j + 1) * page) of
                    sequence b; entries behind a sequence's end are not read
  lens              (B,) int32: tokens of each sequence, new ones included
  status            optional int32 word of sticky error bits: 1 = a table entry
                    that is no page (its tokens are left out), 2 = a length or
                    position below zero or outside the table
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native
from .cache import FoveatedKVCache, compress_layer
from .config import TierConfig

_F16 = torch.float16
_BF16 = torch.bfloat16
_F8 = torch.float8_e4m3fn
_I32 = torch.int32
BAD_PAGE, BAD_POSITION = 1, 2


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 table: torch.Tensor, lens: torch.Tensor, *, cu_new: Optional[torch.Tensor] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False, amplitude: float = 1.0, q_out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write new tokens into their sequences' pages, in one launch.

    k, v (B, Hk, n, D): n tokens for each sequence; or (B, Hk, D): one token
    each; a sequence of length 0 is an empty slot and gets none.  With cu_new
    (B + 1,) int32: packed rows (T, Hk, D), sequence b's are
    [cu_new[b], cu_new[b + 1]), rows behind the last are padding.  The new
    tokens are the last of their sequences (``lens`` counts them), and two
    sequences must not be given the same page to write.  k, v and q must share
    no memory with the pages or their scales, q_out with nothing but q.

    With inv_freq the keys are rotated by their positions before they are
    stored (``apply_rotary``'s arguments), and so is q, which has k's layout
    and Hq heads; the rotated q is returned (q_out, which may be q itself, or a
    new tensor), zeros for tokens that are not stored.  float8 pages quantise
    each row: scale = max(|row|, 2^-100) / 448, a row with an infinity or a NaN
    reads back as NaN.
    """
    return _native.ops().paged_append(k_pages, v_pages, table, lens, k_scale, v_scale, status, k, v, cu_new, q,
                                      inv_freq, interleaved, amplitude, q_out)


def paged_read(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, max_len: int,
               *, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None):
    """The sequences' first max_len tokens as dense (k, v), each
    (B, Hk, max_len, D) of ``dtype`` (the pages' own type, or float16 for
    float8 pages), with zeros behind a sequence's end."""
    return _native.ops().paged_read(k_pages, v_pages, table, lens, k_scale, v_scale, status, max_len, dtype)


def paged_attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, *, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: int = 0,
                 return_lse: bool = False, out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None):
    """Attention of one new token per sequence over its pages.

    q (B, Hq, D) or (B, Hq, 1, D), Hq a multiple of Hk; ``scale`` is 1/sqrt(D) by
    default and ``window`` > 0 attends the last ``window`` tokens only.  The
    pages' own scales must not be negative.  Returns out, of q's shape, and with
    return_lse the natural log-sum-exp of the scaled scores, (B, Hq) float32.

    A sequence without tokens, or with none that has a page, gives zeros and
    -inf.  A score of +inf gives NaN and +inf; scores that are all -inf give NaN
    and -inf; an infinite value gives a non-finite output.  Beside float8 pages
    the softmax weights are rounded to float16.  ``out`` must share memory with
    nothing else.

    Lengths are read on the device, so the call can be captured once and
    replayed as sequences grow within the table; neither they nor the table may
    change while it runs.  The work split follows the table's width and the
    lengths: the same inputs give the same bits, a wider table may round
    differently.
    """
    return _native.ops().paged_attend(k_pages, v_pages, table, lens, k_scale, v_scale, status, q, scale, window,
                                      return_lse, out)


class PagedKVCache:
    """Pages, page table and free list of all layers of a serving batch.

    A slot (row of the batch) holds one sequence.  A step is ``extend(counts)``
    (pages for the new tokens, lengths and table on the device), then for every
    layer ``append`` and ``attend``; ``release(slot)`` gives its pages back.
    With at most one new token per slot, k, v and q of the step have a row per
    slot (rows of slots without a new token are ignored); otherwise they are
    packed, in slot order.  ``append`` and ``attend`` can be captured in a CUDA
    graph between ``extend`` calls of the same kind: the page table, lengths and
    counts they read are updated in place.
    """

    def __init__(self, n_layers: int, n_pages: int, H_kv: int, D: int, *, page: int = 16, max_seqs: int = 1,
                 max_len: int, fmt: str = "16", dtype: torch.dtype = _F16, inv_freq=None, interleaved: bool = False,
                 amplitude: float = 1.0, device="cuda"):
        if fmt not in ("16", "fp8"):
            raise ValueError(f"fmt must be '16' or 'fp8', got {fmt!r}")
        if dtype not in (_F16, _BF16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        if min(n_layers, n_pages, H_kv, max_seqs, max_len) < 1:
            raise ValueError("sizes must be at least 1")
        if D not in (64, 128, 256):
            raise ValueError(f"head dim {D} unsupported (64, 128 or 256)")
        if page < 8 or page > 256 or page & (page - 1):
            raise ValueError(f"page {page} is not a power of two from 8 to 256")
        self.n_layers, self.n_pages, self.H_kv, self.D = n_layers, n_pages, H_kv, D
        self.page, self.max_seqs, self.max_len, self.dtype, self.fmt = page, max_seqs, max_len, dtype, fmt
        self.inv_freq, self.interleaved, self.amplitude = inv_freq, interleaved, float(amplitude)
        shape = (n_pages, H_kv, page, D)
        kind = _F8 if fmt == "fp8" else dtype
        new = lambda: torch.zeros(shape, dtype=torch.uint8 if kind is _F8 else kind, device=device).view(kind)
        scale = lambda: torch.zeros(shape[:3], dtype=torch.float32, device=device) if kind is _F8 else None
        self.layers = [dict(k_pages=new(), v_pages=new(), k_scale=scale(), v_scale=scale()) for _ in range(n_layers)]
        self.width = -(-max_len // page)
        self.table = torch.full((max_seqs, self.width), -1, dtype=_I32, device=device)
        # lengths; lengths of the slots with a new token in this step, else 0; the
        # counts' prefix sums
        self._state = torch.zeros(3 * max_seqs + 1, dtype=_I32, device=device)
        self.lens, self._step_lens, self._cu = self._state.split([max_seqs, max_seqs, max_seqs + 1])
        self.status = torch.zeros(1, dtype=_I32, device=device)
        self.device = self.table.device
        self._packed = None                                                   # None: no step begun
        self._new_rows = 0
        self._lens = [0] * max_seqs
        self._pages = [[] for _ in range(max_seqs)]
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def lengths(self) -> list:
        return list(self._lens)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, counts: Sequence[int]) -> None:
        """Begin a step that adds counts[slot] tokens to each slot: takes pages
        and updates the table and the lengths.  Nothing changes when the pages
        do not suffice or a sequence would pass max_len."""
        counts = [int(c) for c in counts]
        if len(counts) != self.max_seqs or min(counts) < 0:
            raise ValueError(f"extend: need {self.max_seqs} counts of 0 or more")
        lens = [a + c for a, c in zip(self._lens, counts)]
        if max(lens) > self.max_len:
            raise ValueError(f"extend: a sequence of {max(lens)} tokens passes max_len {self.max_len}")
        need = [-(-n // self.page) - len(p) for n, p in zip(lens, self._pages)]
        if sum(need) > len(self._free):
            raise _native.FkvNativeError(f"extend: {sum(need)} pages needed, {len(self._free)} free")
        at = [s * self.width + len(self._pages[s]) + i for s, m in enumerate(need) for i in range(m)]
        ids = self._free[len(self._free) - len(at):][::-1]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        # the device first: if a copy fails, nothing is taken
        upd = self._send([at, ids], torch.int64) if at else None
        state = self._send(lens + [n if c else 0 for n, c in zip(lens, counts)] + cu, _I32)
        if at:
            self.table.view(-1)[upd[0]] = upd[1].to(_I32)
        self._state.copy_(state)
        for j, page in zip(at, ids):
            self._pages[j // self.width].append(page)
        del self._free[len(self._free) - len(at):]
        self._lens = lens
        self._packed = max(counts) > 1
        self._new_rows = sum(counts) if self._packed else self.max_seqs

    def _send(self, values, dtype) -> torch.Tensor:
        """Host values on the device, without waiting for the stream."""
        return torch.tensor(values, dtype=dtype, device="cpu", pin_memory=True).to(self.device, non_blocking=True)

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.max_seqs:
            raise ValueError(f"slot {slot} of {self.max_seqs}")

    def release(self, slot: int) -> None:
        """Empty a slot, between steps; its pages may be given to other
        sequences."""
        self._check_slot(slot)
        self._free.extend(reversed(self._pages[slot]))
        self._pages[slot] = []
        self._lens[slot] = 0
        self.table[slot].fill_(-1)
        self.lens[slot:slot + 1].zero_()
        self._step_lens[slot:slot + 1].zero_()

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None):
        """Write the step's keys and values of one layer; returns q, rotated
        if the cache has rotary frequencies (keys are then stored rotated)."""
        if self._packed is None:
            raise ValueError("append: call extend first")
        if k.shape[0] != self._new_rows if not self._packed else k.shape[0] < self._new_rows:
            raise ValueError(f"append: {k.shape[0]} rows of k, the step has {self._new_rows}")
        if k.dim() == 4 and (self._packed or k.shape[2] != 1):
            raise ValueError(f"append: k {tuple(k.shape)}, expected (rows, H_kv, D)" +
                             ("" if self._packed else " or (slots, H_kv, 1, D)"))
        turn = {} if self.inv_freq is None else dict(inv_freq=self.inv_freq, interleaved=self.interleaved,
                                                     amplitude=self.amplitude, q=q)
        lens, cu = (self.lens, self._cu) if self._packed else (self._step_lens, None)
        r = paged_append(k, v, table=self.table, lens=lens, cu_new=cu, status=self.status, **turn,
                         **self.layers[layer])
        return q if self.inv_freq is None else r

    def attend(self, layer: int, q: torch.Tensor, *, scale: Optional[float] = None, window: int = 0,
               return_lse: bool = False, out: Optional[torch.Tensor] = None):
        """Attention of one token per slot, q (max_seqs, Hq, D), over its sequence."""
        return paged_attend(q, table=self.table, lens=self.lens, scale=scale, window=window, return_lse=return_lse,
                            out=out, status=self.status, **self.layers[layer])

    def read(self, layer: int, slot: int):
        """One sequence as dense keys and values (1, H_kv, length, D)."""
        self._check_slot(slot)
        n = self._lens[slot]
        return paged_read(table=self.table[slot:slot + 1], lens=self.lens[slot:slot + 1], max_len=n,
                          dtype=self.dtype, status=self.status, **self.layers[layer])

    def compress(self, slot: int, cfg: Optional[TierConfig] = None, query=None,
                 keep_archive: bool = True) -> FoveatedKVCache:
        """Hand one sequence to the tiered cache: every layer read back and
        tiered by ``compress_layer``.  The slot keeps its pages."""
        self._check_slot(slot)
        if self._lens[slot] == 0:
            raise ValueError(f"compress: slot {slot} is empty")
        fov = FoveatedKVCache(cfg)
        fov.layers = [compress_layer(*self.read(i, slot), fov.cfg,
                                     query[i] if isinstance(query, (list, tuple)) else query, keep_archive)
                      for i in range(self.n_layers)]
        fov.seq_length = self._lens[slot]
        fov._compressed = True
        return fov

    def check(self) -> None:
        """Raise FkvNativeError if a launch met a bad page or position since
        the last check.  Waits for the current stream."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [t for b, t in ((BAD_PAGE, "a table entry that is no page"),
                                   (BAD_POSITION, "a length or position outside the table")) if bits & b]
            raise _native.FkvNativeError("paged cache: " + " and ".join(what))

    def memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for lay in self.layers for t in lay.values() if t is not None)
