"""Paged cache and rotary entry points: refusals before any CUDA call, and the
wrappers' refusal of host tensors."""

import ctypes as C

import pytest
import torch

import foveated_kv_b200 as fkv
from foveated_kv_b200 import _native
from tests import paged_ref as R

DUMMY = 256                     # never dereferenced: the checks come first


def _cache(**kw):
    d = dict(k_pages=DUMMY, v_pages=DUMMY, k_scale=None, v_scale=None, table=DUMMY, lens=DUMMY, status=None,
             B=2, Hk=2, D=128, page=16, n_pages=10, width=4, table_stride=4, fp8=0, bf16=0, reserved=0)
    d.update(kw)
    return _native.PagedCache(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(D=96), -2), (dict(D=512), -2), (dict(page=24), -2), (dict(page=4), -2), (dict(page=512), -2),
    (dict(B=-1), -1), (dict(Hk=0), -1), (dict(n_pages=-1), -1), (dict(width=-1), -1), (dict(table_stride=3), -1),
    (dict(lens=None), -1), (dict(table=None), -1), (dict(k_pages=None), -1), (dict(fp8=1), -1),
    (dict(k_pages=DUMMY + 8), -1), (dict(width=1 << 28, table_stride=1 << 28), -2), (dict(width=(1 << 26) + 1, table_stride=1 << 27), -2),
])
def test_cache_descriptor_refusals(kw, rc):
    lib = _native.load()
    c = _cache(**kw)
    assert lib.fkv_paged_attend(C.byref(c), 4, 0.1, 0, DUMMY, DUMMY, None, DUMMY, 1 << 30, None) == rc
    assert lib.fkv_paged_read(C.byref(c), 5, DUMMY, DUMMY, None) == rc
    n = _native.PagedNew(T=2, n_uniform=1, k=DUMMY, v=DUMMY)
    assert lib.fkv_paged_append(C.byref(c), C.byref(n), None) == rc
    assert lib.fkv_last_error()


def test_attend_refusals():
    lib = _native.load()
    call = lambda c, Hq=4, window=0, q=DUMMY, out=DUMMY, ws=DUMMY, n=1 << 30: lib.fkv_paged_attend(
        C.byref(c), Hq, 0.1, window, q, out, None, ws, n, None)
    c = _cache()
    assert call(c, Hq=3) == -1 and call(c, Hq=0) == -1 and call(c, window=-1) == -1
    assert call(c, q=None) == -1 and call(c, out=DUMMY + 2) == -1
    assert call(_cache(n_pages=2 ** 31 - 1, Hk=1024), Hq=1024) == -2                    # rows beyond 32 bits
    assert call(_cache(B=2 ** 20, width=2 ** 12, table_stride=2 ** 12)) == -2  # more work units than 31 bits
    assert lib.fkv_paged_attend(None, 4, 0.1, 0, DUMMY, DUMMY, None, DUMMY, 0, None) == -1
    assert call(_cache(B=0)) == 0                                              # nothing to do


def test_workspace_sizes():
    lib = _native.load()
    size = lambda Hq=4, **kw: lib.fkv_paged_attend_workspace_bytes(C.byref(_cache(**kw)), Hq)
    assert size(width=1, table_stride=1) == 0                    # one unit a sequence: nothing to join
    assert size(width=40, table_stride=40) > 0
    assert size(width=400, table_stride=400) >= size(width=40, table_stride=40)
    assert size(Hq=3) == 0 and size(D=96) == 0 and size(page=24) == 0
    assert size(B=512, width=4000, table_stride=4000) < 64 << 20


def test_append_and_rotary_refusals():
    lib = _native.load()
    c = _cache()
    call = lambda **kw: lib.fkv_paged_append(C.byref(c), C.byref(_native.PagedNew(**dict(
        dict(T=2, n_uniform=1, k=DUMMY, v=DUMMY), **kw))), None)
    assert call(T=-1) == -1 and call(T=3) == -1 and call(k=None) == -1 and call(v=DUMMY + 4) == -1
    assert call(rot=12, inv_freq=DUMMY) == -2 and call(rot=136, inv_freq=DUMMY) == -2 and call(rot=64) == -1
    assert call(Hq=4, q=DUMMY, q_out=DUMMY) == -1                # queries without a rotation
    assert call(Hq=4, rot=64, inv_freq=DUMMY) == -1 and call(k_tok=6) == -1
    assert call(T=0, n_uniform=0) == 0
    rot = lambda **kw: lib.fkv_rotary(C.byref(_native.RotaryShape(**dict(
        dict(B=1, S=4, Hq=2, Hk=0, D=64, rot=64), **kw))), DUMMY, None, DUMMY, DUMMY, DUMMY, None, None)
    assert rot(D=60) == -2 and rot(D=2048) == -2 and rot(rot=72) == -2 and rot(rot=0) == -2 and rot(rot=20) == -2
    assert rot(B=-1) == -1 and rot(Hk=1) == -1 and rot(q_tok=2) == -1 and rot(S=0) == 0
    assert rot(B=2 ** 20, S=2 ** 20) == -2


def test_wrappers_refuse_host_tensors():
    f = torch.zeros(32, dtype=torch.float64)
    x, pos = torch.zeros(2, 4, 64, dtype=torch.float16), torch.arange(2)
    pages = torch.zeros(3, 4, 16, 64, dtype=torch.float16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: fkv.apply_rotary(x, None, pos, f), lambda: fkv.paged_attend(x, pages, pages, table, lens),
                 lambda: fkv.paged_append(x, x, pages, pages, table, lens),
                 lambda: fkv.paged_read(pages, pages, table, lens, 4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_frequency_refusals():
    for kw in (dict(rot_dim=12), dict(rot_dim=0), dict(rot_dim=64, scaling="other"), dict(rot_dim=64, base=0.0),
               dict(rot_dim=64, scaling="yarn", factor=2.0), dict(rot_dim=64, scaling="linear", factor=0.0)):
        with pytest.raises(ValueError):
            fkv.rotary_frequencies(device="cpu", **kw)


def test_e4m3_restatement():
    """The tests' own E4M3 rounding against torch's conversion, every code and the midpoints between."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    x = torch.cat([v, (v[1:] + v[:-1]) / 2, (v[1:] + v[:-1]) / 2 * (1 + 1e-6), torch.tensor([0.0, 2.0 ** -11, 448.0])])
    x = torch.cat([x, -x]).float()
    assert torch.equal(R.e4m3(x), x.to(torch.float8_e4m3fn).view(torch.uint8))
    assert R.e4m3(torch.tensor([1e9, float("nan"), -1e9])).tolist() == [0x7E, 0x7F, 0xFE]
