"""Rotary positions on the GPU against the 64-bit form: both layouts, part of
the head, far and negative positions, any strides, in place, turned back."""

import pytest
import torch

import foveated_kv_b200 as fkv
from foveated_kv_b200 import FkvNativeError
from tests import paged_ref as R

pytestmark = pytest.mark.gpu


def _rand(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _flat(x):
    """(B, H, S, D) or (T, H, D) -> (tokens, H, D)"""
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3]) if x.dim() == 4 else x


def _check(x, y, pos, f, **kw):
    a = _flat(x).double()
    ref = R.rotate(a, pos.reshape(-1), f, kw.get("interleaved", False), kw.get("amplitude", 1.0), kw.get("inverse", False))
    slack = R.rotate_slack(a, f, kw.get("interleaved", False), kw.get("amplitude", 1.0))
    err = (_flat(y).double() - ref).abs()
    assert (err <= R.HALF_STEP[x.dtype] * (ref.abs() + slack) + slack + R.SUBNORMAL[x.dtype]).all(), float(err.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 32), (128, 24), (256, 256), (80, 80), (8, 8), (1024, 512), (40, 8)])
def test_layouts_and_partial_heads(D, rot, interleaved, dtype):
    f, _ = fkv.rotary_frequencies(rot)
    q, k = _rand(2, 5, 33, D, dtype=dtype), _rand(2, 2, 33, D, dtype=dtype, seed=1)
    pos = torch.randint(0, 40000, (2, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    qo, ko = fkv.apply_rotary(q, k, pos, f, interleaved=interleaved, amplitude=1.25)
    _check(q, qo, pos, f, interleaved=interleaved, amplitude=1.25)
    _check(k, ko, pos, f, interleaved=interleaved, amplitude=1.25)
    assert torch.equal(qo[..., rot:], q[..., rot:]) and torch.equal(ko[..., rot:], k[..., rot:])


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (1, 1, 32, 8), (64, 1, 14, 2), (1, 700, 3, 1), (3, 129, 28, 4)])
@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64])
def test_sizes_and_position_types(B, S, Hq, Hk, pdtype):
    f, _ = fkv.rotary_frequencies(128)
    q, k = _rand(B, Hq, S, 128, dtype=torch.float16), _rand(B, Hk, S, 128, dtype=torch.float16, seed=1)
    pos = (torch.arange(S)[None] + 11 * torch.arange(B)[:, None]).to(pdtype).cuda()
    qo, ko = fkv.apply_rotary(q, k, pos, f)
    _check(q, qo, pos, f)
    _check(k, ko, pos, f)
    same = pos[0]                                # one row of positions for every sequence
    _check(q, fkv.apply_rotary(q, None, same, f), same[None].expand(B, S), f)


def test_far_and_negative_positions():
    """At 2^30 positions a 32-bit angle would be off by whole turns."""
    f, _ = fkv.rotary_frequencies(128, 500000.0)
    pos = torch.tensor([2 ** 30, 2 ** 30 + 1, 1048575, -1, -12345, 0], device="cuda")
    q = _rand(6, 4, 128, dtype=torch.float16)
    _check(q, fkv.apply_rotary(q, None, pos, f), pos, f)


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_back(interleaved):
    f, _ = fkv.rotary_frequencies(64)
    q, k = _rand(100, 6, 128, dtype=torch.float16), _rand(100, 2, 128, dtype=torch.float16, seed=1)
    pos = torch.arange(100, device="cuda") * 317
    qo, ko = fkv.apply_rotary(q, k, pos, f, interleaved=interleaved)
    q2, k2 = q.clone(), k.clone()
    r = fkv.apply_rotary(q2, k2, pos, f, interleaved=interleaved, out=(q2, k2))
    assert r[0] is q2 and torch.equal(q2, qo) and torch.equal(k2, ko)
    back = fkv.apply_rotary(qo, None, pos, f, interleaved=interleaved, inverse=True)
    _check(qo, back, pos, f, interleaved=interleaved, inverse=True)
    # two roundings of half a step each, the first carried through a turn
    a = R.rotate_slack(q.double(), f, interleaved) * 2 ** 20        # |a| + |b| of the pair
    tol = 2.0 ** -11 * (a + q.double().abs()) + 2.0 ** -17 * a + 2.0 ** -24
    assert ((back.double() - q.double()).abs() <= tol).all()


def test_strides_views_and_alignment():
    f, _ = fkv.rotary_frequencies(128)
    qkv = _rand(50, 12, 128, dtype=torch.bfloat16)               # packed projection rows: q | k | v
    q, k = qkv[:, :8], qkv[:, 8:10]
    pos = torch.arange(50, device="cuda", dtype=torch.int32)
    v = qkv[:, 10:].clone()
    want = fkv.apply_rotary(q.contiguous(), k.contiguous(), pos, f)
    got = fkv.apply_rotary(q, k, pos, f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    fkv.apply_rotary(q, k, pos, f, out=(q, k))                   # in place inside the packed rows
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 10:], v)
    base = _rand(50 * 4 * 128 + 3, dtype=torch.float16)
    odd = base[3:].view(50, 4, 128)                              # 2 bytes off
    assert torch.equal(fkv.apply_rotary(odd, None, pos, f), fkv.apply_rotary(odd.clone(), None, pos, f))
    wide = _rand(50, 4, 256, dtype=torch.float16)[..., ::2]      # elements apart
    assert torch.equal(fkv.apply_rotary(wide, None, pos, f), fkv.apply_rotary(wide.contiguous(), None, pos, f))
    one = _rand(1, 4, 128, dtype=torch.float16).expand(50, 4, 128)   # the same row for every token
    assert torch.equal(fkv.apply_rotary(one, None, pos, f), fkv.apply_rotary(one.contiguous(), None, pos, f))
    step = pos.repeat_interleave(2)[::2]                         # positions with a stride
    assert torch.equal(fkv.apply_rotary(odd, None, step, f), fkv.apply_rotary(odd, None, pos, f))


@pytest.mark.parametrize("H,D,rot,T", [(1, 1024, 1024, 20000), (1, 64, 64, 40000), (300, 64, 32, 5000), (8192, 8, 8, 3)])
def test_many_tokens_or_heads(H, D, rot, T):
    f, _ = fkv.rotary_frequencies(rot)
    q, pos = _rand(T, H, D, dtype=torch.float16), torch.arange(T, device="cuda")
    _check(q, fkv.apply_rotary(q, None, pos, f), pos, f)


def test_overlapping_outputs_are_refused():
    f, _ = fkv.rotary_frequencies(64)
    buf, pos = _rand(11, 4, 64, dtype=torch.float16), torch.arange(10, device="cuda")
    q, k = buf[:10], _rand(10, 4, 64, dtype=torch.float16, seed=1)
    for out in ((buf[1:], k.clone()), (k, k.clone()), (q.clone(), q), (k, q)):
        with pytest.raises(ValueError):
            fkv.apply_rotary(q, k, pos, f, out=out)
    with pytest.raises(ValueError):
        fkv.apply_rotary(q, None, pos, f, out=buf[1:])


def test_empty_and_passed_through_values():
    f, _ = fkv.rotary_frequencies(64)
    pos = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert fkv.apply_rotary(_rand(0, 4, 128, dtype=torch.float16), None, pos, f).shape == (0, 4, 128)
    q = _rand(3, 4, 128, dtype=torch.float16)
    q[1, 2, 100] = float("nan")
    q[2, 0, 127] = float("inf")
    out = fkv.apply_rotary(q, None, torch.arange(3, device="cuda"), f)
    assert torch.equal(out[..., 64:].view(torch.int16), q[..., 64:].view(torch.int16))
    assert torch.isfinite(out[..., :64]).all()
    assert torch.equal(out[0], q[0])                             # position 0 turns nothing


def test_frequencies():
    f, a = fkv.rotary_frequencies(128, 10000.0)
    assert a == 1.0 and f.dtype == torch.float64 and f.shape == (64,)
    assert torch.allclose(f, 10000.0 ** -(torch.arange(64, device="cuda").double() / 64), rtol=1e-14, atol=0)
    lin, _ = fkv.rotary_frequencies(128, scaling="linear", factor=4.0)
    assert torch.allclose(lin * 4, f, rtol=1e-14, atol=0)
    ntk, _ = fkv.rotary_frequencies(128, scaling="ntk", factor=8.0)
    assert float(ntk[0]) == 1.0 and abs(float(f[-1] / ntk[-1]) - 8.0) < 1e-9      # only the slowest slows in full
    y, amp = fkv.rotary_frequencies(128, scaling="yarn", factor=8.0, original_len=4096)
    turns = f * 4096 / (2 * torch.pi)
    assert torch.equal(y[turns > 32], f[turns > 32]) and torch.allclose(y[turns < 1] * 8, f[turns < 1], rtol=1e-14)
    assert (y <= f).all() and (y >= f / 8 * (1 - 1e-14)).all() and abs(amp - 1.2079441541679836) < 1e-12


def test_other_stream_and_graph():
    f, _ = fkv.rotary_frequencies(128)
    q, pos = _rand(64, 8, 128, dtype=torch.float16), torch.arange(64, device="cuda")
    want = fkv.apply_rotary(q, None, pos, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fkv.apply_rotary(q, None, pos, f)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fkv.apply_rotary(q, None, pos, f)
    pos += 100
    g.replay()
    torch.cuda.synchronize()
    _check(q, out, pos, f)


def test_refusals():
    f, _ = fkv.rotary_frequencies(64)
    q, pos = _rand(4, 2, 64, dtype=torch.float16), torch.arange(4, device="cuda")
    for bad in (lambda: fkv.apply_rotary(q.float(), None, pos, f),
                lambda: fkv.apply_rotary(q[0], None, pos, f),
                lambda: fkv.apply_rotary(q, _rand(4, 2, 128, dtype=torch.float16), pos, f),
                lambda: fkv.apply_rotary(q, _rand(5, 2, 64, dtype=torch.float16), pos, f),
                lambda: fkv.apply_rotary(q, q.bfloat16(), pos, f),
                lambda: fkv.apply_rotary(q, None, pos[:3], f),
                lambda: fkv.apply_rotary(q, None, pos.float(), f),
                lambda: fkv.apply_rotary(q, None, pos.cpu(), f),
                lambda: fkv.apply_rotary(q, None, pos, f.float()),
                lambda: fkv.apply_rotary(q, None, pos, f, out=(q, q)),
                lambda: fkv.apply_rotary(q, None, pos, f, out=torch.empty(4, 2, 63, device="cuda", dtype=torch.float16)),
                lambda: fkv.apply_rotary(q, None, pos, f, out=q[:1].expand(4, 2, 64)),
                lambda: fkv.apply_rotary(q.clone().requires_grad_(), None, pos, f)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(FkvNativeError):                          # more rotated than the head has
        fkv.apply_rotary(q, None, pos, fkv.rotary_frequencies(128)[0])
    with pytest.raises(FkvNativeError):
        fkv.apply_rotary(_rand(4, 2, 68, dtype=torch.float16), None, pos, f)
    with torch.no_grad():
        fkv.apply_rotary(q.clone().requires_grad_(), None, pos, f)
