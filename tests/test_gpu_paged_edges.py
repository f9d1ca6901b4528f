"""Edges of the paged cache's and rotary calls on the GPU: tokens that are left
out, lengths that are none, weights far below the largest, calls that are
refused."""

import math

import pytest
import torch

import foveated_kv_b200 as fkv
from foveated_kv_b200 import FkvNativeError, PagedKVCache
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
INF = float("inf")


def _rand(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ---- attention: tokens left out -----------------------------------------------------------------

@pytest.mark.parametrize("D,G", [(64, 4), (64, 16), (128, 8), (256, 2)])
@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("n", [40, 30000])                       # one CTA's work, many CTAs'
def test_tokens_all_left_out(n, dtype, fp8, D, G):
    """No table entry that is a page: as a sequence without tokens."""
    p = R.Pages(1, [n, 33, 5], 2, D, 16, dtype, fp8, width_extra=0)
    q = _rand(3, 2 * G, D, dtype=dtype)
    want, wlse = fkv.paged_attend(q, return_lse=True, **p.kw)
    t, st = p.table.clone(), _status()
    t[0] = -1
    out, lse = fkv.paged_attend(q, return_lse=True, status=st, **dict(p.kw, table=t))
    assert st.item() == 1 and (out[0] == 0).all() and (lse[0] == -INF).all()
    assert torch.equal(out[1:], want[1:]) and torch.equal(lse[1:], wlse[1:])
    t = p.table.clone()                                          # a window wholly on bad pages
    t[0, (n - 20) // 16:] = p.k_pages.shape[0]
    out, lse = fkv.paged_attend(q, return_lse=True, window=20, **dict(p.kw, table=t))
    assert (out[0] == 0).all() and (lse[0] == -INF).all() and torch.isfinite(out[1:]).all()
    t = p.table.clone()                                          # the first half left out
    cut = n // 32 * 16
    t[0, :cut // 16] = -1
    out, lse = fkv.paged_attend(q, return_lse=True, **dict(p.kw, table=t))
    ref, rlse, mag, dot = R.attend(q, [x[:, cut if b == 0 else 0:] for b, x in enumerate(p.sequences("k"))],
                                   [x[:, cut if b == 0 else 0:] for b, x in enumerate(p.sequences("v"))], [n - cut, 33, 5])
    slack = R.attend_slack(dtype, fp8, [n], dot, mag, 6.0)
    tol = R.HALF_STEP[dtype] * (ref.abs() + slack) + slack + R.SUBNORMAL[dtype]
    assert ((out.double() - ref).abs() <= tol).all()
    assert (lse.double() - rlse).abs().max() <= 2.0 ** -18 * float(dot.max()) + (n / 16 + 64) * 2.0 ** -22


@pytest.mark.parametrize("fp8", [False, True])
def test_tokens_of_an_empty_pool(fp8):
    p = R.Pages(2, [0, 0], 2, 64, 16, F16, fp8, spare=0)
    kw = dict(p.kw, lens=torch.tensor([20, 3], dtype=torch.int32, device="cuda"), table=p.table.abs())
    out, lse = fkv.paged_attend(_rand(2, 4, 64, dtype=F16), return_lse=True, **kw)
    assert (out == 0).all() and (lse == -INF).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [40, 30000])
def test_scores_all_minus_infinity(n, dtype):
    """Tokens that are there with scores of -inf are not left out: 0 / 0, with
    a log-sum-exp of -inf, beside pages that are missing as without them."""
    p = R.Pages(3, [n], 1, 64, 16, dtype, False, width_extra=0)
    p.k_pages[p.table[0].long()] = -INF
    q = _rand(1, 4, 64, dtype=dtype).abs() + 0.1
    t = p.table.clone()
    t[0, 1:-1] = -1
    for table in (p.table, t):
        out, lse = fkv.paged_attend(q, return_lse=True, **dict(p.kw, table=table))
        assert torch.isnan(out).all() and (lse == -INF).all()


# ---- attention: shares of several waves ---------------------------------------------------------

@pytest.mark.parametrize("G,Hk,D,lens,waves", [
    (8, 8, 64, [200000], 2),                                     # a descriptor for each stream
    (16, 4, 128, [600000], 2),
    (8, 8, 64, [760000], 3),
    (4, 8, 64, [400000, 77, 0, 300001, 80000], 3),
    (8, 16, 64, [9000 - 37 * i for i in range(48)], 3),
    (8, 16, 64, [4100 - 3 * i for i in range(100)], 3),          # a descriptor for each CTA
])
def test_shares_of_several_waves(G, Hk, D, lens, waves):
    """8-bit pages and much work: falling shares, of the wave count that the
    units of work make, with every token in exactly one of them."""
    per_sm = 2 if G == 16 else 3
    ctas = per_sm * torch.cuda.get_device_properties(0).multi_processor_count
    each = sum(-(-n // 128) for n in lens) * Hk // ctas
    assert {2: 24 <= each < 98, 3: each >= 102}[waves], each     # where two and three waves begin, with some room
    p = R.Pages(10, lens, Hk, D, 64, BF16, True, k_scale=0.1)
    B, Hq = len(lens), G * Hk
    # scores all alike: the sum counts the tokens, the output is the mean value
    q = torch.zeros(B, Hq, D, dtype=BF16, device="cuda")
    out, lse = fkv.paged_attend(q, return_lse=True, **p.kw)
    vs = p.sequences("v")
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == -INF).all()
            continue
        # sums of equal weights are exact; log2 of up to 2^35 and its product to a few steps of 2^-18; a unit is 1.6e-4
        assert (lse[b].double() - math.log(n)).abs().max() < 2.0 ** -16
        mean, mag = vs[b].mean(1).repeat_interleave(G, 0), vs[b].abs().mean(1).repeat_interleave(G, 0)
        tol = (n / 16 + 64) * 2.0 ** -23 * mag + 2.0 ** -11 * mag
        assert ((out[b].double() - mean).abs() <= 2.0 ** -8 * (mean.abs() + tol) + tol).all()
    # one token that takes all the weight of a head, somewhere in each sequence, a place for each head
    rng = torch.Generator().manual_seed(11)
    raw = p.k_pages.view(torch.uint8)
    want, live = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda"), []
    for b, n in enumerate(lens):
        if n < Hq:
            continue
        live.append(b)
        at = torch.randperm(n, generator=rng)[:Hq].cuda()
        head, j = torch.arange(Hq, device="cuda") // G, torch.arange(Hq, device="cuda") % G
        ids, row = p.table[b, at // 64].long(), at % 64
        raw[ids, head, row] = 0
        raw[ids, head, row, j] = 0x7E                            # 448
        p.k_scale[ids, head, row] = 40.0 / 448.0
        want[b] = vs[b][head, at]
        q[b, torch.arange(Hq), j] = 1.0
    out, lse = fkv.paged_attend(q, scale=1.0, return_lse=True, **p.kw)
    # the others' weight: under 2^20 e^(1 - 40) = 2^-36 of values up to 6
    err = (out.double() - want)[live].abs()
    assert (err <= (2.0 ** -8 + 2.0 ** -10) * want[live].abs() + 2.0 ** -30).all()
    assert (lse[live] - 40.0).abs().max() < 2.0 ** -15
    assert torch.equal(fkv.paged_attend(q, scale=1.0, **p.kw), out)


# ---- attention: weights far below the largest ---------------------------------------------------

@pytest.mark.parametrize("bits", [20, 25, 28])
@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("n", [500, 30000])
def test_many_small_weights(n, dtype, fp8, bits):
    """One token with a value of zero takes most of the weight, the others
    2^-bits of it each: the output is the others' sum."""
    p = R.Pages(4, [n], 1, 64, 16, dtype, fp8)
    for x in (p.k_pages, p.v_pages):
        x.view(torch.uint8).zero_()
    ids = p.table[0, :-(-n // 16)].long()
    first = ids[0]
    p.k_pages[first, 0, 0, 0] = 1.0
    v = torch.rand(len(ids), 1, 16, 64, generator=torch.Generator("cuda").manual_seed(5), device="cuda") + 0.5
    v[0, :, 0] = 0.0
    p.v_pages[ids] = (v * (256 if fp8 else 16384)).to(p.v_pages.dtype)
    if fp8:
        p.k_scale.fill_(1.0)
        p.v_scale.fill_(64.0)
    q = torch.zeros(1, 4, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    scale = bits * math.log(2.0)
    out = fkv.paged_attend(q, scale=scale, **p.kw).double()
    ref, _, mag, dot = R.attend(q, p.sequences("k"), p.sequences("v"), [n], 0, scale)
    slack = R.attend_slack(dtype, fp8, [n], dot, mag, 0.0)
    if fp8 or dtype is F16:
        # a part of a weight below f16's normal numbers is off by up to 2^-25 / 2^11, where the largest weight is at least 1
        slack = slack + n * 2.0 ** -36 * 24576.0
    assert ((out - ref).abs() <= R.HALF_STEP[dtype] * (ref.abs() + slack) + slack + R.SUBNORMAL[dtype]).all()


# ---- lengths below zero -------------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [64, 30000])
def test_negative_lengths_are_reported(n, fp8):
    p = R.Pages(5, [5, n, 9], 2, 64, 16, F16, fp8)
    q, st = _rand(3, 4, 64, dtype=F16), _status()
    want = fkv.paged_attend(q, status=st, **p.kw)
    assert st.item() == 0
    for bad in (-1, -2 ** 31):
        kw = dict(p.kw, lens=torch.tensor([bad, n, 9], dtype=torch.int32, device="cuda"))
        out, lse = fkv.paged_attend(q, status=st, return_lse=True, **kw)
        assert st.item() == 2 and (out[0] == 0).all() and (lse[0] == -INF).all()
        assert (out[1:].double() - want[1:].double()).abs().max() < 2.0 ** -8    # the work is split otherwise
        st.zero_()
        k, v = fkv.paged_read(max_len=9, dtype=F16, status=st, **kw)
        assert st.item() == 2 and (k[0] == 0).all() and (v[0] == 0).all()
        st.zero_()


# ---- writing ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, True)])
def test_append_of_padding_alone(dtype, fp8):
    """No sequences at all, rows of padding: their queries are zeros."""
    p = R.Pages(6, [20], 2, 64, 16, dtype, fp8)
    before = [x.view(torch.uint8).clone() for x in (p.k_pages, p.v_pages)]
    kw = dict(p.kw, table=p.table[:0], lens=p.lens[:0])
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, q = _rand(700, 2, 64, dtype=dtype), _rand(700, 6, 64, dtype=dtype)
    f, st = fkv.rotary_frequencies(64)[0], _status()
    new = lambda *shape: torch.full(shape, 7.0, dtype=dtype, device="cuda")
    wide = new(700, 9, 64)
    for got in (new(700, 6, 64), wide[:, 1:7], new(6, 700, 64).transpose(0, 1)):
        fkv.paged_append(k, k, cu_new=cu, q=q, q_out=got, inv_freq=f, status=st, **kw)
        assert (got == 0).all() and st.item() == 0
    assert (wide[:, 0] == 7).all() and (wide[:, 7:] == 7).all()
    assert (fkv.paged_append(k[:1], k[:1], cu_new=cu, q=q[:1], inv_freq=f, **kw) == 0).all()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (p.k_pages, p.v_pages)))
    fkv.paged_append(k, k, cu_new=cu, **kw)
    fkv.paged_append(k[:0], k[:0], **kw)


def test_cache_takes_one_row_per_slot():
    """A step of single tokens given as (slots, heads, n, D) with n other than 1
    would write over tokens that are there."""
    c = PagedKVCache(1, 8, 2, 64, page=8, max_seqs=2, max_len=32)
    c.extend([5, 3])
    old = _rand(8, 2, 64, dtype=F16, seed=1)
    c.append(0, old, old)
    c.extend([1, 1])
    for n in (0, 2, 3):
        k = _rand(2, 2, n, 64, dtype=F16, seed=2)
        with pytest.raises(ValueError, match="append"):
            c.append(0, k, k)
    k = _rand(2, 2, 1, 64, dtype=F16, seed=3)
    c.append(0, k, k)
    got = c.read(0, 0)[0][0]
    assert torch.equal(got[:, :5], old[:5].transpose(0, 1)) and torch.equal(got[:, 5], k[0, :, 0])
    c.extend([2, 0])
    for shape in ((2, 2, 1, 64), (2, 2, 2, 64)):                 # packed rows have three dimensions
        with pytest.raises(ValueError, match="append"):
            c.append(0, k.expand(shape), k.expand(shape))
    c.check()


# ---- shared memory ------------------------------------------------------------------------------

def test_outputs_that_share_memory_are_refused():
    p, e = (R.Pages(8, [20, 100], 2, 64, 16, F16, fp8) for fp8 in (False, True))
    f, pos = fkv.rotary_frequencies(64)[0], torch.arange(2, device="cuda")
    qkv = _rand(2, 8, 64, dtype=F16)                             # packed rows: 4 q, 2 k, 2 v
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    other = lambda x: x.clone()
    half = lambda x, n: x.view(-1).view(torch.uint8)[:n * 128].view(F16).view(2, -1, 64)    # its first rows as f16
    store = torch.zeros(2 ** 14, dtype=F16, device="cuda")
    folded = store.as_strided((2, 4, 64), (256, 32, 1))
    far = torch.zeros(64, dtype=torch.int64, device="cuda")      # positions with rows of f16 over them
    pool = torch.zeros(p.k_pages.shape[0] + 1, *p.k_pages.shape[1:], dtype=F16, device="cuda")
    rotary = lambda **kw: fkv.apply_rotary(**dict(dict(q=q, k=k, positions=pos, inv_freq=f), **kw))
    append = lambda p=p, **kw: fkv.paged_append(**dict(dict(k=k, v=v, q=q, inv_freq=f, **p.kw), **kw))
    attend = lambda p=p, **kw: fkv.paged_attend(**dict(dict(q=other(q), **p.kw), **kw))
    bad = [
        lambda: rotary(out=(qkv[:, 1:5], other(k))), lambda: rotary(k=None, out=qkv[:, 1:5]),
        lambda: rotary(out=(qkv[:, 2:6], other(k))), lambda: rotary(out=(other(q), qkv[:, 3:5])),
        lambda: rotary(out=(folded, other(k))),
        lambda: rotary(out=(store[:512].view(2, 4, 64), store[256:512].view(2, 2, 64))),
        lambda: rotary(q=other(q)[:, :1], k=None, positions=far[:2], out=far.view(F16)[:128].view(2, 1, 64)),
        lambda: rotary(q=other(q)[:, :1], k=None, out=f.view(F16)[:128].view(2, 1, 64)),
        lambda: append(q_out=qkv[:, 1:5]), lambda: append(q_out=qkv[:, 2:6]), lambda: append(q_out=qkv[:, 4:]),
        lambda: append(q_out=folded), lambda: append(k=half(p.k_pages, 4)), lambda: append(v=half(p.k_pages, 4)),
        lambda: append(k=p.k_pages[:2, :, 3]), lambda: append(q=p.v_pages[:2, :, 3]),
        lambda: append(e, k=half(e.v_scale, 4)), lambda: append(e, q_out=half(e.k_pages, 8)), lambda: append(e, q_out=half(e.k_scale, 8)),
        lambda: append(k_pages=pool[1:], v_pages=pool[:-1]),
        lambda: attend(q=q, out=q), lambda: attend(out=half(p.v_pages, 8)), lambda: attend(e, out=half(e.k_scale, 8)),
        lambda: attend(e, out=half(e.v_pages, 8)),
    ]
    keep = [x.clone() for x in (qkv, p.k_pages.view(torch.int16), p.v_pages.view(torch.int16), e.k_scale.view(torch.int32))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")
    for x, y in zip(keep, (qkv, p.k_pages.view(torch.int16), p.v_pages.view(torch.int16), e.k_scale.view(torch.int32))):
        assert torch.equal(x, y)                                 # nothing ran
    # what shares no memory still runs: beside each other in packed rows, in one store
    want = rotary()
    x = other(qkv)
    got = fkv.apply_rotary(x[:, :4], x[:, 4:6], pos, f, out=(x[:, :4], x[:, 4:6]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(x[:, 6:], v)
    got = rotary(out=(store[:512].view(2, 4, 64), store[512:768].view(2, 2, 64)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    append(k_pages=pool[:4], v_pages=pool[4:8], table=torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda"),
           lens=torch.tensor([20, 30], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool[5, :, 3], v[0]) and torch.equal(pool[7, :, 13], v[1])
    assert attend(out=store[:512].view(2, 4, 64)).data_ptr() == store.data_ptr()


# ---- inputs written just before -----------------------------------------------------------------

def test_frequencies_written_by_the_kernel_before():
    """Small calls start beside their predecessor; what it writes is waited for."""
    p = R.Pages(9, [20, 30], 2, 64, 16, F16, False)
    q, k, pos = _rand(2, 4, 64, dtype=F16), _rand(2, 2, 64, dtype=F16), torch.arange(2, device="cuda") + 5
    base = [fkv.rotary_frequencies(64, 10000.0 + 50 * i)[0] for i in range(40)]
    want = [fkv.apply_rotary(q, None, pos, b) for b in base]
    f = torch.zeros_like(base[0])
    got = []
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for b in base:
            f.copy_(b)
            got.append(fkv.apply_rotary(q, None, pos, f))
            f.mul_(0)
            f.add_(b)
            got.append(fkv.paged_append(k, k, q=q, inv_freq=f, **dict(p.kw, lens=(pos + 1).int(), table=p.table)))
    for _ in range(5):
        g.replay()
        for i, x in enumerate(got):
            assert torch.equal(x, want[i // 2]), i


def test_cache_under_a_default_device():
    """torch.device as a context changes where host tensors are made, not the cache's own."""
    f = fkv.rotary_frequencies(64, scaling="yarn", factor=4.0, original_len=512)
    with torch.device("cuda"):
        g = fkv.rotary_frequencies(64, scaling="yarn", factor=4.0, original_len=512)
        assert torch.equal(f[0], g[0]) and f[1] == g[1]
        c = PagedKVCache(1, 8, 2, 64, page=8, max_seqs=2, max_len=32, inv_freq=f[0])
        c.extend([9, 3])
        k = _rand(12, 2, 64, dtype=F16)
        c.append(0, k, k, k)
        c.extend([1, 1])
        c.attend(0, c.append(0, k[:2], k[:2], k[:2]))
        assert torch.equal(c.read(0, 0)[1][0, :, :9], k[:9].transpose(0, 1))
        c.release(0)
        c.check()


# ---- gradients ----------------------------------------------------------------------------------

def test_frequencies_and_tangents_are_refused():
    p = R.Pages(7, [20, 30], 2, 64, 16, F16, False)
    q, k = _rand(2, 4, 64, dtype=F16), _rand(2, 2, 64, dtype=F16)
    pos, f = torch.arange(2, device="cuda"), fkv.rotary_frequencies(64)[0]
    g = f.clone().requires_grad_()
    rotary = lambda **kw: fkv.apply_rotary(**dict(dict(q=q, k=k, positions=pos, inv_freq=f), **kw))
    append = lambda **kw: fkv.paged_append(**dict(dict(k=k, v=k.clone(), q=q, inv_freq=f, **p.kw), **kw))
    attend = lambda **kw: fkv.paged_attend(**dict(dict(q=q, **p.kw), **kw))
    for call in (lambda: rotary(inv_freq=g), lambda: append(inv_freq=g)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        dual = lambda x: ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: rotary(q=dual(q)), lambda: rotary(k=dual(k)), lambda: rotary(inv_freq=dual(f)),
                     lambda: rotary(out=(dual(q.clone()), k.clone())), lambda: append(k=dual(k)), lambda: append(v=dual(k)),
                     lambda: append(q=dual(q)), lambda: append(inv_freq=dual(f)), lambda: attend(q=dual(q)),
                     lambda: attend(k_pages=dual(p.k_pages)), lambda: attend(out=dual(torch.empty_like(q)))):
            with pytest.raises(ValueError, match="gradient"):
                call()
        rotary(), append(), attend()
