"""The paged cache on the GPU: writing, reading back and attending, against
64-bit forms.  Every place of the pages that belongs to no token holds NaN, so
a read of one shows."""

import numpy as np
import pytest
import torch

import foveated_kv_b200 as fkv
from foveated_kv_b200 import FkvNativeError, PagedKVCache, TierConfig, compress_layer
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
LENS = [0, 1, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1000]


def _rand(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _attend(p, Hq, window=0, seed=9, **kw):
    B, D = len(p.lens_host), p.k_pages.shape[3]
    q = _rand(B, Hq, D, dtype=p.dtype, seed=seed) * 1.5
    out, lse = fkv.paged_attend(q, window=window, return_lse=True, **p.kw, **kw)
    R.check_attend(p, q, out, lse, window, kw.get("scale"))
    return q, out, lse


# ---- attention --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 7, 12])
def test_attend_ragged(D, G, dtype, fp8):
    p = R.Pages(1, LENS, 2, D, 16, dtype, fp8)
    _attend(p, 2 * G)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, True)])
def test_attend_page_sizes(page, dtype, fp8):
    p = R.Pages(2, [page * 3, page * 3 + 1, page - 1, 1, 333], 3, 128, page, dtype, fp8)
    _attend(p, 12)


@pytest.mark.parametrize("window", [1, 5, 16, 17, 64, 100, 5000])
@pytest.mark.parametrize("D,fp8", [(64, True), (128, False), (128, True)])
def test_attend_window(window, D, fp8):
    p = R.Pages(3, LENS + [4097], 2, D, 8, F16, fp8)
    _attend(p, 8, window=window)


@pytest.mark.parametrize("Hq,Hk", [(8, 8), (16, 1), (17, 1), (33, 1), (40, 2), (20, 4)])
@pytest.mark.parametrize("D,fp8", [(64, False), (128, True), (256, False)])
def test_attend_head_groups(Hq, Hk, D, fp8):
    p = R.Pages(4, [500, 3, 0, 77], Hk, D, 32, BF16, fp8)
    _attend(p, Hq)


@pytest.mark.parametrize("B,Hk,D,n,dtype,fp8", [
    (1, 1, 128, 20000, F16, False),      # one stream over the whole device
    (1, 2, 64, 70001, BF16, True),
    (200, 4, 64, 300, F16, False),       # a CTA per stream, more streams than CTAs at once
    (120, 4, 64, 1500, F16, False),      # more streams than CTAs, cut into units
    (120, 4, 128, 1500, BF16, True),
    (64, 8, 64, 3100, F16, True),        # two waves of CTAs
    (48, 16, 64, 8000, BF16, True),      # three
])
def test_attend_work_splits(B, Hk, D, n, dtype, fp8):
    lens = [n - (i * 37) % (n // 3) for i in range(B)]
    p = R.Pages(5, lens, Hk, D, 64, dtype, fp8)
    q, out, lse = _attend(p, 4 * Hk)
    again = fkv.paged_attend(q, **p.kw)
    assert torch.equal(again, out)                               # bit for bit


def test_attend_long_offsets():
    """Rows beyond 2^31 bytes and elements into the pages."""
    page, Hk, D = 64, 8, 128
    P = (1 << 31) // (Hk * page * D) + 40                        # over 2^31 elements, 4 GB a side
    k = torch.zeros(P, Hk, page, D, dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    ids = torch.tensor([P - 1, P - 3, 5, P // 2 + 9], dtype=torch.int32)
    p = R.Pages(6, [4 * page - 5], Hk, D, page, F16, False)
    k[ids.long().cuda()] = p.k_pages[p.table[0, :4].long()]
    v[ids.long().cuda()] = p.v_pages[p.table[0, :4].long()]
    q = _rand(1, 32, D, dtype=F16)
    got, lse = fkv.paged_attend(q, k, v, ids[None].cuda(), p.lens, return_lse=True)
    R.check_attend(p, q, got, lse)
    new = _rand(1, Hk, D, dtype=F16, seed=3)
    fkv.paged_append(new, new, k, v, ids[None].cuda(), torch.tensor([page], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[P - 1, :, page - 1], new[0])


def test_attend_scale_out_and_query_forms():
    p = R.Pages(7, [40, 900], 2, 128, 16, F16, False)
    q, out, lse = _attend(p, 4, scale=0.3)
    dst = torch.full_like(q, float("nan"))
    assert fkv.paged_attend(q, scale=0.3, out=dst, **p.kw) is dst and torch.equal(dst, out)
    q4 = q[:, :, None]
    assert torch.equal(fkv.paged_attend(q4, scale=0.3, **p.kw), out[:, :, None])
    strided = torch.stack([q, q], 2)[:, :, 0]
    odd = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)
    assert torch.equal(fkv.paged_attend(strided, scale=0.3, **p.kw), out)
    assert torch.equal(fkv.paged_attend(odd, scale=0.3, **p.kw), out)
    wide = torch.full((2, p.table.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    wide[:, :p.table.shape[1]] = p.table
    kw = dict(p.kw, table=wide[:, :p.table.shape[1]])            # rows of a larger table
    assert torch.equal(fkv.paged_attend(q, scale=0.3, **kw), out)


def test_attend_large_and_small_values():
    """Scores far apart, rows of very different scales, a large common offset."""
    p = R.Pages(8, [700, 64], 2, 128, 16, F16, False, k_scale=30.0)
    _attend(p, 8)                                                # near one-hot
    for mult in (1e-4, 1e-2, 50.0):
        p = R.Pages(9, [700, 64], 2, 128, 16, BF16, True)
        p.v_scale[::2] *= mult
        p.v_scale[1::3] *= mult * mult
        _attend(p, 8)
    p = R.Pages(9, [300], 1, 64, 16, BF16, True)
    p.k_scale *= 1e-30
    q = _rand(1, 2, 64, dtype=BF16, seed=1) * 1e30               # beyond the range of f16
    out, lse = fkv.paged_attend(q, return_lse=True, **p.kw)
    R.check_attend(p, q, out, lse)
    p.k_scale *= 1e30
    q = _rand(1, 2, 64, dtype=BF16, seed=1) * 1e-30
    out, lse = fkv.paged_attend(q, return_lse=True, **p.kw)
    R.check_attend(p, q, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
def test_attend_infinities_and_nan(fp8):
    p = R.Pages(10, [100, 100, 100, 5], 1, 64, 16, F16, fp8)
    q = _rand(4, 2, 64, dtype=F16).abs() + 0.1
    ids = p.table[:, 0].long()
    if fp8:
        p.k_scale[ids[0], 0, 3] = float("nan")
        p.v_scale[ids[1], 0, 4] = float("nan")
        p.k_pages.view(torch.uint8)[ids[2], 0, 5, 0] = 0x7F
    else:
        p.k_pages[ids[0], 0, 3] = float("inf")                   # +inf score: NaN
        p.v_pages[ids[1], 0, 4, 0] = float("inf")                # inf in one element of the output
        p.k_pages[ids[2], 0, 5] = float("-inf")                  # -inf score: no weight
        p.k_pages[ids[3], 0, :5] = float("-inf")                 # no weight anywhere: NaN
    out, lse = fkv.paged_attend(q, return_lse=True, **p.kw)
    ref, rlse, _, _ = R.attend(q, p.sequences("k"), p.sequences("v"), p.lens_host)
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(torch.isinf(out), torch.isinf(ref))
    assert torch.equal(torch.isnan(lse), torch.isnan(rlse)) and torch.equal(torch.isinf(lse), torch.isinf(rlse))
    fin = torch.isfinite(ref)
    assert fin[3 if fp8 else 2].all() and (out[fin].double() - ref[fin]).abs().max() < 2e-3


def test_attend_scales_of_zero():
    p = R.Pages(11, [50], 1, 128, 16, F16, True)
    p.v_scale.zero_()
    out, lse = fkv.paged_attend(_rand(1, 2, 128, dtype=F16), return_lse=True, **p.kw)
    assert (out == 0).all() and torch.isfinite(lse).all()


def test_attend_nothing_to_do():
    p = R.Pages(12, [0, 0, 0], 2, 128, 16, F16, False)
    out, lse = fkv.paged_attend(torch.full((3, 4, 128), 7.0, dtype=F16, device="cuda"), return_lse=True, **p.kw)
    assert (out == 0).all() and (lse == float("-inf")).all()
    kw = dict(p.kw, table=p.table[:0], lens=p.lens[:0])
    assert fkv.paged_attend(torch.empty(0, 4, 128, dtype=F16, device="cuda"), **kw).shape == (0, 4, 128)
    kw = dict(p.kw, table=p.table[:, :0])                        # a table of no pages
    assert (fkv.paged_attend(torch.ones(3, 4, 128, dtype=F16, device="cuda"), **kw) == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_a_pool_of_no_pages(fp8):
    p = R.Pages(14, [0, 0], 2, 64, 16, F16, fp8, spare=0)
    assert p.k_pages.shape[0] == 0
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k = _rand(2, 4, 64, dtype=F16), _rand(2, 2, 64, dtype=F16)
    assert (fkv.paged_attend(q, status=st, **p.kw) == 0).all() and st.item() == 0
    kw = dict(p.kw, lens=torch.tensor([20, 3], dtype=torch.int32, device="cuda"), table=p.table.abs())
    fkv.paged_attend(q, status=st, **kw)
    assert st.item() == 1
    st.zero_()
    fkv.paged_append(k, k, status=st, **kw)
    assert st.item() == 1
    dense = fkv.paged_read(max_len=20, **kw)
    assert (dense[0] == 0).all() and (dense[1] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_attend_bad_pages_and_lengths(fp8):
    """A table entry that is no page leaves its tokens out; a length beyond the
    table is cut; the status word says so."""
    p = R.Pages(13, [100, 64, 90], 2, 128, 16, F16, fp8, width_extra=0)
    q = _rand(3, 4, 128, dtype=F16)
    want = fkv.paged_attend(q, **p.kw)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(fkv.paged_attend(q, status=st, **p.kw), want) and st.item() == 0
    for bad in (-1, p.k_pages.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = p.table.clone()
        t[0, 2] = bad
        out = fkv.paged_attend(q, status=st, **dict(p.kw, table=t))
        assert st.item() == 1 and torch.equal(out[1:], want[1:])
        st.zero_()
        ks, vs = p.sequences("k"), p.sequences("v")
        left = [torch.cat([x[:, :32], x[:, 48:]], 1) for x in (ks[0], vs[0])]
        ref = R.attend(q[:1], [left[0]], [left[1]], [84])[0]
        assert (out[:1].double() - ref).abs().max() < 2e-3
    far = torch.tensor([10 ** 9, 64, 90], dtype=torch.int32, device="cuda")
    full = dict(p.kw, lens=torch.tensor([112, 64, 90], dtype=torch.int32, device="cuda"))
    k2, v2 = p.k_pages.clone(), p.v_pages.clone()
    if fp8:
        full["k_scale"], full["v_scale"] = full["k_scale"].nan_to_num(0.5), full["v_scale"].nan_to_num(0.5)
        k2.view(torch.uint8)[k2.isnan()] = 0x30
        v2.view(torch.uint8)[v2.isnan()] = 0x30
    else:
        k2, v2 = k2.nan_to_num(0.5), v2.nan_to_num(0.5)
    full.update(k_pages=k2, v_pages=v2)
    a = fkv.paged_attend(q, **full)
    b = fkv.paged_attend(q, status=st, **dict(full, lens=far))
    assert torch.equal(a, b) and st.item() == 2
    st.zero_()
    neg = fkv.paged_attend(q, status=st, **dict(full, lens=torch.tensor([-5, 64, 90], dtype=torch.int32, device="cuda")))
    assert (neg[0] == 0).all() and torch.equal(neg[1:], a[1:])


def test_attend_two_streams_at_once_and_graphs():
    """Calls share no state: two streams at once, two captured graphs replayed
    at once, and a replay after the sequences grew."""
    ps = [R.Pages(20 + i, [5000 + i, 3000, 12], 4, 128, 16, F16, bool(i)) for i in range(2)]
    qs = [_rand(3, 16, 128, dtype=F16, seed=i) for i in range(2)]
    want = [fkv.paged_attend(q, **p.kw) for q, p in zip(qs, ps)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fkv.paged_attend(qs[i], **ps[i].kw))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([fkv.paged_attend(qs[i], **ps[i].kw) for _ in range(3)])
        graphs.append(g)
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in outs[i])
    for n in (1, 4999, 0, 700):                                  # lengths are read on the device
        ps[0].lens[0] = n
        ps[0].lens_host[0] = n
        graphs[0].replay()
        R.check_attend(ps[0], qs[0], outs[0][2])


# ---- writing ------------------------------------------------------------------------------------

def _fresh(lens, Hk, D, page, dtype, fp8, seed=30):
    """A cache whose pages hold known bytes everywhere."""
    p = R.Pages(seed, lens, Hk, D, page, dtype, fp8)
    for x in (p.k_pages, p.v_pages):
        raw = x.view(torch.uint8)
        raw.copy_(torch.randint(0, 120, raw.shape, dtype=torch.uint8, device="cuda"))
    if fp8:
        p.k_scale.fill_(0.25)
        p.v_scale.fill_(0.5)
    return p


def _places(p, new):
    """(page, row, sequence, position) of each new token, packed order."""
    t = p.table.cpu()
    out = []
    for b, (n, m) in enumerate(zip(p.lens_host, new)):
        out += [(int(t[b, x // p.page]), x % p.page, b, x) for x in range(n - m, n)]
    return out


def _check_append(p, new, k, v, q, kw, run):
    before = [x.view(torch.uint8).clone() for x in (p.k_pages, p.v_pages)]
    scales = [None if s is None else s.clone() for s in (p.k_scale, p.v_scale)]
    got = run()
    at = _places(p, new)
    T = len(at)
    pid = torch.tensor([a[0] for a in at], device="cuda", dtype=torch.long)
    row = torch.tensor([a[1] for a in at], device="cuda", dtype=torch.long)
    pos = torch.tensor([a[3] for a in at], device="cuda", dtype=torch.long)
    f = kw.get("inv_freq")
    il, amp = kw.get("interleaved", False), kw.get("amplitude", 1.0)
    for name, x, pages, scale, old, olds in (("k", k, p.k_pages, p.k_scale, before[0], scales[0]),
                                             ("v", v, p.v_pages, p.v_scale, before[1], scales[1])):
        x = x[:T]
        there = pages.view(torch.uint8)[pid, :, row].view(pages.dtype)
        if name == "k" and f is not None:
            ref = R.rotate(x.double(), pos, f, il, amp)
            slack = R.rotate_slack(x.double(), f, il, amp)
            if p.fp8:
                s = scale[pid, :, row].double()
                most = ref.abs().amax(-1)
                # the scale follows the 32-bit maximum, rounded twice
                assert ((s * 448 - most).abs() <= slack.amax(-1) + most * 2.0 ** -22).all()
                err = (there.double() * s[..., None] - ref).abs()
                assert (err <= 2.0 ** -4 * (ref.abs() + slack) + 2.0 ** -10 * s[..., None] + slack).all()
            else:
                err = (there.double() - ref).abs()
                assert (err <= R.HALF_STEP[p.dtype] * (ref.abs() + slack) + slack + R.SUBNORMAL[p.dtype]).all()
        elif p.fp8:
            codes, s = R.e4m3_rows(x)
            assert torch.equal(there.view(torch.uint8).cpu(), codes)
            assert torch.equal(scale[pid, :, row].cpu().view(torch.int32), s.view(torch.int32))
        else:
            assert torch.equal(there.view(torch.int16), x.contiguous().view(torch.int16))
        mask = torch.ones(pages.shape[0], p.page, dtype=torch.bool, device="cuda")
        mask[pid, row] = False                                   # every other place is as it was
        m = mask[:, None].expand(-1, pages.shape[1], -1)
        assert torch.equal(pages.view(torch.uint8)[m], old[m])
        if p.fp8:
            assert torch.equal(scale[m], olds[m])
    if q is not None:
        ref = R.rotate(q[:T].double(), pos, f, il, amp)
        slack = R.rotate_slack(q[:T].double(), f, il, amp)
        assert ((got[:T].double() - ref).abs() <= R.HALF_STEP[p.dtype] * (ref.abs() + slack) + slack
                + R.SUBNORMAL[p.dtype]).all()
        assert (got[T:] == 0).all()                              # padding
    return got


@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("D,page", [(64, 8), (128, 16), (256, 64)])
@pytest.mark.parametrize("turn", ["none", "half", "interleaved", "part"])
def test_append_packed(turn, D, page, dtype, fp8):
    lens, new, Hk, Hq = [5, 0, 200, 33, 64, 9], [5, 0, 150, 1, 0, 3], 2, 6
    p = _fresh(lens, Hk, D, page, dtype, fp8)
    T = sum(new) + 4                                             # 4 rows of padding
    k, v, q = (_rand(T, h, D, dtype=dtype, seed=s) for h, s in ((Hk, 1), (Hk, 2), (Hq, 3)))
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    kw = {}
    if turn != "none":
        rot = 24 if turn == "part" else D
        kw = dict(inv_freq=fkv.rotary_frequencies(rot)[0], interleaved=turn == "interleaved", amplitude=1.5)
    else:
        q = None
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_append(p, new, k, v, q, kw, lambda: fkv.paged_append(k, v, cu_new=cu, q=q, status=st, **kw, **p.kw))
    assert st.item() == 0


@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("fp8", [False, True])
def test_append_uniform(n, fp8):
    lens, Hk, Hq, D = [40, 100, 64, 1000], 3, 6, 128
    p = _fresh(lens, Hk, D, 16, F16, fp8)
    k, v, q = (_rand(4, h, n, D, dtype=F16, seed=s) for h, s in ((Hk, 1), (Hk, 2), (Hq, 3)))
    flat = lambda x: x.transpose(1, 2).reshape(-1, x.shape[1], D)
    kw = dict(inv_freq=fkv.rotary_frequencies(128)[0])
    _check_append(p, [n] * 4, flat(k), flat(v), flat(q), kw,
                  lambda: flat(fkv.paged_append(k, v, q=q, **kw, **p.kw)))
    if n == 1:                                                   # (B, heads, D): the same step
        p2 = _fresh(lens, Hk, D, 16, F16, fp8)
        k3, v3, q3 = (x[:, :, 0] for x in (k, v, q))
        _check_append(p2, [1] * 4, k3, v3, q3, kw, lambda: fkv.paged_append(k3, v3, q=q3, **kw, **p2.kw))


def test_append_empty_slots_views_and_in_place():
    p = _fresh([0, 17, 0, 5], 2, 128, 16, BF16, False)
    qkv = _rand(4, 10, 128, dtype=BF16)                          # packed rows: 6 q, 2 k, 2 v
    keep = qkv.clone()
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    f = fkv.rotary_frequencies(128)[0]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    live = [1, 3]
    cmp = _fresh([17, 5], 2, 128, 16, BF16, False)
    want = fkv.paged_append(keep[live, 6:8], keep[live, 8:], q=keep[live, :6], inv_freq=f, **cmp.kw)
    got = fkv.paged_append(k, v, q=q, q_out=q, inv_freq=f, status=st, **p.kw)
    assert got is q and torch.equal(q[live], want) and (q[[0, 2]] == 0).all() and st.item() == 0
    assert torch.equal(qkv[:, 6:], keep[:, 6:])
    seq = [x for x in p.sequences("k") if x.shape[1]]
    for a, b in zip(seq, cmp.sequences("k")):
        assert torch.equal(a[:, -1], b[:, -1])
    odd = torch.cat([k.flatten()[:1], k.flatten()])[1:].view(k.shape)      # 2 bytes off
    p2 = _fresh([0, 17, 0, 5], 2, 128, 16, BF16, False)
    fkv.paged_append(odd, v, inv_freq=f, **p2.kw)
    assert torch.equal(p2.table, p.table) and torch.equal(p2.sequences("k")[1][:, -1], p.sequences("k")[1][:, -1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_special_rows(dtype):
    """Zero rows, one large element, the type's extremes, infinities and NaN."""
    D, rows = 128, 9
    k = torch.zeros(rows, 1, D, dtype=dtype, device="cuda")
    big = torch.finfo(dtype).max
    k[1, 0, 5] = big
    k[2] = -big
    k[3, 0, :2] = torch.tensor([torch.finfo(dtype).tiny, 1.0], dtype=dtype)
    k[4, 0, 3] = torch.finfo(dtype).smallest_normal / 8          # subnormal
    k[5] = _rand(1, D, dtype=dtype)
    k[5, 0, 7] = float("inf")
    k[6] = _rand(1, D, dtype=dtype)
    k[6, 0, 100] = float("nan")
    k[7] = torch.linspace(-448, 448, D).to(dtype)                # scale 1: every rounding case
    k[8] = (torch.arange(D) * 2.0 ** -9 - 0.1).to(dtype)
    p = _fresh([rows], 1, D, 16, dtype, True)
    fkv.paged_append(k.transpose(0, 1)[None], k.transpose(0, 1)[None], **p.kw)
    codes, scale = R.e4m3_rows(k)
    back, _ = fkv.paged_read(max_len=rows, dtype=dtype, **p.kw)
    ids = p.table[0, 0].long()
    assert torch.equal(p.k_pages.view(torch.uint8)[ids, 0, :rows].cpu()[[0, 1, 2, 3, 4, 7, 8]],
                       codes[:, 0][[0, 1, 2, 3, 4, 7, 8]])
    assert torch.equal(p.k_scale[ids, 0, :rows].cpu()[[0, 1, 2, 3, 4, 7, 8]], scale[:, 0][[0, 1, 2, 3, 4, 7, 8]])
    assert torch.isnan(back[0, 0, 5]).all() and torch.isnan(back[0, 0, 6]).all()
    fine = [0, 1, 2, 3, 4, 7, 8]
    x = k[fine, 0].double()
    s = scale[fine, 0].double().cuda()[:, None]
    assert torch.isfinite(back[0, 0, fine]).all()
    err = (back[0, 0, fine].double() - x).abs()
    assert (err <= (2.0 ** -4 + 2 * R.HALF_STEP[dtype]) * x.abs() + 2.0 ** -10 * s + R.SUBNORMAL[dtype]).all()


def test_append_out_of_place_is_reported_not_written():
    """Positions outside the table and entries that are no pages: nothing is
    written, the status word says which."""
    p = _fresh([40, 30, 20], 2, 64, 16, F16, True)
    k = _rand(3, 2, 64, dtype=F16)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    raw = lambda: [x.view(torch.uint8).clone() for x in (p.k_pages, p.v_pages, p.k_scale, p.v_scale)]
    before = raw()
    for lens, table, bits in (([10 ** 9, -3, 2 ** 31 - 1], p.table, 2),
                              ([40, 30, 20], torch.full_like(p.table, -1), 1),
                              ([40, 30, 20], torch.full_like(p.table, p.k_pages.shape[0]), 1),
                              ([10 ** 9, 30, 20], torch.full_like(p.table, 2 ** 31 - 1), 3)):
        kw = dict(p.kw, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        q = fkv.paged_append(k, k, q=k, inv_freq=fkv.rotary_frequencies(64)[0], status=st, **kw)
        assert st.item() == bits and (q == 0).all()
        assert all(torch.equal(a, b) for a, b in zip(before, raw()))
        st.zero_()
    # more new tokens than the length counts
    fkv.paged_append(_rand(1, 2, 8, 64, dtype=F16), _rand(1, 2, 8, 64, dtype=F16), status=st,
                     **dict(p.kw, table=p.table[:1], lens=torch.tensor([3], dtype=torch.int32, device="cuda")))
    assert st.item() == 2


# ---- reading back -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fp8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("D,page,lens,max_len", [(64, 8, [1, 0, 65, 129], 131), (128, 64, [300], 300),
                                                 (256, 16, [17, 40], 20), (128, 16, [5], 1)])
def test_read(D, page, lens, max_len, dtype, fp8):
    p = R.Pages(40, lens, 3, D, page, dtype, fp8)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = fkv.paged_read(max_len=max_len, dtype=dtype, status=st, **p.kw)
    assert k.shape == v.shape == (len(lens), 3, max_len, D) and k.dtype == v.dtype == dtype and st.item() == 0
    for got, seqs in ((k, p.sequences("k")), (v, p.sequences("v"))):
        for b, n in enumerate(lens):
            n = min(n, max_len)
            ref = seqs[b][:, :n]
            # a row's product is taken in 32 bits and rounded to 16
            ref = ref.float().to(dtype) if fp8 else ref.to(dtype)
            assert torch.equal(got[b, :, :n], ref) and (got[b, :, n:] == 0).all()


def test_read_bad_pages():
    p = R.Pages(41, [40, 20], 2, 128, 16, F16, False, width_extra=0)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, _ = fkv.paged_read(max_len=40, **p.kw)
    t = p.table.clone()
    t[0, 1] = p.k_pages.shape[0]
    got, _ = fkv.paged_read(max_len=40, status=st, **dict(p.kw, table=t))
    assert st.item() == 1 and (got[0, :, 16:32] == 0).all()
    assert torch.equal(got[0, :, :16], want[0, :, :16]) and torch.equal(got[1], want[1])
    st.zero_()
    fkv.paged_read(max_len=64, status=st, **dict(p.kw, lens=torch.tensor([40, 10 ** 6], dtype=torch.int32, device="cuda"),
                                                 table=p.table.clamp(min=0)))
    assert st.item() == 2


# ---- the three together -------------------------------------------------------------------------

@pytest.mark.parametrize("fmt,dtype", [("16", F16), ("fp8", BF16)])
def test_serving_run(fmt, dtype):
    """Prompts of several lengths, decode steps, a sequence that leaves, one
    that takes its pages, and a hand-over to the tiered cache."""
    L, Hk, Hq, D, page = 2, 2, 8, 128, 16
    f, amp = fkv.rotary_frequencies(64, scaling="yarn", factor=4.0, original_len=128)
    c = PagedKVCache(L, 60, Hk, D, page=page, max_seqs=3, max_len=400, fmt=fmt, dtype=dtype, inv_freq=f, amplitude=amp)
    ks, vs = ([[torch.zeros(0, Hk, D, device="cuda", dtype=torch.float64) for _ in range(3)] for _ in range(L)]
              for _ in range(2))
    seed = [100]

    def step(counts):
        had = c.lengths
        c.extend(counts)
        packed = max(counts) > 1
        rows = sum(counts) if packed else 3
        outs = []
        for i in range(L):
            seed[0] += 1
            k, v, q = (_rand(rows, h, D, dtype=dtype, seed=seed[0] * 10 + j) for j, h in enumerate((Hk, Hk, Hq)))
            qr = c.append(i, k, v, q)
            at = 0
            for s, m in enumerate(counts):
                src = slice(at, at + m) if packed else slice(s, s + m)
                at += m
                pos = torch.arange(had[s], had[s] + m, device="cuda")
                kr = R.rotate(k[src].double(), pos, f, False, amp)
                ks[i][s] = torch.cat([ks[i][s], kr])
                vs[i][s] = torch.cat([vs[i][s], v[src].double()])
                if m:
                    ref = R.rotate(q[src].double(), pos, f, False, amp)
                    slack = R.rotate_slack(q[src].double(), f, False, amp)
                    assert ((qr[src].double() - ref).abs() <= R.HALF_STEP[dtype] * (ref.abs() + slack) + slack).all()
            if not packed:
                out = c.attend(i, qr)
                n = c.lengths
                ref, _, mag, _ = R.attend(qr, [x.transpose(0, 1) for x in ks[i]], [x.transpose(0, 1) for x in vs[i]], n)
                # stored rows are off by half a step of their type, keys inside the exponent:
                # |dx| <= step * sum |q||k| / sqrt(D) <= 0.5 (fp8), 0.04 (bf16), with D = 128 here
                err = (out.double() - ref).norm() / ref.norm()
                assert err < (0.1 if fmt == "fp8" else 0.01)
                outs.append(out)
        c.check()
        return outs

    step([37, 1, 130])
    step([1, 1, 1])
    step([0, 1, 1])
    free = c.free_pages
    c.release(1)
    for i in range(L):
        ks[i][1], vs[i][1] = ks[i][1][:0], vs[i][1][:0]
    assert c.free_pages == free + 1 and c.lengths == [38, 0, 132]
    step([1, 0, 1])                                              # an empty slot in the batch
    step([0, 60, 2])                                             # a new sequence in it, and a chunk
    for _ in range(3):
        step([1, 1, 1])
    want = [fkv.paged_read(table=c.table, lens=c.lens, max_len=200, dtype=dtype, **c.layers[i])[0] for i in range(L)]
    for i in range(L):
        k, v = c.read(i, 2)
        n = c.lengths[2]
        assert k.shape == (1, Hk, n, D) and torch.equal(k[0], want[i][2, :, :n])
        ref = ks[i][2].transpose(0, 1)
        tol = 2.0 ** -4 if fmt == "fp8" else 2.0 ** -11
        # the row's largest element is exact to the step; the smallest steps are 2^-10 of 1/448 of it
        assert ((k[0].double() - ref).abs() <= (tol + 2.0 ** -8) * ref.abs() + ref.abs().amax(-1, keepdim=True) * 2.0 ** -17
                ).all()
    cfg = TierConfig(window_size=16)
    fov = c.compress(2, cfg)
    assert fov.seq_length == c.lengths[2] and len(fov.layers) == L
    for i, lay in enumerate(fov.layers):
        ref = compress_layer(*c.read(i, 2), cfg)
        assert torch.equal(lay.far_k, ref.far_k) and torch.equal(lay.near_v, ref.near_v)
    q = _rand(1, Hq, 1, D, dtype=F16)
    assert fov.attend(0, q).shape == (1, Hq, 1, D)


def test_decode_step_in_a_graph():
    """append + attend of all layers captured once, replayed while extend() moves the lengths."""
    L, Hk, Hq, D = 2, 2, 4, 64
    f = fkv.rotary_frequencies(64)[0]
    c, e = (PagedKVCache(L, 40, Hk, D, page=8, max_seqs=2, max_len=100, inv_freq=f) for _ in range(2))
    k, v, q = (_rand(2, h, D, dtype=F16, seed=s) for h, s in ((Hk, 1), (Hk, 2), (Hq, 3)))

    def run(cache):
        return [cache.attend(i, cache.append(i, k, v, q)) for i in range(L)]

    for x in (c, e):
        x.extend([13, 7])
        for i in range(L):
            x.append(i, *(_rand(20, Hk, D, dtype=F16, seed=50 + i + j) for j in range(2)))
        x.extend([1, 1])
    run(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run(c)
    for n in range(25):
        g.replay()
        want = run(e)
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), n
        for t, s in ((k, 1), (v, 2), (q, 3)):
            t.copy_(_rand(*t.shape, dtype=F16, seed=1000 * n + s))
        c.extend([1, 1])
        e.extend([1, 1])
    c.check()


def test_cache_limits_change_nothing():
    c = PagedKVCache(1, 4, 2, 64, page=8, max_seqs=2, max_len=24)
    c.extend([20, 5])
    table, lens = c.table.clone(), c.lens.clone()
    with pytest.raises(FkvNativeError):
        c.extend([4, 4])                                         # 5 pages of 4
    with pytest.raises(ValueError):
        c.extend([5, 0])                                         # 25 of 24 tokens
    with pytest.raises(ValueError):
        c.extend([1])
    with pytest.raises(ValueError):
        c.extend([-1, 0])
    assert c.lengths == [20, 5] and c.free_pages == 0
    assert torch.equal(c.table, table) and torch.equal(c.lens, lens)
    with pytest.raises(ValueError):
        c.append(0, _rand(24, 2, 64, dtype=F16), _rand(24, 2, 64, dtype=F16))
    c.table[0, 0] = 99
    c.attend(0, _rand(2, 2, 64, dtype=F16))
    with pytest.raises(FkvNativeError):
        c.check()
    c.check()                                                    # reported once
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 64, max_len=8).append(0, _rand(1, 2, 64, dtype=F16), _rand(1, 2, 64, dtype=F16))
    for call in (lambda: c.release(2), lambda: c.read(0, -1), lambda: c.compress(5)):
        with pytest.raises(ValueError):
            call()
    c.release(1)
    with pytest.raises(ValueError):
        c.compress(1)
    assert c.read(0, 1)[0].shape == (1, 2, 0, 64)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 96, max_len=8)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 64, max_len=8, page=24)


def test_refusals():
    p = R.Pages(50, [20, 30], 2, 64, 16, F16, False)
    e = R.Pages(50, [20, 30], 2, 64, 16, F16, True)
    q, k = _rand(2, 4, 64, dtype=F16), _rand(2, 2, 64, dtype=F16)
    f = fkv.rotary_frequencies(64)[0]
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    A, W = fkv.paged_attend, fkv.paged_append
    bad = [
        lambda: A(q.bfloat16(), **p.kw), lambda: A(q.float(), **p.kw), lambda: A(q[:1], **p.kw),
        lambda: A(q[:, :3], **p.kw), lambda: A(q[..., :32], **p.kw), lambda: A(q, window=-1, **p.kw),
        lambda: A(q, **dict(p.kw, table=p.table.long())), lambda: A(q, **dict(p.kw, lens=p.lens[:1])),
        lambda: A(q, **dict(p.kw, lens=p.lens.cpu())), lambda: A(q, **dict(p.kw, table=p.table.t().contiguous().t())),
        lambda: A(q, **dict(p.kw, table=p.table[:1].expand(2, -1))),
        lambda: A(q, **dict(p.kw, k_pages=p.k_pages.transpose(1, 2))),
        lambda: A(q, **dict(p.kw, v_pages=p.v_pages[:1])), lambda: A(q, **dict(p.kw, k_scale=e.k_scale)),
        lambda: A(q, **dict(e.kw, k_scale=None)), lambda: A(q, **dict(e.kw, v_scale=e.v_scale.half())),
        lambda: A(q, out=q[:, :2], **p.kw), lambda: A(q, out=q.bfloat16(), **p.kw),
        lambda: A(q, status=torch.zeros(2, dtype=torch.int32, device="cuda"), **p.kw),
        lambda: A(q.clone().requires_grad_(), **p.kw),
        lambda: W(k, k[:1], **p.kw), lambda: W(k[:, :1], k[:, :1], **p.kw), lambda: W(k[:1], k[:1], **p.kw),
        lambda: W(k, k, q=q, **p.kw), lambda: W(k, k, q_out=q, **p.kw), lambda: W(k, k, q=q[:1], inv_freq=f, **p.kw),
        lambda: W(k, k, cu_new=cu[:2], **p.kw), lambda: W(k, k, cu_new=cu.long(), **p.kw),
        lambda: W(k[:, :, None], k[:, :, None], cu_new=cu, **p.kw), lambda: W(k, k, inv_freq=f.float(), **p.kw),
        lambda: W(k, k, q=q, inv_freq=f, q_out=q[:, :1].expand(2, 4, 64), **p.kw),
        lambda: W(k.clone().requires_grad_(), k, **p.kw), lambda: W(k.bfloat16(), k.bfloat16(), **p.kw),
        lambda: A(q, out=q, **p.kw), lambda: W(k, k, **dict(p.kw, v_pages=p.k_pages)),
        lambda: W(k, k, **dict(e.kw, v_scale=e.k_scale)),
        lambda: W(k, k.clone(), q=k.clone(), q_out=k, inv_freq=f, **p.kw),
        lambda: fkv.paged_read(max_len=-1, **p.kw), lambda: fkv.paged_read(max_len=4, dtype=BF16, **p.kw),
        lambda: fkv.paged_read(max_len=4, dtype=torch.float32, **e.kw),
    ]
    for i, f_ in enumerate(bad):
        with pytest.raises(ValueError):
            f_()
            pytest.fail(f"case {i} was accepted")
    for D, page in ((96, 16), (64, 24), (64, 4), (64, 512)):
        kp = torch.zeros(4, 2, page, D, dtype=F16, device="cuda")
        with pytest.raises(FkvNativeError):
            A(_rand(2, 4, D, dtype=F16), kp, kp.clone(), p.table, p.lens)
    with pytest.raises(FkvNativeError):
        W(k, k, inv_freq=fkv.rotary_frequencies(128)[0], **p.kw)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device():
    p = R.Pages(60, [500, 20], 2, 128, 16, F16, False)
    q = _rand(2, 4, 128, dtype=F16)
    want = fkv.paged_attend(q, **p.kw)
    kw = {k: None if v is None else v.to("cuda:1") for k, v in p.kw.items()}
    assert torch.equal(fkv.paged_attend(q.to("cuda:1"), **kw).to("cuda:0"), want)


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured (kernels load and workspaces are made there)."""
    import os
    import subprocess
    import sys
    code = """
import torch, foveated_kv_b200 as fkv
kp, vp = (torch.randn(20, 2, 16, 128, device="cuda").bfloat16() for _ in range(2))
table = torch.arange(20, dtype=torch.int32, device="cuda").view(1, 20)
lens = torch.tensor([300], dtype=torch.int32, device="cuda")
q, k = (torch.randn(1, h, 128, device="cuda").bfloat16() for h in (8, 2))
f = fkv.rotary_frequencies(128)[0]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    qr = fkv.paged_append(k, k, kp, vp, table, lens, q=q, inv_freq=f)
    o = fkv.paged_attend(qr, kp, vp, table, lens)
    r = fkv.apply_rotary(q, None, lens - 1, f)
    d = fkv.paged_read(kp, vp, table, lens, 300)
g.replay()
torch.cuda.synchronize()
assert torch.equal(r, qr)
assert torch.equal(o, fkv.paged_attend(qr, kp, vp, table, lens))
assert torch.equal(d[1][0, :, 299], k[0])
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=root)


def test_written_tensors_beside_autograd():
    """A graph that saved a tensor written here says so in its backward pass;
    outputs that overlap the pages, or require a gradient, are refused."""
    p = R.Pages(51, [20, 30], 2, 64, 16, F16, False)
    e = R.Pages(51, [20, 30], 2, 64, 16, F16, True)
    f, pos = fkv.rotary_frequencies(64)[0], torch.arange(2, device="cuda")
    q, k = _rand(2, 4, 64, dtype=F16), _rand(2, 2, 64, dtype=F16, seed=1)
    cases = [
        (q, lambda: fkv.apply_rotary(q, None, pos, f, out=q)),
        (k, lambda: fkv.apply_rotary(q, k, pos, f, out=(q, k))),
        (q, lambda: fkv.paged_attend(q.clone(), out=q, **p.kw)),
        (q, lambda: fkv.paged_append(k, k, q=q, q_out=q, inv_freq=f, **p.kw)),
        (p.v_pages, lambda: fkv.paged_append(k, k, **p.kw)),
        (e.k_scale, lambda: fkv.paged_append(k, k, **e.kw)),
    ]
    for saved, write in cases:
        w = torch.ones((), dtype=saved.dtype, device="cuda", requires_grad=True)
        y = (w * saved).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        i = _rand(2, 4, 64, dtype=F16)
    fkv.apply_rotary(i, None, pos, f, out=i)                     # no version to count
    grad = torch.zeros(2, 4, 64, dtype=F16, device="cuda", requires_grad=True)
    rows = p.k_pages.view(-1)[:2 * 4 * 64].view(2, 4, 64)
    for write in (lambda: fkv.apply_rotary(q, None, pos, f, out=grad), lambda: fkv.paged_attend(q, out=grad, **p.kw),
                  lambda: fkv.paged_attend(q, out=rows, **p.kw),
                  lambda: fkv.paged_attend(q, **dict(p.kw, k_pages=p.k_pages.clone().requires_grad_())),
                  lambda: fkv.paged_append(k, k, q=q, q_out=rows, inv_freq=f, **p.kw)):
        with pytest.raises(ValueError):
            write()
    with torch.no_grad():
        fkv.paged_attend(q, out=grad, **p.kw)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attend_scale_of_any_sign(scale, fp8):
    _attend(R.Pages(52, [1, 40, 900], 2, 128, 16, BF16, fp8), 8, scale=scale)
