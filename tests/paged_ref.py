"""Plain 64-bit forms of rotary positions and the paged cache, for the tests.

E4M3 codes of unrotated rows follow the definition in IEEE single precision
(scale = most / 448, code = e4m3(x * (448 / most))) so they compare bit for bit.
"""

import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # relative to the value
SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}    # half the smallest step


def rotate(x, pos, inv_freq, interleaved=False, amplitude=1.0, inverse=False):
    """x (tokens, heads, D) float64, pos (tokens,), inv_freq (rot/2,) float64."""
    half = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq[None]
    c, s = torch.cos(ang)[:, None] * amplitude, torch.sin(ang)[:, None] * amplitude
    if inverse:
        s = -s
    y = x.clone()
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def rotate_slack(x, inv_freq, interleaved=False, amplitude=1.0):
    """Bound on the 32-bit rotation's error: the angle is off by under 2^-21
    (its remainder rounded to 32 bits, 2^-25 of a turn, and the 64-bit product
    at 2^30 positions) and sine and cosine by 2 units of 2^-24, times |a| + |b|;
    2^-20 covers both and the two products' roundings."""
    half = inv_freq.numel()
    y = torch.zeros_like(x)
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    t = (x[..., ia].abs() + x[..., ib].abs()) * (amplitude * 2.0 ** -20)
    y[..., ia], y[..., ib] = t, t
    return y


def e4m3_rows(x):
    """(codes uint8, scale float32) of rows x (..., D) held exactly in float32."""
    x = x.detach().float().cpu().numpy().astype(np.float32)
    with np.errstate(all="ignore"):
        most = np.abs(x).max(-1)                               # NaN if any is
        most = np.where(most < np.float32(2.0 ** -100), np.float32(2.0 ** -100), most).astype(np.float32)
        y = x * (np.float32(448.0) / most)[..., None]
        scale = most / np.float32(448.0)
    return e4m3(torch.from_numpy(y)), torch.from_numpy(scale.astype(np.float32))


def e4m3(y):
    """Nearest E4M3 code, ties to even, magnitudes over 448 to 448, NaN to 0x7F."""
    y = y.double()
    a = y.abs().clamp(max=448.0)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).clamp(-6, 8)
    step = torch.exp2(e - 3)
    n = torch.round(a / step)                                  # 0..16 steps of this binade
    up = n == 16
    e, n = torch.where(up, e + 1, e), torch.where(up, torch.full_like(n, 8.0), n)
    code = torch.where(n >= 8, (e + 7) * 8 + (n - 8), n).nan_to_num(127.0)
    code = torch.where(torch.isnan(y), torch.full_like(code, 127.0), code)
    sign = torch.signbit(y) & ~torch.isnan(y)
    return (code + 128.0 * sign).to(torch.uint8)


def dequant(codes, scale):
    """codes float8 (..., D), scale (...): the values they stand for."""
    return codes.double() * scale.double()[..., None]


def attend(q, keys, values, lens, window=0, scale=None):
    """q (B, Hq, D); keys/values: per sequence (Hk, n, D) float64.  Returns
    (out, lse, weighted mean magnitude, largest sum of |q||k|) in 64 bits."""
    B, Hq, D = q.shape
    dev = q.device
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64, device=dev)
    dot = torch.zeros(B, Hq, dtype=torch.float64, device=dev)
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        k, v = keys[b][:, lo:n], values[b][:, lo:n]
        Hk = k.shape[0]
        qb = q[b].double().reshape(Hk, Hq // Hk, D)
        x = qb @ k.transpose(-1, -2) * scale
        p = torch.softmax(x, -1)
        out[b] = (p @ v).reshape(Hq, D)
        mag[b] = (p @ v.abs()).reshape(Hq, D)
        lse[b] = torch.logsumexp(x, -1).reshape(Hq)
        dot[b] = (qb.abs() @ k.abs().transpose(-1, -2) * abs(scale)).amax(-1).reshape(Hq)
    return out, lse, mag, dot


def attend_slack(dtype, fp8, lens, dot, mag, vmax):
    """Bounds (relative to the weighted mean magnitude, and absolute) on the
    kernel's error before the output's rounding.

    A score is off by 2^-19 of the sum of |q||k| (at most 16 accumulations,
    each truncated to 2^-23 of it) and its exponential by 2^-20 more (the
    argument's rounding, ex2 to 2^-22); numerator and denominator each take
    that.  The sums over n tokens go in n / 16 + 64 additions of 2^-23.  A
    weight is held in two parts, the first cut off below it so that a positive
    remainder is left: of at most 2^-7 for bf16, whose rounding is 2^-8 of
    that, 2^-15; of at most 2^-9 for f16, rounded to 2^-11, 2^-20.  Beside
    8-bit pages it is one f16 part, 2^-11.  An f16 part below 2^-14 is off by
    up to 2^-25 instead, where the largest weight is at least 1."""
    n = max(max(lens), 1)
    bf = dtype is torch.bfloat16
    rel = 2 * (2.0 ** -19 * dot[..., None] + 2.0 ** -20) + 2 * (n / 16 + 64) * 2.0 ** -23
    rel = rel + (2.0 ** -11 if fp8 else 2.0 ** -15 if bf else 2.0 ** -20)
    return rel * mag + (n * 2.0 ** -25 * vmax if fp8 or not bf else 0.0)


class Pages:
    """A random paged cache: shuffled pages, NaN in every place that belongs to no token."""

    def __init__(self, seed, lens, Hk, D, page, dtype, fp8, spare=3, width_extra=2, fill=True, k_scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        h = torch.Generator().manual_seed(seed)
        B = len(lens)
        need = [-(-n // page) for n in lens]
        P = sum(need) + spare
        self.lens_host, self.page, self.dtype, self.fp8 = list(lens), page, dtype, fp8
        W = max(need + [0]) + width_extra
        table = torch.full((B, W), -7, dtype=torch.int32)
        ids = torch.randperm(P, generator=h).to(torch.int32)
        self.owned = torch.zeros(P, page, dtype=torch.bool)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = ids[at:at + m]
            for j in range(m):
                self.owned[int(ids[at + j]), :max(0, min(page, lens[b] - j * page))] = True
            at += m
        self.table = table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32)
        dead = ~self.owned[:, None].expand(P, Hk, page).cuda()
        nan = float("nan")
        if fp8:
            def make(f):
                c = (rn(P, Hk, page, D) * 130).clamp(-448, 448).to(torch.float8_e4m3fn)
                s = (torch.rand(P, Hk, page, generator=g, device="cuda") + 0.5) * (f / 130)
                c.view(torch.uint8)[dead] = 0x7F
                s[dead] = nan
                return c, s
            (self.k_pages, self.k_scale), (self.v_pages, self.v_scale) = make(k_scale), make(1.0)
        else:
            self.k_pages, self.v_pages = (rn(P, Hk, page, D) * k_scale).to(dtype), rn(P, Hk, page, D).to(dtype)
            self.k_pages[dead] = nan
            self.v_pages[dead] = nan
            self.k_scale = self.v_scale = None

    @property
    def kw(self):
        return dict(k_pages=self.k_pages, v_pages=self.v_pages, table=self.table, lens=self.lens,
                    k_scale=self.k_scale, v_scale=self.v_scale)

    def sequences(self, which):
        """Per sequence (Hk, n, D) float64 values."""
        pages, scale = (self.k_pages, self.k_scale) if which == "k" else (self.v_pages, self.v_scale)
        out = []
        for b, n in enumerate(self.lens_host):
            ids = self.table[b, :-(-n // self.page)].long()
            x = pages.view(torch.uint8)[ids].view(pages.dtype) if self.fp8 else pages[ids]
            x = dequant(x, scale[ids]) if self.fp8 else x.double()
            out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n])
        return out


def check_attend(p, q, got, lse=None, window=0, scale=None):
    """Holds a paged_attend result to the 64-bit form."""
    ks, vs = p.sequences("k"), p.sequences("v")
    ref, rlse, mag, dot = attend(q.reshape(q.shape[0], q.shape[1], -1), ks, vs, p.lens_host, window, scale)
    vmax = max([float(v.abs().amax()) for v in vs if v.numel()] + [0.0])
    slack = attend_slack(p.dtype, p.fp8, p.lens_host, dot, mag, vmax)
    got = got.reshape(ref.shape).double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    err = (got - ref).abs()
    tol = HALF_STEP[p.dtype] * (ref.abs() + slack) + slack + SUBNORMAL[p.dtype]
    bad = (err > tol) & ~torch.isnan(ref)
    assert not bad.any(), f"worst {float((err - tol)[bad].max()):.3g} over at {bad.nonzero()[0].tolist()}"
    if lse is not None:
        fin = torch.isfinite(rlse)
        assert torch.equal(lse[~fin].double(), rlse[~fin])
        n = max(max(p.lens_host), 1)
        lt = 2.0 ** -19 * dot + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -23 + rlse.abs() * 2.0 ** -22
        assert ((lse.double() - rlse).abs()[fin] <= lt[fin]).all()
