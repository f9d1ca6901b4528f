"""Measured cases of the paged key-value cache: rotary positions, writing and quantising tokens into
pages, reading pages back, and attention of one new token over them.

Pages are (pages, kv heads, page size, D): one page holds `page` consecutive tokens of one sequence,
`table[b, j]` names the page of tokens [j * page, (j + 1) * page) and `lens[b]` counts the tokens of
sequence b, those written by the call included.  In the 8-bit format a row (one token of one kv head)
is E4M3 codes times one 32-bit scale.

With `own` false every operator runs in its plain form (elementary torch operations in 32 bits, angles
in 64); with `own` true it runs through foveated_kv_b200.
"""

import math

import torch

own = False

_PI2 = 2.0 * math.pi
_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_F8 = torch.float8_e4m3fn
_ROW_FLOOR = 2.0 ** -100        # a row's largest magnitude counts as at least this


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def _rotary(B, Hq, Hk, S, D, rot, dtype, interleaved, scaling, pos, packed):
    return dict(op="rotary", B=B, Hq=Hq, Hk=Hk, S=S, D=D, rot=rot, dtype=dtype, interleaved=interleaved,
                scaling=scaling, pos=pos, packed=packed)


def _append(B, Hq, Hk, D, page, dtype, fp8, len_lo, len_hi, new_lo, new_hi, rot, interleaved, scaling):
    return dict(op="append", B=B, Hq=Hq, Hk=Hk, D=D, page=page, dtype=dtype, fp8=fp8, len_lo=len_lo,
                len_hi=len_hi, new_lo=new_lo, new_hi=new_hi, rot=rot, interleaved=interleaved, scaling=scaling)


def _read(B, Hk, D, page, dtype, fp8, len_lo, len_hi):
    return dict(op="read", B=B, Hk=Hk, D=D, page=page, dtype=dtype, fp8=fp8, len_lo=len_lo, len_hi=len_hi)


def _attend(B, Hq, Hk, D, page, dtype, fp8, len_lo, len_hi, window, lse):
    return dict(op="attend", B=B, Hq=Hq, Hk=Hk, D=D, page=page, dtype=dtype, fp8=fp8, len_lo=len_lo,
                len_hi=len_hi, window=window, lse=lse)


def listed():
    return [
        # one decode step of a batch of 64: a row of queries and keys per sequence, latency
        dict(_rotary(64, 32, 8, 1, 128, 128, "float16", False, "none", 32768, False), name="rotary_step_b64"),
        # a 16K prompt at far positions, interleaved pairs over half of each head, scaled frequencies
        dict(_rotary(1, 32, 8, 16384, 128, 64, "bfloat16", True, "yarn", 1 << 20, False), name="rotary_prompt_16k"),
        # one decode step written to the cache: the new row of each of 64 sequences, rotated, in 8 bits
        dict(_append(64, 32, 8, 128, 16, "float16", True, 64, 2048, 1, 1, 128, False, "none"), name="append_step_b64_fp8"),
        # ragged prompts and chunks of seven sequences together, rotated in part, in 8 bits
        dict(_append(7, 28, 4, 128, 32, "bfloat16", True, 700, 9001, 1, 8192, 64, True, "yarn"), name="append_ragged_fp8"),
        # a 4K prompt into 16-bit pages, as many kv heads as query heads, keys rotated before
        dict(_append(1, 32, 32, 128, 16, "float16", False, 4096, 4096, 4096, 4096, 0, False, "none"), name="append_prompt_4k"),
        # a 16K sequence handed from 8-bit pages to the tier compressor
        dict(_read(1, 8, 128, 64, "float16", True, 16384, 16384), name="read_16k_fp8"),
        # a few short ragged sequences of small heads out of 16-bit pages
        dict(_read(5, 2, 64, 8, "bfloat16", False, 1, 777), name="read_short_ragged"),
        # the smallest: one sequence of 1K tokens, 14 query heads on 2 kv heads of 64
        dict(_attend(1, 14, 2, 64, 16, "float16", False, 1000, 1000, 0, False), name="attend_1k_d64"),
        # one 16K sequence, as many kv heads as query heads
        dict(_attend(1, 32, 32, 128, 16, "float16", False, 16384, 16384, 0, False), name="attend_16k_mha"),
        # a serving batch: empty to 16K tokens, a sliding window, statistics for a later merge
        dict(_attend(33, 28, 4, 128, 32, "bfloat16", False, 0, 16384, 4096, True), name="attend_ragged_window"),
        # 64 long sequences of 8-bit pages
        dict(_attend(64, 32, 8, 128, 64, "float16", True, 16384, 32768, 0, False), name="attend_b64_32k_fp8"),
        # one sequence of a million tokens
        dict(_attend(1, 32, 8, 128, 128, "bfloat16", True, 1 << 20, 1 << 20, 0, True), name="attend_1m_fp8"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "read", "attend", "attend"])
    dtype = rng.choice(["float16", "bfloat16"])
    Hk, G = rng.choice([(8, 4), (4, 7), (2, 7), (32, 1), (1, 16), (3, 5), (8, 1), (2, 12)])
    D = rng.choice([64, 128, 128, 256])
    rot = rng.choice([D, D, D // 2, D // 4, 24])
    scaling = rng.choice(["none", "linear", "yarn"])
    inter = rng.choice([False, True])
    page = rng.choice([8, 16, 32, 64, 128])
    fp8 = rng.choice([False, True])
    if op == "rotary":
        B = _log(rng, 1, 64)
        S = _log(rng, 1, max(1, 16384 // B))
        return _rotary(B, Hk * G, Hk, S, D, rot, dtype, inter, scaling, _log(rng, S + 1, 1 << 20) + S, rng.choice([False, True]))
    if op == "append":
        B = _log(rng, 1, 64)
        new_hi = _log(rng, 1, max(1, 32768 // B))
        new_lo = rng.choice([1, new_hi])
        len_lo = new_hi + rng.choice([0, _log(rng, 1, 1000)])
        len_hi = len_lo + _log(rng, 1, max(2, 65536 // B))
        return _append(B, Hk * G, Hk, D, page, dtype, fp8, len_lo, len_hi, new_lo, new_hi, rng.choice([0, rot, rot]), inter, scaling)
    B = _log(rng, 1, 128)
    most = (3 << 28) // (B * Hk * D)             # at most 3 GB of 16-bit keys and values
    len_hi = _log(rng, 1, max(2, min(most, (1 << 20) if op == "attend" else 65536 // B)))
    len_lo = rng.choice([0, 1, len_hi, len_hi // 2])
    if op == "read":
        return _read(B, Hk, D, page, dtype, fp8, min(len_lo, len_hi), len_hi)
    window = rng.choice([0, 0, _log(rng, 1, len_hi)])
    return _attend(B, Hk * G, Hk, D, page, dtype, fp8, min(len_lo, len_hi), len_hi, window, rng.choice([False, True]))


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo, evenly."""
    return [hi] if n == 1 else [hi - (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    c = case
    if c["op"] == "rotary":
        rows = c["B"] * c["S"] * (c["Hq"] + c["Hk"])
        return {"bytes": rows * c["D"] * 4 + c["B"] * c["S"] * 8, "flops": rows * c["rot"] * 3}
    row = c["D"] * 2                             # bytes of a 16-bit row
    stored = c["D"] + 4 if c["fp8"] else row
    lens = _spread(c["len_lo"], c["len_hi"], c["B"])
    if c["op"] == "append":
        T = sum(_spread(c["new_lo"], c["new_hi"], c["B"]))
        q = 2 * c["Hq"] * row if c["rot"] else 0
        ops = 3 * c["rot"] * (c["Hq"] + c["Hk"]) + (4 * c["D"] * c["Hk"] if c["fp8"] else 0)
        return {"bytes": T * (2 * c["Hk"] * (row + stored) + q), "flops": T * ops}
    if c["op"] == "read":
        n = sum(lens)
        out = c["B"] * max(lens)                 # rows behind a sequence's end are written too, as zeros
        return {"bytes": 2 * c["Hk"] * (n * stored + out * row), "flops": 2 * c["Hk"] * n * c["D"] if c["fp8"] else 0}
    n = sum(min(x, c["window"]) if c["window"] else x for x in lens)
    return {"bytes": 2 * n * c["Hk"] * stored + 2 * c["B"] * c["Hq"] * row, "flops": 4 * n * c["Hq"] * c["D"]}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _frequencies(rot, scaling, pos):
    """Radians per position of each pair, 64 bits, and the amplitude.  "linear" stretches positions by 4;
    "yarn" stretches slow pairs by 8, keeps fast ones (over 32 turns in an eighth of the reach) and ramps."""
    base = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    f = 10000.0 ** -base
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        turns = f * (pos / 8.0) / _PI2
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / 8.0 * (1.0 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    dt = _TYPES[c["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    s = {"case": c}
    if c["op"] in ("rotary", "append") and c["rot"]:
        f, s["amplitude"] = _frequencies(c["rot"], c["scaling"], c.get("pos", c.get("len_hi", 0)))
        s["inv_freq"] = f.to(dev)
    if c["op"] == "rotary":
        B, S = c["B"], c["S"]
        start = torch.randint(0, c["pos"] - S + 1, (B, 1), generator=host)
        pos = (start + torch.arange(S)[None]).to(dev)
        if c["packed"]:                          # (tokens, heads, D), as a projection gives them
            s["q"], s["k"], s["pos"] = randn(B * S, c["Hq"], c["D"]), randn(B * S, c["Hk"], c["D"]), pos.reshape(-1)
        else:                                    # (B, heads, S, D)
            s["q"], s["k"], s["pos"] = randn(B, c["Hq"], S, c["D"]), randn(B, c["Hk"], S, c["D"]), pos
        return s

    B, Hk, D, page = c["B"], c["Hk"], c["D"], c["page"]
    order = torch.randperm(B, generator=host)
    lens = torch.tensor(_spread(c["len_lo"], c["len_hi"], B))[order]
    pages_of = (lens + page - 1) // page
    width = max(1, int(pages_of.max()))
    total = int(pages_of.sum())
    pool = total + 3                             # pages that belong to nobody
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[torch.arange(width)[None] < pages_of[:, None]] = torch.randperm(pool, generator=host)[:total].to(torch.int32)
    s["table"], s["lens"], s["max_len"] = table.to(dev), lens.to(torch.int32).to(dev), max(1, int(lens.max()))
    if c["fp8"]:
        def codes():
            x = torch.empty((pool, Hk, page, D), dtype=_F8, device=dev)
            x.copy_(randn(pool, Hk, page, D, dtype=torch.float16).mul_(140.0).clamp_(-448.0, 448.0))
            return x

        def scales():
            return (torch.rand((pool, Hk, page), generator=g, device=dev) + 0.5) / 140.0
        s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"] = codes(), codes(), scales(), scales()
    else:
        s["k_pages"], s["v_pages"] = randn(pool, Hk, page, D), randn(pool, Hk, page, D)
        s["k_scale"] = s["v_scale"] = None
    if c["op"] == "append":
        new = torch.tensor(_spread(c["new_lo"], c["new_hi"], B))[order]
        cu = torch.zeros(B + 1, dtype=torch.int64)
        cu[1:] = new.cumsum(0)
        T = int(cu[-1])
        s["cu_new"] = cu.to(torch.int32).to(dev)
        s["k"], s["v"] = randn(T, Hk, D), randn(T, Hk, D)
        s["k"] *= 1.0 + 7.0 * (torch.rand((D,), generator=g, device=dev) > 0.95).to(dt)   # a few large channels
        s["q"] = randn(T, c["Hq"], D) if c["rot"] else None
    elif c["op"] == "attend":
        s["q"] = randn(B, c["Hq"], D) * 1.5
    return s


# ---------------------------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------------------------

def _own(s):
    import foveated_kv_b200 as fkv
    c = s["case"]
    if c["op"] == "rotary":
        return fkv.apply_rotary(s["q"], s["k"], s["pos"], s["inv_freq"], interleaved=c["interleaved"],
                                amplitude=s["amplitude"])
    if c["op"] == "append":
        turn = dict(inv_freq=s["inv_freq"], interleaved=c["interleaved"], amplitude=s["amplitude"]) if c["rot"] else {}
        step = c["new_lo"] == c["new_hi"] == 1   # a decode step: one new token of each sequence
        q = fkv.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                             cu_new=None if step else s["cu_new"], k_scale=s["k_scale"], v_scale=s["v_scale"], q=s["q"], **turn)
        return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]
    if c["op"] == "read":
        return fkv.paged_read(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["max_len"], k_scale=s["k_scale"],
                              v_scale=s["v_scale"], dtype=_TYPES[c["dtype"]])
    return fkv.paged_attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], k_scale=s["k_scale"],
                            v_scale=s["v_scale"], window=c["window"], return_lse=c["lse"])


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------

def _turned(x, pos, inv_freq, amplitude, interleaved):
    """x (..., tokens, heads, D) in 32 bits, rotated by its token's position."""
    half = inv_freq.numel()
    angle = pos.to(torch.float64)[..., None] * inv_freq
    cos = (angle.cos() * amplitude).float()[..., None, :]
    sin = (angle.sin() * amplitude).float()[..., None, :]
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    c, dt = s["case"], _TYPES[s["case"]["dtype"]]

    def one(x):
        y = x.float() if c["packed"] else x.float().transpose(1, 2)
        y = _turned(y, s["pos"], s["inv_freq"], s["amplitude"], c["interleaved"]).to(dt)
        return y if c["packed"] else y.transpose(1, 2).contiguous()
    return one(s["q"]), one(s["k"])


def _places(s):
    """Sequence and position of each new token, and the page and row it goes to."""
    cu, page = s["cu_new"].long(), s["case"]["page"]
    t = torch.arange(s["k"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = s["lens"].long()[b] - cu[b + 1] + t
    return pos, s["table"].long()[b, pos // page], pos % page


def _plain_append(s):
    c, dt = s["case"], _TYPES[s["case"]["dtype"]]
    pos, pid, row = _places(s)
    k, v, q = s["k"].float(), s["v"].float(), None
    if c["rot"]:
        k = _turned(k, pos, s["inv_freq"], s["amplitude"], c["interleaved"])
        q = _turned(s["q"].float(), pos, s["inv_freq"], s["amplitude"], c["interleaved"]).to(dt)
    if c["fp8"]:
        def put(x, pages, scale):
            most = x.abs().amax(-1).clamp(min=_ROW_FLOOR)
            codes = (x * (448.0 / most)[..., None]).clamp(-448.0, 448.0).to(_F8)
            pages.view(torch.uint8)[pid, :, row] = codes.view(torch.uint8)
            scale[pid, :, row] = most / 448.0
        put(k, s["k_pages"], s["k_scale"])
        put(v, s["v_pages"], s["v_scale"])
    else:
        s["k_pages"][pid, :, row] = k.to(dt)
        s["v_pages"][pid, :, row] = v.to(dt)
    return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]


def _gathered(pages, scale, table, n):
    """(B, kv heads, n, D) in 32 bits: the first n places of each sequence."""
    pid = table.long().clamp(min=0)
    B, W = pid.shape
    _, H, page, D = pages.shape
    x = pages.view(torch.uint8)[pid].view(_F8) if scale is not None else pages[pid]
    x = x.float()
    if scale is not None:
        x = x * scale[pid][..., None]
    return x.transpose(1, 2).reshape(B, H, W * page, D)[:, :, :n]


def _plain_read(s):
    n, dt = s["max_len"], _TYPES[s["case"]["dtype"]]
    inside = (torch.arange(n, device=s["lens"].device)[None] < s["lens"][:, None])[:, None, :, None]

    def one(pages, scale):
        x = _gathered(pages, scale, s["table"], n)
        return torch.where(inside, x, torch.zeros_like(x)).to(dt)
    return one(s["k_pages"], s["k_scale"]), one(s["v_pages"], s["v_scale"])


def _plain_attend(s):
    c, dt = s["case"], _TYPES[s["case"]["dtype"]]
    B, Hq, Hk, D, n = c["B"], c["Hq"], c["Hk"], c["D"], s["max_len"]
    at = torch.arange(n, device=s["lens"].device)[None]
    lens = s["lens"][:, None]
    inside = at < lens
    if c["window"]:
        inside = inside & (at >= lens - c["window"])
    q = s["q"].float().reshape(B, Hk, Hq // Hk, D) / math.sqrt(D)
    x = q @ _gathered(s["k_pages"], s["k_scale"], s["table"], n).transpose(-1, -2)
    x = x.masked_fill(~inside[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["v_pages"], s["v_scale"], s["table"], n).masked_fill(~inside[:, None, :, None], 0.0)
    out = (p @ v / total.masked_fill(total == 0, 1.0)).reshape(B, Hq, D).to(dt)
    return (out, (top + total.log()).reshape(B, Hq)) if c["lse"] else out


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "attend": _plain_attend}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def _rotation(x, pos, inv_freq, amplitude, interleaved):
    """The rotation as a product of complex numbers: x (tokens, heads, D) in 64 bits."""
    half = inv_freq.numel()
    unit = torch.polar(torch.full_like(pos, amplitude, dtype=torch.float64)[:, None].expand(-1, half).contiguous(),
                       pos.double()[:, None] * inv_freq)[:, None]
    y = x.clone()
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous()) * unit
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _e4m3(x):
    """The nearest number of 4 significant bits (fewer below 2^-6), ties to the even one, at most 448."""
    _, e = torch.frexp(x)                        # |x| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(x), e.clamp(min=-5) - 4)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":
        def one(x):
            flat = x.double() if c["packed"] else x.double().transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])
            y = _rotation(flat, s["pos"].reshape(-1), s["inv_freq"], s["amplitude"], c["interleaved"])
            return y if c["packed"] else y.reshape(c["B"], c["S"], -1, c["D"]).transpose(1, 2).contiguous()
        return one(s["q"]), one(s["k"])

    page, lens, table = c["page"], s["lens"].tolist(), s["table"].tolist()
    if c["op"] == "append":
        cu = s["cu_new"].tolist()
        place = [(lens[b] - cu[b + 1] + t, b) for b in range(c["B"]) for t in range(cu[b], cu[b + 1])]
        pos = torch.tensor([p for p, _ in place], device="cuda")
        line = torch.tensor([table[b][p // page] * page + p % page for p, b in place], device="cuda")
        k, v, q = s["k"].double(), s["v"].double(), None
        if c["rot"]:
            k = _rotation(k, pos, s["inv_freq"], s["amplitude"], c["interleaved"])
            q = _rotation(s["q"].double(), pos, s["inv_freq"], s["amplitude"], c["interleaved"])

        def after(pages, scale, x):
            pool, H, _, D = pages.shape
            lines = pages.double().transpose(1, 2).reshape(pool * page, H, D).contiguous()
            rows = None if scale is None else scale.double().transpose(1, 2).reshape(pool * page, H).contiguous()
            if scale is not None:
                unit = x.abs().amax(-1).clamp(min=_ROW_FLOOR) / 448.0
                x, rows[line] = _e4m3(x / unit[..., None]), unit
                rows = rows.reshape(pool, page, H).transpose(1, 2).contiguous()
            lines[line] = x
            return lines.reshape(pool, page, H, D).transpose(1, 2).contiguous(), rows
        kp, ks = after(s["k_pages"], s["k_scale"], k)
        vp, vs = after(s["v_pages"], s["v_scale"], v)
        return [q, kp, vp, ks, vs]

    def sequence(pages, scale, b, lo):
        """Tokens lo.. of sequence b: (kv heads, tokens, D) in 64 bits."""
        ids = s["table"][b, lo // page:-(-lens[b] // page)].long()
        x = pages.view(torch.uint8)[ids].view(_F8).double() if scale is not None else pages[ids].double()
        if scale is not None:
            x *= scale[ids].double()[..., None]
        x = x.transpose(0, 1).reshape(c["Hk"], -1, c["D"])
        skip = lo - lo // page * page
        return x[:, skip:skip + lens[b] - lo]

    if c["op"] == "read":
        outs = []
        for pages, scale in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
            out = torch.zeros((c["B"], c["Hk"], s["max_len"], c["D"]), dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                out[b, :, :n] = sequence(pages, scale, b, 0)
            outs.append(out)
        return tuple(outs)

    out = torch.zeros((c["B"], c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
    lse = torch.full((c["B"], c["Hq"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n:
            lo = max(0, n - c["window"]) if c["window"] else 0
            q = s["q"][b].double().reshape(c["Hk"], -1, c["D"])
            x = torch.einsum("hgd,hnd->hgn", q, sequence(s["k_pages"], s["k_scale"], b, lo)) * c["D"] ** -0.5
            lse[b] = torch.logsumexp(x, -1).reshape(-1)
            out[b] = torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1),
                                  sequence(s["v_pages"], s["v_scale"], b, lo)).reshape(c["Hq"], c["D"])
    return (out, lse) if c["lse"] else out
