"""The operators of a transformer that keeps the keys and values of what several requests share, as this framework is timed
on them: rotary positions by table, a cache of keys and values held in 8 bits, and attention for a batch that shares a long
prefix of that cache.

``run`` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
``own`` is set, through the framework's entry points. ``exact`` states the definitions in 64 bits, apart from both.

A cached row is the key or value of one token and head: codes in e4m3 (sign, 4 bits of exponent, 3 of mantissa; 448 the
largest) under one power of two 2**(byte - 127), the smallest that brings the row's largest magnitude to 448 or less (the
byte at least 1). Keys are rotated as they are written: in 32 bits, rounded once, then to the nearest code, ties to even.
"""
import math
import random
import types

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}   # the C entry points' element types
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALING = ("none", "linear", "base", "turns")   # the C entry points' kinds


def listed():
    return [
        # the tables of a model whose context is stretched to eight times its trained length, made once at its start
        {"name": "table_131072", "kind": "table", "n": 131072, "first": 0, "rot": 128, "scaling": "turns", "factor": 8.0},
        # queries and keys of a guided 10 s request, half of each head rotated
        {"name": "rotary_172", "kind": "rotary", "B": 2, "N": 172, "H": 16, "G": 1, "D": 64, "rot": 32, "npos": 172,
         "pair": "half", "x": "f16", "layout": "heads", "pos": "first"},
        # four long prompts of packed documents, whose positions begin anew, out of a fused projection
        {"name": "rotary_8192", "kind": "rotary", "B": 4, "N": 8192, "H": 16, "G": 4, "D": 128, "rot": 128, "npos": 131072,
         "pair": "interleaved", "x": "bf16", "layout": "tokens", "pos": "given"},
        # one new token of each of 64 sequences into the cache: a single short launch
        {"name": "write_1", "kind": "write", "B": 64, "N": 1, "H": 16, "G": 4, "D": 128, "rot": 64, "cap": 8192,
         "pair": "interleaved", "x": "bf16", "layout": "tokens", "ragged": False, "q": True},
        # the benchmark's guided pair of 60 s, of different lengths
        {"name": "write_1296", "kind": "write", "B": 2, "N": 1296, "H": 16, "G": 1, "D": 64, "rot": 32, "cap": 1360,
         "pair": "half", "x": "f16", "layout": "heads", "ragged": True, "q": True},
        # an encoder's states of odd number and width in fp32, without positions
        {"name": "write_1037", "kind": "write", "B": 3, "N": 1037, "H": 8, "G": 1, "D": 80, "rot": 0, "cap": 1040,
         "pair": "half", "x": "f32", "layout": "tokens", "ragged": True, "q": False},
        # four long prompts at once, and the cache read back for a layer that wants it in 16 bits
        {"name": "write_16384", "kind": "write", "B": 4, "N": 16384, "H": 8, "G": 1, "D": 128, "rot": 128, "cap": 16384,
         "pair": "half", "x": "bf16", "layout": "tokens", "ragged": False, "q": False},
        # four variants of a guided 10 s request: two prompts, each read by four sequences
        {"name": "attend_172", "kind": "attend", "B": 8, "P": 2, "Nq": 172, "H": 16, "G": 1, "D": 64, "prefix": 257,
         "own": 0, "causal": False, "ragged": True, "x": "f16"},
        # one new token of each of 32 sequences behind a common prompt
        {"name": "attend_1", "kind": "attend", "B": 32, "P": 1, "Nq": 1, "H": 16, "G": 4, "D": 128, "prefix": 8192,
         "own": 512, "causal": True, "ragged": True, "x": "bf16"},
        # one new token of each of 8 sequences behind a very long document: the prefix's bytes
        {"name": "attend_1_131072", "kind": "attend", "B": 8, "P": 1, "Nq": 1, "H": 16, "G": 4, "D": 128, "prefix": 131072,
         "own": 64, "causal": True, "ragged": True, "x": "bf16"},
        # the benchmark's 60 s sequences, all of whose tokens see each other and a common context
        {"name": "attend_1296", "kind": "attend", "B": 4, "P": 1, "Nq": 1296, "H": 16, "G": 1, "D": 64, "prefix": 2048,
         "own": 1296, "causal": False, "ragged": False, "x": "f16"},
        # the next 512 tokens of each of 8 sequences, behind a common prompt and what they hold already
        {"name": "attend_512", "kind": "attend", "B": 8, "P": 1, "Nq": 512, "H": 16, "G": 4, "D": 128, "prefix": 8192,
         "own": 1024, "causal": True, "ragged": True, "x": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("table", "rotary", "rotary", "write", "write", "attend", "attend", "attend"))
    if kind == "table":
        return {"kind": kind, "n": _log_int(rng, 64, 131072), "first": rng.choice((0, 0, _log_int(rng, 1, 1 << 20))),
                "rot": 2 * rng.randint(8, 64), "scaling": rng.choice(SCALING), "factor": rng.choice((1.5, 2.0, 4.0, 8.0))}
    D, G = rng.choice((32, 64, 64, 80, 96, 128, 128)), rng.choice((1, 1, 2, 4))
    H, pair = G * rng.choice((1, 2, 4, 8)), rng.choice(("half", "interleaved"))
    rot = rng.choice((D, D, D // 2, D - 6))
    if kind == "rotary":
        B, x = _log_int(rng, 1, 64), rng.choice(("f32", "f16", "bf16"))
        N = _log_int(rng, 1, max(1, min(16384, 4 * 8192 * 20 * 128 * 2 // (B * (H + H // G) * D * SIZE[x]))))
        given = rng.random() < 0.5
        return {"kind": kind, "B": B, "N": N, "H": H, "G": G, "D": D, "rot": rot,
                "npos": _log_int(rng, 64, 131072) if given else 2 * N + 64, "pair": pair, "x": x,
                "layout": rng.choice(("heads", "tokens")), "pos": "given" if given else "first"}
    if kind == "write":
        B, x = _log_int(rng, 1, 64), rng.choice(("f32", "f16", "bf16"))
        q = rng.random() < 0.5
        N = _log_int(rng, 1, max(1, min(16384, 4 * 16384 * 8 * 128 * 2 // (B * (H // G + q * H) * D * SIZE[x]))))
        return {"kind": kind, "B": B, "N": N, "H": H, "G": G, "D": D, "rot": rng.choice((0, rot, rot)),
                "cap": N + _log_int(rng, 1, 1024), "pair": pair, "x": x, "layout": rng.choice(("heads", "tokens")),
                "ragged": rng.random() < 0.6, "q": q}
    P, prefix = rng.choice((1, 1, 1, 2, 4)), _log_int(rng, 16, 131072)
    B = P * _log_int(rng, 1, 64 // P)
    mine = rng.choice((0, _log_int(rng, 1, 2048), _log_int(rng, 1, 2048)))
    most = 8 * 512 * 16 * 9216 * 128 // (B * H * (prefix + mine) * max(D, 64))   # no more work than the largest listed case
    Nq = _log_int(rng, 1, max(1, min(1296, most)))
    causal = mine > Nq and rng.random() < 0.6
    return {"kind": kind, "B": B, "P": P, "Nq": Nq, "H": H, "G": G, "D": D, "prefix": prefix, "own": mine, "causal": causal,
            "ragged": rng.random() < 0.6, "x": rng.choice(("f16", "bf16"))}


# ---- inputs ----

def _randn(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(sigma)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _counts(case, seed):
    """Tokens of each sequence: spread between a quarter and all, one of three or more without any."""
    B, N = case["B"], case["N"]
    if not case["ragged"]:
        return None
    n = [max(1, N * (4 * B - 3 * i) // (4 * B)) for i in range(B)]
    if B > 2:
        n[-1] = 0
    random.Random(seed).shuffle(n)
    return n


def _lengths(case, seed):
    """Keys of each prefix and of each sequence's own part, and where in it the sequence's first query stands."""
    P, B, Nq = case["P"], case["B"], case["Nq"]
    lp, lo = [case["prefix"]] * P, [case["own"]] * B
    if case["ragged"]:
        least = Nq if case["causal"] else 0
        lp = [max(1, case["prefix"] * (4 * P - i) // (4 * P)) for i in range(P)]
        lo = [least + (case["own"] - least) * (B - i) // B for i in range(B)]
        random.Random(seed).shuffle(lo)
    return lp, lo, [n - Nq for n in lo]


def _frequencies(rot, scaling="none", factor=1.0, base=10000.0, trained=16384.0, low=1.0, high=32.0):
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "turns":   # pairs that turn often over the trained length stay, those that hardly turn are stretched
        w = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (w + (1 - w) / factor)
    return f


def _angles(first, n, f):
    return torch.arange(first, first + n, dtype=torch.float64, device="cuda")[:, None] * f


def _states(g, case, heads, layout, channel=None):
    """[B, N, heads, D] of the case's type, tokens or heads first in memory."""
    t = _randn(g, case["B"], case["N"], heads, case["D"])
    if channel is not None:
        t = t * channel
    t = t.to(DTYPE[case["x"]])
    return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "heads" else t


def prepare(case, seed):
    kind = case["kind"]
    s = types.SimpleNamespace(kind=kind, case=case, plan=None, gain=1.0)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "table":
        s.base = 10000.0 * (1 + seed % 7 / 100)
        s.f = _frequencies(case["rot"], case["scaling"], case["factor"], s.base)
        s.gain = 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "turns" else 1.0
    if kind in ("rotary", "write"):
        B, N, H, D = (case[k] for k in ("B", "N", "H", "D"))
        hk, fused = H // case["G"], case["layout"] == "tokens"
        s.npos = case["npos"] if kind == "rotary" else case["cap"]
        if case["rot"]:
            a = _angles(0, s.npos, _frequencies(case["rot"]))
            s.cos, s.sin = a.cos().float(), a.sin().float()
        s.pos, n = None, _counts(case, seed) if kind == "write" else None
        s.count = _ints(n) if n else None
        r = random.Random(seed)
        if kind == "rotary" and case["pos"] == "given":   # documents of unequal length, each from a place of its own
            t = torch.arange(N, device="cuda")[None, :] + torch.randint(0, s.npos, (B, 1), generator=g, device="cuda")
            t = t + torch.randint(0, s.npos, (B, N // 512 + 1), generator=g, device="cuda").repeat_interleave(512, 1)[:, :N]
            s.pos = (t % s.npos).to(torch.int32)
        s.first = None if s.pos is not None else _ints([r.randint(0, s.npos - N) for _ in range(B)])
        if fused:   # sections of one projection's rows
            both = _states(g, case, H + 2 * hk, "tokens", torch.exp(_randn(g, H + 2 * hk, D, sigma=0.5)))
            s.q, s.k, s.v = both[:, :, :H], both[:, :, H:H + hk], both[:, :, H + hk:]
        else:
            s.q, s.k, s.v = (_states(g, case, h, "heads", torch.exp(_randn(g, h, D, sigma=0.5))) for h in (H, hk, hk))
    if kind == "attend":
        B, P, Nq, H, D = (case[k] for k in ("B", "P", "Nq", "H", "D"))
        hk, dt = H // case["G"], DTYPE[case["x"]]

        def unit(t):   # as the head norms leave q and k
            return t.mul_(math.sqrt(D) / t.norm(dim=-1, keepdim=True))

        s.q = unit(_randn(g, B, Nq, H, D)).to(dt).transpose(1, 2)
        lp, lo, first = _lengths(case, seed)
        s.prefix_len, s.own_len, s.first = _ints(lp), _ints(lo), _ints(first) if case["causal"] else None
        s.cache = []
        for n, cap in ((P, case["prefix"]), (B, case["own"])):
            for data in (unit(_randn(g, n, hk, cap, D)) if cap else _randn(g, n, hk, cap, D), _randn(g, n, hk, cap, D)):
                code, byte = _quantise(data.to(dt).float())
                s.cache += [code.to(torch.float8_e4m3fn).view(torch.uint8), byte.to(torch.uint8)]
        # what lies behind a sequence's keys was never written: NaN
        for i, n in ((0, s.prefix_len), (4, s.own_len)):
            gone = torch.arange(s.cache[i].shape[2], device="cuda")[None, None, :] >= n[:, None, None]
            for j in (0, 2):
                s.cache[i + j].masked_fill_(gone[..., None], 0x7F)
                s.cache[i + j + 1].masked_fill_(gone, 0xFF)
    torch.cuda.synchronize()
    return s


# ---- the plain form ----

def _quantise(x):
    """Rows of fp32: the values of their codes and each row's byte [...]."""
    top = x.abs().amax(-1) if x.numel() else x.new_zeros(x.shape[:-1])
    m, e = torch.frexp(top)                                # top = m 2^e, m in [0.5, 1)
    byte = torch.where(top > 0, (e + 118 + (m > 0.875)).clamp(min=1), 1)
    v = x * ((254 - byte) << 23).to(torch.int32).view(torch.float32)[..., None]
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1].clamp(min=-5) - 4)
    return torch.round(v / step) * step, byte


def _value(code, byte):
    return code.view(torch.float8_e4m3fn).float() * (byte.to(torch.int32) << 23).view(torch.float32)[..., None]


def _rotate(x, cos, sin, pair, rot):
    """x [B, N, heads, D] by cos / sin [B, N, rot / 2], in the tables' type."""
    cos, sin = cos[:, :, None], sin[:, :, None]
    if pair == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _places(s):
    """The position of every token [B, N]."""
    return s.pos.long() if s.pos is not None else s.first.long()[:, None] + torch.arange(s.case["N"], device="cuda")[None, :]


def _plain_states(s):
    c = s.case
    dt, at = DTYPE[c["x"]], _places(s)
    if s.kind == "rotary":
        cos, sin = s.cos[at], s.sin[at]
        return [_rotate(t.float(), cos, sin, c["pair"], c["rot"]).to(dt) for t in (s.q, s.k)]
    k, q = s.k.float(), s.q.float()
    if c["rot"]:
        cos, sin = s.cos[at].double(), s.sin[at].double()   # next to a border between codes 32 bits lose what matters
        k = _rotate(k.double(), cos, sin, c["pair"], c["rot"]).float()
        if c["q"]:
            q = _rotate(q, s.cos[at], s.sin[at], c["pair"], c["rot"])
    out = []
    for t in (k, s.v.float()):
        code, byte = _quantise(t)
        out.append((code * (byte << 23).to(torch.int32).view(torch.float32)[..., None]).to(dt))
    if c["q"]:
        out.append(q.to(dt))
    if s.count is not None:
        gone = (torch.arange(c["N"], device="cuda")[None, :] >= s.count[:, None])[:, :, None, None]
        out = [t.masked_fill(gone, 0.0) for t in out]
    return out


def _plain_attend(s):
    c = s.case
    B, P, Nq, H, D = (c[k] for k in ("B", "P", "Nq", "H", "D"))
    hk, np_, no, dev = H // c["G"], c["prefix"], c["own"], s.q.device
    q = s.q.float().reshape(B, hk, c["G"] * Nq, D)
    shared = q.reshape(P, B // P, hk, -1, D).transpose(1, 2).reshape(P, hk, -1, D)   # every row that reads a prefix
    ok_p = torch.arange(np_, device=dev)[None, :] < s.prefix_len[:, None]
    ok_o = torch.arange(no, device=dev)[None, :] < s.own_len[:, None]
    kp, vp, ko, vo = (_value(*s.cache[i:i + 2]) for i in (0, 2, 4, 6))
    kp, vp = (torch.where(ok_p[:, None, :, None], t, 0.0) for t in (kp, vp))
    ko, vo = (torch.where(ok_o[:, None, :, None], t, 0.0) for t in (ko, vo))
    sp = torch.matmul(shared, kp.transpose(-1, -2).contiguous()).masked_fill_(~ok_p[:, None, None, :], -torch.inf)
    sp = sp.reshape(P, hk, B // P, c["G"] * Nq, np_).transpose(1, 2).reshape(B, hk, c["G"] * Nq, np_)
    so = torch.matmul(q, ko.transpose(-1, -2).contiguous()).reshape(B, H, Nq, no)
    ok = ok_o[:, None, None, :].expand(B, 1, Nq, no)
    if s.first is not None:
        t = s.first[:, None] + torch.arange(Nq, device=dev)[None, :]
        ok = ok & (torch.arange(no, device=dev)[None, None, :] <= t[:, :, None])[:, None]
    so = so.masked_fill_(~ok, -torch.inf).reshape(B, hk, c["G"] * Nq, no)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True)) if no else sp.amax(-1, keepdim=True)
    top = top.clamp(min=torch.finfo(torch.float32).min)
    sp, so = (t.sub_(top).mul_(1 / math.sqrt(D)).exp_() for t in (sp, so))
    n = (sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)).clamp(min=torch.finfo(torch.float32).tiny)
    wide = sp.reshape(P, B // P, hk, -1, np_).transpose(1, 2).reshape(P, hk, -1, np_)
    o = torch.matmul(wide, vp).reshape(P, hk, B // P, -1, D).transpose(1, 2).reshape(B, hk, -1, D)
    o = (o + torch.matmul(so, vo)) / n
    return o.reshape(B, H, Nq, D).transpose(1, 2).reshape(B, Nq, H * D).to(DTYPE[c["x"]])


def _plain(s):
    if s.kind == "table":
        a = _angles(s.case["first"], s.case["n"], s.f)
        return [(a.cos() * s.gain).float(), (a.sin() * s.gain).float()]
    return _plain_attend(s) if s.kind == "attend" else _plain_states(s)


# ---- the framework's calls ----

def _ptr(t):
    return t.data_ptr() if t is not None else None


def _strides(a, name, t):
    """t [B, N, heads, D]"""
    for axis, dim in (("batch", 0), ("token", 1), ("head", 2)):
        setattr(a, "%s_%s" % (name, axis), t.stride(dim))


def _cache(aria_amd, code, byte, code_v, byte_v):
    """codes [B, heads, cap, D] and bytes [B, heads, cap] as the entry points take them"""
    B, hk, cap, D = code.shape
    return aria_amd.KVCache(k=code.data_ptr(), v=code_v.data_ptr(), k_scale=byte.data_ptr(), v_scale=byte_v.data_ptr(), B=B,
                            Hkv=hk, D=D, cap=cap, batch=hk * cap * D, head=cap * D, token=D, s_batch=hk * cap, s_head=cap)


def _plan(s):
    """What a user's program keeps between calls: outputs, the cache, the workspace and the descriptions."""
    import aria_amd
    c, L = s.case, aria_amd.lib()
    p = types.SimpleNamespace(L=L, check=aria_amd.check)
    if s.kind == "table":
        p.y = [torch.empty(c["n"], c["rot"] // 2, device="cuda") for _ in range(2)]
        p.a = aria_amd.RotaryScaling(rot=c["rot"], kind=SCALING.index(c["scaling"]), base=s.base, factor=c["factor"],
                                     trained=16384.0, low=1.0, high=32.0, gain=s.gain)
    elif s.kind == "rotary":
        B, N, H, D = (c[k] for k in ("B", "N", "H", "D"))
        p.y = [torch.empty(t.shape, device="cuda", dtype=t.dtype) for t in (s.q, s.k)]
        a = p.a = aria_amd.Rotary(q=s.q.data_ptr(), k=s.k.data_ptr(), q_out=p.y[0].data_ptr(), k_out=p.y[1].data_ptr(),
                                  cos=s.cos.data_ptr(), sin=s.sin.data_ptr(), pos=_ptr(s.pos), first=_ptr(s.first),
                                  pos_stride=N, type=CODE[c["x"]], B=B, N=N, Hq=H, Hk=H // c["G"], D=D, rot=c["rot"],
                                  npos=s.npos, interleaved=c["pair"] == "interleaved")
        for name, t in (("q", s.q), ("k", s.k), ("qo", p.y[0]), ("ko", p.y[1])):
            _strides(a, name, t)
    elif s.kind == "write":
        B, N, H, D = (c[k] for k in ("B", "N", "H", "D"))
        hk = H // c["G"]
        p.code = [torch.zeros(B, hk, c["cap"], D, device="cuda", dtype=torch.uint8) for _ in range(2)]
        p.byte = [torch.zeros(B, hk, c["cap"], device="cuda", dtype=torch.uint8) for _ in range(2)]
        p.y = [torch.zeros(t.shape, device="cuda", dtype=t.dtype) for t in ((s.k, s.v, s.q) if c["q"] else (s.k, s.v))]
        cache = _cache(aria_amd, p.code[0], p.byte[0], p.code[1], p.byte[1])
        a = p.a = aria_amd.KVWrite(cache=cache, k=s.k.data_ptr(), v=s.v.data_ptr(), pos=None, first=s.first.data_ptr(),
                                   count=_ptr(s.count), type=CODE[c["x"]], N=N, rot=c["rot"], npos=s.npos,
                                   interleaved=c["pair"] == "interleaved")
        if c["rot"]:
            a.cos, a.sin = s.cos.data_ptr(), s.sin.data_ptr()
        _strides(a, "k", s.k)
        _strides(a, "v", s.v)
        if c["q"]:
            a.q, a.q_out, a.Hq = s.q.data_ptr(), p.y[2].data_ptr(), H
            _strides(a, "q", s.q)
            _strides(a, "qo", p.y[2])
        r = p.r = aria_amd.KVRead(cache=cache, k=p.y[0].data_ptr(), v=p.y[1].data_ptr(), first=s.first.data_ptr(),
                                  count=_ptr(s.count), type=CODE[c["x"]], N=N)
        _strides(r, "k", p.y[0])
        _strides(r, "v", p.y[1])
    else:
        B, Nq, H, D = (c[k] for k in ("B", "Nq", "H", "D"))
        p.y = torch.empty(B, Nq, H * D, device="cuda", dtype=DTYPE[c["x"]])
        a = p.a = aria_amd.PrefixAttention(q=s.q.data_ptr(), out=p.y.data_ptr(), prefix=_cache(aria_amd, *s.cache[:4]),
                                           own=_cache(aria_amd, *s.cache[4:]), prefix_len=s.prefix_len.data_ptr(),
                                           own_len=s.own_len.data_ptr(), first=_ptr(s.first), type=CODE[c["x"]], B=B, H=H,
                                           Nq=Nq, scale=1 / math.sqrt(D))
        _strides(a, "q", s.q.transpose(1, 2))
        _strides(a, "o", p.y.view(B, Nq, H, D))
        p.ws = torch.empty(int(L.aria_hip_prefix_attention_ws_bytes(a)), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    return p


def _own(s):
    if s.plan is None:
        s.plan = _plan(s)
    p = s.plan
    if s.kind == "table":
        p.check(p.L.aria_hip_rotary_table_dev(p.y[0].data_ptr(), p.y[1].data_ptr(), p.a, s.case["first"], s.case["n"], None),
                "table")
    elif s.kind == "rotary":
        p.check(p.L.aria_hip_rotary_dev(p.a, None), "rotary")
    elif s.kind == "write":
        p.check(p.L.aria_hip_kv_write_dev(p.a, None), "write")
        p.check(p.L.aria_hip_kv_read_dev(p.r, None), "read")
    else:
        p.check(p.L.aria_hip_prefix_attention_dev(p.a, p.ws.data_ptr(), None), "attention")
    return p.y


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "table":
        n = case["n"] * case["rot"] // 2
        return {"bytes": 8 * n, "flops": 2 * n}
    H, D, x = case["H"], case["D"], SIZE[case["x"]]
    hk = H // case["G"]
    if kind == "rotary":
        rows = case["B"] * case["N"]
        table = min(case["npos"], rows) * case["rot"] * 4
        return {"bytes": 2 * rows * (H + hk) * D * x + table, "flops": 3 * rows * (H + hk) * case["rot"]}
    if kind == "write":
        rows = sum(_counts(case, 0) or [case["N"]] * case["B"])
        table = min(case["cap"], rows) * case["rot"] * 4
        cached = 2 * rows * hk
        return {"bytes": cached * (2 * D * x + D + 1) + 2 * rows * H * D * x * case["q"] + table, "flops": 2 * cached * D}
    lp, lo, first = _lengths(case, 0)
    B, Nq = case["B"], case["Nq"]
    cached = (sum(lp) + sum(lo)) * hk * 2 * (D + 1)
    seen = Nq * sum(lp) * (B // case["P"])
    if case["causal"]:
        seen += sum(Nq * (f + 1) + Nq * (Nq - 1) // 2 for f in first)
    else:
        seen += Nq * sum(lo)
    return {"bytes": cached + 2 * B * Nq * H * D * x, "flops": 4 * H * D * seen}


# ---- the definitions in 64 bits ----

def _e4m3():
    """The values of codes 0 .. 126."""
    return torch.tensor([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device="cuda")


def _exact_row(x):
    """Each value of x [..., D] as the nearest one that its row can hold."""
    values = _e4m3()
    middles = (values[1:] + values[:-1]) / 2
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448))
    e = torch.where(top > torch.ldexp(torch.full_like(top, 448.0), e), e + 1, e)
    e = torch.where(top <= torch.ldexp(torch.full_like(top, 448.0), e - 1), e - 1, e)
    e = torch.where(top > 0, e, -126.0).clamp(min=-126)
    a = torch.ldexp(x.abs(), -e)
    i = torch.searchsorted(middles, a)                       # middles below a; a tie goes to the even code
    i = i + ((i < 126) & (i % 2 == 1) & (middles[i.clamp(max=125)] == a))
    return torch.ldexp(values[i], e) * torch.sign(x)


def _exact_cache(code, byte):
    low, sign = code.long() % 128, torch.where(code >= 128, -1.0, 1.0).double()
    return torch.ldexp(_e4m3()[low.clamp(max=126)] * sign, byte.double()[..., None] - 127)


def _exact_states(s):
    c = s.case
    at = _places(s)

    def turned(t):
        t = t.double()
        if not c["rot"]:
            return t
        z = torch.complex(s.cos[at].double(), s.sin[at].double())[:, :, None]
        half = c["rot"] // 2
        pairs = torch.stack((t[..., :half], t[..., half:2 * half]), -1) if c["pair"] == "half" else \
            t[..., :c["rot"]].unflatten(-1, (half, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        y = torch.cat((y[..., 0], y[..., 1]), -1) if c["pair"] == "half" else y.flatten(-2)
        return torch.cat((y, t[..., c["rot"]:]), -1)

    if s.kind == "rotary":
        return [turned(s.q), turned(s.k)]
    out = [_exact_row(turned(s.k).float().double()), _exact_row(s.v.double())] + ([turned(s.q)] if c["q"] else [])
    if s.count is not None:
        for b in range(c["B"]):
            for t in out:
                t[b, int(s.count[b]):] = 0.0
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "table":
        a = _angles(case["first"], case["n"], s.f)
        return [torch.cos(a) * s.gain, torch.sin(a) * s.gain]
    if s.kind != "attend":
        return _exact_states(s)
    B, P, Nq, H, D = (case[k] for k in ("B", "P", "Nq", "H", "D"))
    lp, lo, first = _lengths(case, seed)
    out = torch.zeros(B, Nq, H, D, dtype=torch.float64, device="cuda")
    kp, vp, ko, vo = ((s.cache[i], s.cache[i + 1]) for i in (0, 2, 4, 6))
    for p in range(P):
        for h in range(H // case["G"]):
            a, v = (_exact_cache(t[0][p, h, :lp[p]], t[1][p, h, :lp[p]]) for t in (kp, vp))
            for b in range(p * B // P, (p + 1) * B // P):
                k1, v1 = (_exact_cache(t[0][b, h, :lo[b]], t[1][b, h, :lo[b]]) for t in (ko, vo))
                k, w = torch.cat((a, k1)), torch.cat((v, v1))
                place = torch.arange(len(k), device="cuda") - lp[p]
                for g in range(h * case["G"], (h + 1) * case["G"]):
                    score = s.q[b, g].double() @ k.T / math.sqrt(D)
                    if case["causal"]:
                        t = first[b] + torch.arange(Nq, device="cuda")
                        score = score.masked_fill(place[None, :] > t[:, None], -torch.inf)
                    out[b, :, g] = torch.softmax(score, -1) @ w
    return out.reshape(B, Nq, H * D)
