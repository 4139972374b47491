"""The operators of a text-conditioned transformer layer whose weights are microscaled 4-bit floating point (MXFP4), as
this framework is timed on them: quantisation, the product, the gated feed-forward's up-projection, and cross attention
to an encoder's states whose number differs from sequence to sequence.

``run`` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
``own`` is set, through the framework's entry points. ``exact`` states the definitions in 64 bits, apart from both.

MXFP4: blocks of 32 values along K share a power of two, 2**(byte - 127); a value is a 4-bit code, sign and magnitude
out of 0, 0.5, 1, 1.5, 2, 3, 4, 6. A packed row holds 16 bytes per block (the even element in the low nibble) and a byte
per block; the tail of the last block is zeros. Block exponent floor(log2(amax)) - 2, ties to the even code, saturating.
"""
import math
import random
import types

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}   # the C entry points' element types
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # packing one feed-forward projection of the 1024-wide DiT and reading the pack back, as a calibration does
        {"name": "mx4_weight", "kind": "quant", "rows": 4096, "K": 1024, "pad": 0, "x": "f32"},
        # activations of odd width that are a section of a wider row
        {"name": "mx4_rows_odd", "kind": "quant", "rows": 2592, "K": 1037, "pad": 3, "x": "bf16"},
        # the conditioning vectors of a guided pair through the modulation projection: two rows, latency counts
        {"name": "linear_2", "kind": "linear", "M": 2, "K": 1024, "N": 6144, "x": "f32", "y": "f32", "bias": True},
        # the feed-forward's second projection of a guided 10 s request
        {"name": "linear_344", "kind": "linear", "M": 344, "K": 4096, "N": 1024, "x": "f16", "y": "f16", "bias": True},
        # the benchmark's GEMM shape with fp32 in and out, as the framework's other linears take it
        {"name": "linear_2592", "kind": "linear", "M": 2592, "K": 1024, "N": 4096, "x": "f32", "y": "f32", "bias": False},
        # a large batch on wide layers: the matrix cores' rate
        {"name": "linear_8192", "kind": "linear", "M": 8192, "K": 4096, "N": 8192, "x": "bf16", "y": "bf16", "bias": False},
        # the gated feed-forward of a 10 s request and of the benchmark's guided 60 s pair
        {"name": "glu_172", "kind": "glu", "M": 172, "K": 1024, "inner": 4096, "x": "f16", "y": "f16", "bias": True},
        {"name": "glu_2592", "kind": "glu", "M": 2592, "K": 1024, "inner": 4096, "x": "bf16", "y": "bf16", "bias": True},
        # one 10 s request over its prompt: a single short launch
        {"name": "cross_172", "kind": "cross", "B": 1, "H": 16, "G": 1, "Nq": 172, "Nk": 257, "D": 64, "x": "f16",
         "layout": "heads", "ragged": False, "mask": False},
        # the benchmark's guided pair, the two prompts of different lengths
        {"name": "cross_1296", "kind": "cross", "B": 2, "H": 16, "G": 1, "Nq": 1296, "Nk": 257, "D": 64, "x": "f16",
         "layout": "heads", "ragged": True, "mask": False},
        # one new token of each of 16 sequences over long encoder states, four query heads to a key head
        {"name": "cross_one", "kind": "cross", "B": 16, "H": 16, "G": 4, "Nq": 1, "Nk": 8192, "D": 128, "x": "bf16",
         "layout": "tokens", "ragged": True, "mask": False},
        # a batch of long sequences over long encoder states with a key mask, straight from the fused k/v projection
        {"name": "cross_4096", "kind": "cross", "B": 4, "H": 16, "G": 1, "Nq": 4096, "Nk": 2048, "D": 64, "x": "bf16",
         "layout": "tokens", "ragged": True, "mask": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quant", "linear", "linear", "glu", "cross", "cross"))
    t = ("f32", "f16", "bf16")
    if kind == "quant":
        K = _log_int(rng, 8, 8192)
        return {"kind": kind, "rows": _log_int(rng, 1, 8192), "K": K, "pad": rng.choice((0, 0, 8, 13)), "x": rng.choice(t)}
    if kind == "linear":
        K = _log_int(rng, 32, 4096)
        K = K if rng.random() < 0.3 else max(32, K // 32 * 32)
        return {"kind": kind, "M": _log_int(rng, 1, 8192), "K": K, "N": _log_int(rng, 8, 8192), "x": rng.choice(t),
                "y": rng.choice(t), "bias": rng.random() < 0.5}
    if kind == "glu":
        return {"kind": kind, "M": _log_int(rng, 1, 2592), "K": max(32, _log_int(rng, 32, 4096) // 32 * 32),
                "inner": _log_int(rng, 16, 4096), "x": rng.choice(t), "y": rng.choice(t), "bias": rng.random() < 0.5}
    B, G, D = _log_int(rng, 1, 16), rng.choice((1, 1, 2, 4)), rng.choice((32, 64, 64, 72, 96, 128))
    H, Nk = G * rng.choice((1, 2, 4, 6)), _log_int(rng, 1, 8192)
    most = min(4096, 4 * 16 * 4096 * 2048 * 64 // (B * H * Nk * max(D, 64)))   # no more work than the largest listed case
    return {"kind": kind, "B": B, "H": H, "G": G, "Nq": _log_int(rng, 1, max(1, most)), "Nk": Nk, "D": D,
            "x": rng.choice(("f16", "bf16")), "layout": rng.choice(("heads", "tokens")), "ragged": rng.random() < 0.6,
            "mask": rng.random() < 0.4}


# ---- inputs ----

def _randn(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(sigma)


def _lengths(case, seed):
    """Valid keys of each sequence: spread between a quarter and all, one of three or more without any (no prompt)."""
    B, Nk = case["B"], case["Nk"]
    if not case["ragged"]:
        return None
    n = [max(1, Nk * (4 * B - 3 * i) // (4 * B)) for i in range(B)]
    if B > 2:
        n[-1] = 0
    random.Random(seed).shuffle(n)
    return n


def _activations(case, seed, rows, K, pad=0):
    """Rows as a norm leaves them, with a few channels that run larger."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = _randn(g, rows, K + pad) * torch.exp(_randn(g, K + pad, sigma=0.5))
    return g, x.to(DTYPE[case["x"]])


def prepare(case, seed):
    kind = case["kind"]
    s = types.SimpleNamespace(kind=kind, case=case, plan=None)
    if kind == "quant":
        _, s.x = _activations(case, seed, case["rows"], case["K"], case["pad"])
    elif kind in ("linear", "glu"):
        n = case["N"] if kind == "linear" else 2 * case["inner"]
        g, s.x = _activations(case, seed, case["M"], case["K"])
        s.q, s.scale = _pack(_randn(g, n, case["K"], sigma=0.02))
        s.bias = _randn(g, n, sigma=0.02) if case["bias"] else None
    else:
        B, H, Nq, Nk, D = (case[k] for k in ("B", "H", "Nq", "Nk", "D"))
        hk, dt = H // case["G"], DTYPE[case["x"]]
        g = torch.Generator(device="cuda").manual_seed(seed)

        def unit(t):   # as the head norms leave q and k
            return t.mul_(math.sqrt(D) / t.norm(dim=-1, keepdim=True))

        if case["layout"] == "heads":
            s.q = unit(_randn(g, B, H, Nq, D)).to(dt)
            s.k, s.v = unit(_randn(g, B, hk, Nk, D)).to(dt), _randn(g, B, hk, Nk, D).to(dt)
        else:
            s.q = unit(_randn(g, B, Nq, H, D)).to(dt).transpose(1, 2)
            kv = torch.stack((unit(_randn(g, B, Nk, hk, D)), _randn(g, B, Nk, hk, D)), 2).to(dt)
            s.k, s.v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        n = _lengths(case, seed)
        s.len = torch.tensor(n, dtype=torch.int32, device="cuda") if n else None
        s.mask = (torch.rand(B, Nk, generator=g, device="cuda") > 0.125).to(torch.uint8) if case["mask"] else None
        if n:   # what lies behind a sequence's states was never written
            gone = torch.arange(Nk, device="cuda")[None, :] >= s.len[:, None]
            s.k.masked_fill_(gone[:, None, :, None], float("nan"))
            s.v.masked_fill_(gone[:, None, :, None], float("nan"))
    torch.cuda.synchronize()
    return s


# ---- the plain form ----

def _scale_and_codes(x):
    """Rows of fp32 as blocks: each block's byte [rows, nb, 1] and its values over the scale [rows, nb, 32]."""
    rows, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % 32)).reshape(rows, -1, 32)
    bits = b.abs().amax(-1, keepdim=True).view(torch.int32)
    byte = ((bits >> 23) - 2).clamp(min=0)
    v = b * ((254 - byte) << 23).view(torch.float32)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return byte, torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _pow2(byte):
    """2**(byte - 127) in fp32, the smallest (a subnormal) among them."""
    return torch.where(byte > 0, (byte << 23).view(torch.float32), 2.0 ** -127)


def _values(x):
    byte, v = _scale_and_codes(x.float())
    return (v * _pow2(byte)).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _pack(w):
    byte, v = _scale_and_codes(w)
    code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device=w.device)[(v.abs() * 2).long()]
    code = (code | torch.signbit(v).long() << 3).reshape(w.shape[0], -1, 2)
    return (code[..., 0] | code[..., 1] << 4).to(torch.uint8), byte[..., 0].to(torch.uint8)


def _unpack(q, scale, K):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
    v = table[torch.stack((q & 15, q >> 4), -1).long()].reshape(q.shape[0], -1, 32)
    return (v * _pow2(scale.int())[..., None]).reshape(q.shape[0], -1)[:, :K]


def _plain(s):
    c = s.case
    if s.kind == "quant":
        return _values(s.x[:, :c["K"]])
    if s.kind in ("linear", "glu"):
        y = torch.matmul(_values(s.x), _unpack(s.q, s.scale, c["K"]).t())
        if s.bias is not None:
            y = y + s.bias
        if s.kind == "glu":
            v, g = y[:, :c["inner"]], y[:, c["inner"]:]
            y = v * (g / (1 + torch.exp(-g)))
        return y.to(DTYPE[c["y"]])
    B, H, Nq, Nk, D = (c[k] for k in ("B", "H", "Nq", "Nk", "D"))
    q = s.q.float().reshape(B, H // c["G"], c["G"] * Nq, D)
    k, v = s.k.float().transpose(-1, -2).contiguous(), s.v.float().contiguous()
    score = torch.matmul(q, k).mul_(1 / math.sqrt(D))
    if s.len is not None or s.mask is not None:
        ok = torch.ones(B, Nk, dtype=torch.bool, device=q.device) if s.mask is None else s.mask != 0
        if s.len is not None:
            ok = ok & (torch.arange(Nk, device=q.device)[None, :] < s.len[:, None])
        ok = ok[:, None, None, :]
        score.masked_fill_(~ok, -torch.inf)
        v = torch.where(ok.transpose(-1, -2), v, 0.0)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    o = torch.matmul(score, v) / score.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return o.reshape(B, H, Nq, D).transpose(1, 2).reshape(B, Nq, H * D).to(DTYPE[c["x"]])


# ---- the framework's calls ----

def _ptr(t):
    return t.data_ptr() if t is not None else None


def _plan(s):
    """What a user's program keeps between calls: its output, its workspace, the attention's description."""
    import aria_amd
    c, L = s.case, aria_amd.lib()
    p = types.SimpleNamespace(L=L, check=aria_amd.check)
    if s.kind == "quant":
        nb = (c["K"] + 31) // 32
        p.q = torch.empty(c["rows"], 16 * nb, device="cuda", dtype=torch.uint8)
        p.scale = torch.empty(c["rows"], nb, device="cuda", dtype=torch.uint8)
        p.y = torch.empty(c["rows"], c["K"], device="cuda")
    elif s.kind in ("linear", "glu"):
        p.y = torch.empty(c["M"], c["N"] if s.kind == "linear" else c["inner"], device="cuda", dtype=DTYPE[c["y"]])
        p.ws = torch.empty(int(L.aria_hip_mx4_ws_bytes(c["M"], c["K"])), device="cuda", dtype=torch.uint8)
    else:
        B, H, Nq, Nk, D = (c[k] for k in ("B", "H", "Nq", "Nk", "D"))
        p.y = torch.empty(B, Nq, H * D, device="cuda", dtype=DTYPE[c["x"]])
        a = aria_amd.CrossAttention(q=s.q.data_ptr(), k=s.k.data_ptr(), v=s.v.data_ptr(), out=p.y.data_ptr(),
                                    kv_len=_ptr(s.len), mask=_ptr(s.mask), type=CODE[c["x"]], B=B, H=H, Hkv=H // c["G"],
                                    Nq=Nq, Nk=Nk, D=D, scale=1 / math.sqrt(D), mask_stride=Nk)
        for name, t in (("q", s.q), ("k", s.k), ("v", s.v)):
            for axis, dim in (("batch", 0), ("head", 1), ("token", 2)):
                setattr(a, "%s_%s" % (name, axis), t.stride(dim))
        a.o_batch, a.o_head, a.o_token = Nq * H * D, D, H * D
        p.a = a
        p.ws = torch.empty(int(L.aria_hip_cross_attention_ws_bytes(a)), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    return p


def _own(s):
    c = s.case
    if s.plan is None:
        s.plan = _plan(s)
    p = s.plan
    L, check = p.L, p.check
    if s.kind == "quant":
        check(L.aria_hip_mx4_quant_dev(p.q.data_ptr(), p.scale.data_ptr(), s.x.data_ptr(), CODE[c["x"]], c["rows"], c["K"],
                                       c["K"] + c["pad"], None), "quant")
        check(L.aria_hip_mx4_dequant_dev(p.y.data_ptr(), 0, p.q.data_ptr(), p.scale.data_ptr(), c["rows"], c["K"], None),
              "dequant")
    elif s.kind == "linear":
        check(L.aria_hip_linear_mx4_dev(p.y.data_ptr(), CODE[c["y"]], s.x.data_ptr(), CODE[c["x"]], c["K"], s.q.data_ptr(),
                                        s.scale.data_ptr(), _ptr(s.bias), c["M"], c["K"], c["N"], p.ws.data_ptr(), None),
              "linear")
    elif s.kind == "glu":
        check(L.aria_hip_glu_mx4_dev(p.y.data_ptr(), CODE[c["y"]], s.x.data_ptr(), CODE[c["x"]], c["K"], s.q.data_ptr(),
                                     s.scale.data_ptr(), _ptr(s.bias), c["M"], c["K"], c["inner"], p.ws.data_ptr(), None),
              "glu")
    else:
        check(L.aria_hip_cross_attention_dev(p.a, p.ws.data_ptr(), None), "cross attention")
    return p.y


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "quant":
        n = case["rows"] * case["K"]
        return {"bytes": n * (SIZE[case["x"]] + 4), "flops": 0}
    if kind in ("linear", "glu"):
        M, K = case["M"], case["K"]
        n, out = (case["N"], case["N"]) if kind == "linear" else (2 * case["inner"], case["inner"])
        return {"bytes": M * K * SIZE[case["x"]] + n * ((K + 31) // 32) * 17 + 4 * n * case["bias"] + M * out * SIZE[case["y"]],
                "flops": 2 * M * K * n}
    B, H, Nq, Nk, D = (case[k] for k in ("B", "H", "Nq", "Nk", "D"))
    n = sum(_lengths(case, 0) or [Nk] * B)
    return {"bytes": 2 * D * (2 * B * H * Nq + 2 * n * H // case["G"]) + B * Nk * case["mask"], "flops": 4 * H * Nq * n * D}


# ---- the definitions in 64 bits ----

def _exact_mx4(x):
    """Each value of x [rows, K] as the nearest representable one of its block."""
    K = x.shape[1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    middles = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
    steps = (0.5, 0.5, 0.5, 0.5, 1.0, 1.0, 2.0)
    whole = K // 32 * 32
    for lo, hi, width in ((0, whole, 32), (whole, K, K - whole)):
        if hi > lo:
            b = x[:, lo:hi].double().reshape(x.shape[0], -1, width)
            top = b.abs().amax(-1, keepdim=True)
            e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)
            a, m = torch.ldexp(b.abs(), -e), torch.zeros_like(b)
            for (middle, up), step in zip(middles, steps):   # a tie goes to the code with an even last bit
                m += step * ((a >= middle) if up else (a > middle))
            out[:, lo:hi] = torch.ldexp(m * torch.sign(b), e).reshape(x.shape[0], -1)
    return out


def _exact_weight(q, scale, K):
    code = torch.stack((q % 16, q // 16), -1).reshape(q.shape[0], -1).double()
    sign, m = torch.where(code >= 8, -1.0, 1.0), code % 8
    e = (m / 2).floor()
    v = sign * torch.where(e > 0, (1 + (m % 2) / 2) * 2 ** (e - 1), m / 2)
    return torch.ldexp(v, scale.double().repeat_interleave(32, 1) - 127)[:, :K]


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "quant":
        return _exact_mx4(s.x[:, :case["K"]])
    if s.kind in ("linear", "glu"):
        y = _exact_mx4(s.x) @ _exact_weight(s.q, s.scale, case["K"]).T
        y = y if s.bias is None else y + s.bias.double()
        if s.kind == "glu":
            v, g = y.chunk(2, -1)
            y = v * g * torch.sigmoid(g)
        return y
    B, H, Nq, Nk, D = (case[k] for k in ("B", "H", "Nq", "Nk", "D"))
    out = torch.zeros(B, Nq, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        ok = torch.ones(Nk, dtype=torch.bool, device="cuda") if s.mask is None else s.mask[b].bool()
        if s.len is not None:
            ok[int(s.len[b]):] = False
        if bool(ok.any()):
            for h in range(H):
                k, v = (t[b, h // case["G"]][ok].double() for t in (s.k, s.v))
                p = torch.softmax(s.q[b, h].double() @ k.T.contiguous() / math.sqrt(D), -1)
                out[b, :, h] = p @ v
    return out.reshape(B, Nq, H * D)
