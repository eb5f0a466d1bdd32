"""Cases of the operators that an encoder's training and serving add: attention over packed texts
with its gradients, the gated projection of a feed-forward block with its gradients, and an
AdamW step over many tensors with states in 32 or 8 bits.

``own`` False: the plain forms (elementary torch operations in fp32, rounded once at the
end); True: the package's calls. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

DEV = torch.device("cuda", 0)

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 128  # elements that share an exponent in 8-bit states; tensors' states begin at multiples of it


def listed():
    return [
        # Attention. Latency: one query of 32 tokens encoded while a search waits for it.
        dict(name="attention 1 query", op="attention", B=1, lo=32, hi=32, H=12, KV=12, D=64, dtype="bf16", mask="text", cap=0.0,
             bias=False, fused=False, train=False),
        # A training batch's documents without their padding, 32 to 300 tokens, one projection's thirds.
        dict(name="attention 128 documents", op="attention", B=128, lo=32, hi=300, H=12, KV=12, D=64, dtype="bf16", mask="text",
             cap=0.0, bias=True, fused=True, train=True),
        # A decoder's layer as an encoder: a prefix that sees itself, then causal, shared heads, capped scores, odd lengths.
        dict(name="attention prefix capped", op="attention", B=37, lo=1, hi=701, H=8, KV=2, D=128, dtype="fp16", mask="prefix", cap=30.0,
             bias=False, fused=True, train=True),
        # The same checked in fp32: few short texts.
        dict(name="attention fp32", op="attention", B=16, lo=20, hi=180, H=4, KV=4, D=96, dtype="fp32", mask="text", cap=0.0, bias=True,
             fused=False, train=True),
        # Two long documents.
        dict(name="attention 2 x 8192", op="attention", B=2, lo=8192, hi=8192, H=12, KV=12, D=64, dtype="bf16", mask="text", cap=0.0,
             bias=True, fused=False, train=True),
        # Gated projections. Latency: one token's.
        dict(name="gated 1 token", op="gated", N=1, d=768, F=2048, dtype="bf16", act="silu", train=False),
        # Odd numbers of tokens and of columns.
        dict(name="gated 1229 gelu", op="gated", N=1229, d=768, F=2043, dtype="fp16", act="gelu", train=True),
        # The same checked in fp32.
        dict(name="gated fp32", op="gated", N=500, d=256, F=683, dtype="fp32", act="silu", train=True),
        # A batch's tokens through a wide block.
        dict(name="gated 16384", op="gated", N=16384, d=1024, F=4096, dtype="bf16", act="silu", train=True),
        # AdamW. Latency: a projection head alone.
        dict(name="adamw head", op="adamw", layers=0, d=768, V=128, grads="fp32", copies="", bits=32, clips=False),
        # An encoder with 8-bit states: bf16 gradients, clipped in the step, fp32 parameters and the bf16 ones that the next pass reads.
        dict(name="adamw encoder 8 bits", op="adamw", layers=12, d=768, V=30011, grads="bf16", copies="bf16", bits=8, clips=True),
        # A larger encoder in fp32 throughout.
        dict(name="adamw encoder fp32", op="adamw", layers=24, d=1024, V=32000, grads="fp32", copies="", bits=32, clips=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "gated", "gated", "adamw"])
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "bf16", "fp32"])
    if op == "attention":
        D = rng.choice([32, 64, 64, 96, 128])
        KV = rng.choice([1, 2, 4, 12])
        H = KV * rng.choice([1, 1, 1, 2, 4]) if KV < 12 else 12
        hi = _log(rng, 1, 8192)
        most = 2 * 8192 * 8192 * 12 * 64 // (2 if dtype != "fp32" else 30)
        B = max(1, min(_log(rng, 1, 512), most // (hi * hi * H * D)))
        return dict(op=op, B=B, lo=rng.choice([0, 1, (hi + 1) // 2, hi]), hi=hi, H=H, KV=KV, D=D, dtype=dtype,
                    mask=rng.choice(["text", "text", "causal", "prefix"]), cap=rng.choice([0.0, 0.0, 20.0]), bias=rng.random() < 0.5,
                    fused=rng.random() < 0.5, train=rng.random() < 0.75)
    if op == "gated":
        d, F = rng.choice([64, 77, 128, 256, 384, 768, 1024]), _log(rng, 16, 4096)
        most = 16384 * 1024 * 4096 // (2 if dtype != "fp32" else 20)
        return dict(op=op, N=max(1, min(_log(rng, 1, 16384), most // (d * F))), d=d, F=F, dtype=dtype,
                    act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]), train=rng.random() < 0.75)
    return dict(op=op, layers=rng.randint(0, 12), d=rng.choice([96, 256, 384, 513, 768, 1024]), V=_log(rng, 100, 32000),
                grads=dtype, copies=rng.choice(["", "fp16", "bf16"]), bits=rng.choice([8, 32]), clips=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _lengths(c):
    """The texts' lengths: of the case alone, so that its work is known without a seed."""
    rng = random.Random(c["B"] * 1000003 + c["hi"])
    lens = [c["hi"]] + [rng.randint(c["lo"], c["hi"]) for _ in range(c["B"] - 1)]
    if c["B"] >= 16:
        lens[c["B"] // 2] = 0  # a text that came out empty
    return lens


def _behind(c):
    return 5 if c["B"] > 1 else 0  # rows behind the last text: a batch brought to a whole size


def _prefixes(c):
    """How many of its first tokens each text sees as a whole, before it goes on causally."""
    lens = _lengths(c)
    return [0 if c["mask"] == "causal" else n // 3 if c["mask"] == "prefix" else n for n in lens]


def _shapes(layers, d, V):
    """The parameters of an encoder of `layers` layers with gated feed-forward blocks: embeddings,
    attention, the block's three matrices, norms, and the projection to 128 dimensions."""
    f = (8 * d // 3 + 63) // 64 * 64
    shapes = [(V, d), (d,)] if layers else [(V, d)]
    for _ in range(layers):
        shapes += [(d, d)] * 4 + [(f, d), (f, d), (d, f), (d,), (d,)]
    return shapes + [(128, d), (128,)]


def _places(shapes):
    """Where each tensor begins in a flat buffer, and the buffer's size."""
    at, places = 0, []
    for s in shapes:
        places.append(at)
        at += (math.prod(s) + BLOCK - 1) // BLOCK * BLOCK
    return places, at


def _views(flat, shapes):
    return [flat[a:a + math.prod(s)].view(s) for a, s in zip(_places(shapes)[0], shapes)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if c["op"] == "attention":
        dt, H, KV, D = DTYPES[c["dtype"]], c["H"], c["KV"], c["D"]
        lens = _lengths(c)
        T = sum(lens) + _behind(c)
        offsets = torch.tensor([0] + lens, device=DEV).cumsum(0)
        G = normal(T, H, D)
        # queries look for a few of their text's keys: scores spread over several units
        if c["fused"]:
            x = normal(T, H + 2 * KV, D)
            x[:, :H] *= 1.5
            q, k, v = x.to(dt).split([H, KV, KV], 1)
        else:
            q, k, v = (1.5 * normal(T, H, D)).to(dt), normal(T, KV, D).to(dt), normal(T, KV, D).to(dt)
        if T:
            v[offsets[-1]:] = math.nan  # what nothing may read
        if c["train"]:
            q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        return dict(c=c, q=q, k=k, v=v, offsets=offsets, G=G.to(dt), cap=c["cap"] or None,
                    prefix=None if c["mask"] == "text" else torch.tensor(_prefixes(c), device=DEV),
                    slopes=torch.exp2(-8 * torch.arange(1, H + 1, device=DEV) / H) if c["bias"] else None)
    if c["op"] == "gated":
        dt, N, d, F = DTYPES[c["dtype"]], c["N"], c["d"], c["F"]
        x = normal(N, d).to(dt)  # normalised hidden states
        wg, wu = (normal(F, d) * (1.5 / math.sqrt(d))).to(dt), (normal(F, d) / math.sqrt(d)).to(dt)
        if c["train"]:
            x, wg, wu = (t.requires_grad_(True) for t in (x, wg, wu))
        return dict(c=c, x=x, wg=wg, wu=wu, G=normal(N, F).to(dt))
    shapes = _shapes(c["layers"], c["d"], c["V"])
    places, size = _places(shapes)
    gt = DTYPES[c["grads"]]
    here = torch.zeros(size, dtype=torch.bool, device=DEV)
    std = torch.zeros(size, device=DEV)
    for i, (a, s) in enumerate(zip(places, shapes)):
        here[a:a + math.prod(s)] = True
        std[a:a + math.prod(s)] = 1e-3 * (1 + i % 7)
    grads = (std * normal(size)).to(gt)
    flat = torch.where(here, 0.02 * normal(size), torch.zeros(size, device=DEV))
    s = dict(c=c, flat=flat, grads=grads, params=_views(flat, shapes), glist=_views(grads, shapes), lr=1e-3,
             steps=torch.full((len(shapes),), 500, device=DEV), copy=None, copies=None, most=None)
    if c["copies"]:
        s["copy"] = torch.zeros(size, dtype=DTYPES[c["copies"]], device=DEV)
        s["copies"] = _views(s["copy"], shapes)
    if c["clips"]:
        s["most"] = 0.3 * math.sqrt(float((std.double() ** 2).sum()))
    if c["bits"] == 32:
        s["m"], s["v"] = 0.3 * std * normal(size), std * std * (0.3 + torch.rand(size, generator=g, device=DEV))
        return s
    # 8 bits: any codes of the upper octaves, with the exponents that the gradients' size gives
    top = torch.log2(std.view(-1, BLOCK)[:, :1].clamp(min=1e-6))[:, 0]
    m = torch.randint(60, 112, (size,), generator=g, device=DEV) + 128 * torch.randint(0, 2, (size,), generator=g, device=DEV)
    v = torch.randint(200, 240, (size,), generator=g, device=DEV)
    none = torch.zeros((), dtype=torch.int64, device=DEV)
    s["m"], s["v"] = torch.where(here, m, none).to(torch.uint8), torch.where(here, v, none).to(torch.uint8)
    s["m_exp"], s["v_exp"] = (127 + top).to(torch.uint8), (127 + 2 * top).to(torch.uint8)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["c"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        if c["op"] == "attention":
            return _plain_attention(s, c)
        if c["op"] == "gated":
            return _plain_gated(s, c)
        return _plain_adamw(s, c)


def _run_own(s, c):
    import tilemaxsim_amd as tms
    if c["op"] == "attention":
        out = tms.packed_attention(s["q"], s["k"], s["v"], s["offsets"], prefix=s["prefix"], cap=s["cap"], slopes=s["slopes"])
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["G"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "gated":
        h = tms.gated_linear(s["x"], s["wg"], s["wu"], activation=c["act"])
        if not c["train"]:
            return {"h": h}
        dx, dwg, dwu = torch.autograd.grad(h, (s["x"], s["wg"], s["wu"]), s["G"])
        return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}
    if "state" not in s:  # a program keeps it from step to step
        s["state"] = tms.AdamWState(s["params"], bits=c["bits"])
        s["state"].load_state_dict({"steps": s["steps"], **{k: s[k] for k in ("m", "v", "m_exp", "v_exp") if k in s}})
    norm = tms.grad_norm(s["glist"]) if c["clips"] else None
    tms.adamw_(s["params"], s["glist"], s["state"], lr=s["lr"], norm=norm, max_norm=s["most"], copies=s["copies"])
    m, v = s["state"].moments()
    return {"params": s["flat"], "m": m, "v": v, **({"copies": s["copy"]} if c["copies"] else {})}


def _visible(c, offsets, prefix, L):
    """Rows of the padded texts (B, L) in the packed tensors, which exist, and (B, L, L) what they see."""
    lens = offsets[1:] - offsets[:-1]
    place = torch.arange(L, device=DEV)
    real = place < lens[:, None]
    rows = torch.where(real, offsets[:-1, None] + place, torch.zeros_like(real, dtype=torch.int64))
    sees = (real[:, :, None] & real[:, None, :])
    if prefix is not None:
        sees = sees & ((place[None, :] <= place[:, None])[None] | (place < prefix[:, None])[:, None, :])
    return rows, real, sees


def _padded(x, rows, real, heads):
    """(T, h, D) -> (B, heads, L, D) in fp32, shared heads repeated, zeros where no token is."""
    x = torch.where(real[:, :, None, None], x[rows].float(), torch.zeros((), device=DEV))
    return x.transpose(1, 2).repeat_interleave(heads // x.shape[2], 1).contiguous()


def _packed(x, rows, real, like):
    """The reverse; repeated heads' values are added up."""
    B, H, L, D = x.shape
    kv = like.shape[1]
    out = torch.zeros(like.shape, device=DEV)
    out[rows[real]] = x.view(B, kv, H // kv, L, D).sum(2).transpose(1, 2)[real]
    return out.to(like.dtype)


def _plain_attention(s, c):
    H, D = c["H"], c["D"]
    scale = 1 / math.sqrt(D)
    L = max(_lengths(c))
    rows, real, sees = _visible(c, s["offsets"], s["prefix"], L)
    q, k, v = (_padded(s[n], rows, real, H) for n in "qkv")
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    t = None
    if s["cap"]:
        t = torch.tanh(x / s["cap"])
        x = s["cap"] * t
    if s["slopes"] is not None:
        place = torch.arange(L, device=DEV)
        x = x - s["slopes"][:, None, None] * (place[:, None] - place).abs()
    x = x.masked_fill(~sees[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p, v)
    if not c["train"]:
        return {"out": _packed(out, rows, real, s["q"])}
    G = _padded(s["G"], rows, real, H)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), G)
    ds = p * (torch.matmul(G, v.transpose(2, 3).contiguous()) - (G * out).sum(-1, keepdim=True)) * scale
    if t is not None:
        ds = ds * (1 - t * t)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return {"out": _packed(out, rows, real, s["q"]), "dq": _packed(dq, rows, real, s["q"]), "dk": _packed(dk, rows, real, s["k"]),
            "dv": _packed(dv, rows, real, s["v"])}


def _act(g, kind):
    """An activation's values and its derivative's."""
    if kind == "silu":
        y = 1 / (1 + torch.exp(-g))
        return g * y, y * (1 + g * (1 - y))
    if kind == "gelu":
        y = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * y, y + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)
    t = torch.tanh(u)
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


def _plain_gated(s, c):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, c["act"])
    h = (a * u).to(s["x"].dtype)
    if not c["train"]:
        return {"h": h}
    G = s["G"].float()
    dg, du = G * u * da, G * a
    dt = s["x"].dtype
    return {"h": h, "dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt)}


B1, B2, EPS, DECAY = 0.9, 0.999, 1e-8, 0.01


def _mix(x):
    """32 mixed bits of each 32-bit number (as int64)."""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _decode(codes, exps, octaves, magnitude):
    """The numbers that 8-bit codes stand for: three bits below the leading one, `octaves` octaves below the block's exponent."""
    c = codes.long()
    base = (exps.long() - octaves).repeat_interleave(BLOCK) * 8
    bits = ((c & magnitude) + base).clamp(min=0) << 20
    x = bits.to(torch.int32).view(torch.float32)
    x = torch.where((c & magnitude) == 0, torch.zeros_like(x), x)
    return torch.where(c > magnitude, -x, x)


def _encode(x, dither, octaves, magnitude, keep):
    """8-bit codes of x and its blocks' exponents: `dither` (16 bits) is added below the last bit kept
    before the rest is cut off. `keep`: what is below the range becomes the smallest number;
    otherwise that, or zero, as the dither says."""
    a = x.abs()
    bits = a.view(torch.int32).long()
    top = (bits >> 23).view(-1, BLOCK).amax(1)
    base = (top - octaves).repeat_interleave(BLOCK) * 8
    code = ((bits + (dither << 4)) >> 20) - base
    least = ((base + 1).clamp(min=0) << 20).to(torch.int32).view(torch.float32)
    under = torch.ones_like(code) if keep else (a >= dither.float() / 65536 * least).long()
    code = torch.where(code < 1, under, code)
    code = torch.where(a == 0, torch.zeros_like(code), code)
    code = torch.where(x < 0, code + magnitude + 1, code)
    return code.to(torch.uint8), top.to(torch.uint8)


def _plain_adamw(s, c):
    g = s["grads"].float()
    if c["clips"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * torch.clamp(torch.full_like(norm, s["most"]) / (norm + 1e-6), max=1.0)
    s["steps"] += 1
    step = s["steps"][0].double()  # of all tensors alike here
    small = c["bits"] == 8
    m, v = (_decode(s["m"], s["m_exp"], 14, 127), _decode(s["v"], s["v_exp"], 30, 255)) if small else (s["m"], s["v"])
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    to = (s["lr"] / (1 - B1 ** step)).float()
    root = (1 / torch.sqrt(1 - B2 ** step)).float()
    s["flat"].copy_((1 - s["lr"] * DECAY) * s["flat"] - to * m / (v.sqrt() * root + EPS))
    if small:
        at = torch.arange(g.numel(), device=DEV)
        mixed = _mix((at & 0xffffffff) ^ _mix((s["steps"][0] + (at >> 32) * 0x9e3779b1) & 0xffffffff))
        s["m"], s["m_exp"] = _encode(m, mixed & 0xffff, 14, 127, False)
        s["v"], s["v_exp"] = _encode(v, mixed >> 16, 30, 255, True)
        m, v = _decode(s["m"], s["m_exp"], 14, 127), _decode(s["v"], s["v_exp"], 30, 255)
    else:
        s["m"], s["v"] = m, v
    out = {"params": s["flat"], "m": m, "v": v}
    if c["copies"]:
        s["copy"].copy_(s["flat"])
        out["copies"] = s["copy"]
    return out


def work(case):
    c = case
    if c["op"] == "attention":
        size, lens = DTYPES[c["dtype"]].itemsize, _lengths(c)
        T, H, KV, D = sum(lens), c["H"], c["KV"], c["D"]
        # token i of a text sees max(i + 1, prefix) of its tokens
        pairs = sum(n * (n + 1) // 2 + p * (p - 1) // 2 if p else n * (n + 1) // 2 for n, p in zip(lens, _prefixes(c)))
        qkv = T * (H + 2 * KV) * D * size
        if not c["train"]:
            return {"bytes": qkv + T * H * D * size + 8 * (c["B"] + 1), "flops": 4 * pairs * H * D}
        return {"bytes": 2 * qkv + 2 * T * H * D * size + 8 * (c["B"] + 1), "flops": 12 * pairs * H * D}
    if c["op"] == "gated":
        size, N, d, F = DTYPES[c["dtype"]].itemsize, c["N"], c["d"], c["F"]
        operands = (N * d + 2 * F * d) * size
        if not c["train"]:
            return {"bytes": operands + N * F * size, "flops": 4 * N * F * d}
        return {"bytes": 2 * operands + 2 * N * F * size, "flops": 12 * N * F * d}
    n = sum(math.prod(x) for x in _shapes(c["layers"], c["d"], c["V"]))
    states = 16 if c["bits"] == 32 else 4 + 4 / BLOCK + 8  # 8 bits: the values are written out beside them
    return {"bytes": int(n * (8 + states + DTYPES[c["grads"]].itemsize + (2 if c["copies"] else 0))), "flops": 16 * n}


# ---------------------------------------------------------------- 64 bits

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s, case)
    if case["op"] == "gated":
        return _exact_gated(s, case)
    return _exact_adamw(s, case)


def _exact_attention(s, c):
    H, D = c["H"], c["D"]
    many = H // c["KV"]
    q, k, v, G = (s[n].detach().double() for n in ("q", "k", "v", "G"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = 0
    for n, p in zip(_lengths(c), _prefixes(c)):  # one text at a time, one head at a time
        i = torch.arange(n, device=DEV)
        hidden = (i[None, :] > i[:, None]) & (i[None, :] >= p)
        far = (i[:, None] - i[None, :]).abs().double()
        for h in range(H if n else 0):
            a, b = slice(at, at + n), h // many
            z = q[a, h] @ k[a, b].t() / math.sqrt(D)
            slope = torch.ones_like(z)
            if s["cap"]:
                t = torch.tanh(z / s["cap"])
                z, slope = s["cap"] * t, 1 - t ** 2
            if s["slopes"] is not None:
                z = z - float(s["slopes"][h]) * far
            w = torch.softmax(z.masked_fill(hidden, -math.inf), 1)
            out[a, h] = w @ v[a, b]
            if c["train"]:
                dw = G[a, h] @ v[a, b].t()
                dz = w * (dw - (w * dw).sum(1, keepdim=True)) * slope / math.sqrt(D)
                dq[a, h] = dz @ k[a, b]
                dk[a, b] += dz.t() @ q[a, h]
                dv[a, b] += w.t() @ G[a, h]
        at += n
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"out": out}


def _exact_gated(s, c):
    x, wg, wu, G = (s[n].detach().double() for n in ("x", "wg", "wu", "G"))
    g = (x @ wg.t()).requires_grad_(True)
    u = x @ wu.t()
    with torch.enable_grad():
        if c["act"] == "silu":
            a = torch.nn.functional.silu(g)
        else:
            a = torch.nn.functional.gelu(g, approximate="tanh" if c["act"] == "gelu_tanh" else "none")
        da = torch.autograd.grad(a.sum(), g)[0]
    a = a.detach()
    if not c["train"]:
        return {"h": a * u}
    dg, du = G * u * da, G * a
    return {"h": a * u, "dx": dg @ wg + du @ wu, "dwg": dg.t() @ x, "dwu": du.t() @ x}


def _exact_adamw(s, c):
    g = s["grads"].double()
    if c["clips"]:
        g = g * min(1.0, s["most"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    if c["bits"] == 8:
        def number(codes, exps, octaves, bits):  # (1 + last three bits / 8) times a power of two
            k = codes.long() % (1 << bits)
            e = exps.long().repeat_interleave(BLOCK) - octaves - 127 + k // 8
            x = torch.ldexp(1 + (k % 8).double() / 8, e.double())
            return torch.where(k == 0, torch.zeros_like(x), torch.where(codes.long() >= 1 << bits, -x, x))
        m, v = number(s["m"], s["m_exp"], 14, 7), number(s["v"], s["v_exp"], 30, 8)
    else:
        m, v = s["m"].double(), s["v"].double()
    t = int(s["steps"][0]) + 1
    m, v = m.lerp(g, 1 - B1), v.lerp(g * g, 1 - B2)
    p = s["flat"].double()
    p = p - s["lr"] * (DECAY * p + (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS))
    out = {"params": p, "m": m, "v": v}
    if c["bits"] == 8:
        out["m"] = out["v"] = None  # the rounding to 8 bits goes by thresholds: no value in 64 bits
    if c["copies"]:
        out["copies"] = p
    return out
