"""The training operators' cases: MaxSim of query and document batches with its gradients,
softmax cross entropy over a large vocabulary from the hidden states and the vocabulary's
weights, and the global gradient norm with clipping, from calls where latency counts to the
largest a training step makes.

``own`` False: the plain forms (elementary torch operations in fp32, rounded once at the
end); True: the package's calls. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

DEV = torch.device("cuda", 0)

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
IGNORE = -100


def listed():
    return [
        # MaxSim. Latency: the smallest batch whose loss has a negative, two queries of 32
        # tokens and two documents of 180 (the token counts of the repository's benchmark).
        dict(name="maxsim train 2x2", op="maxsim", own_docs=False, nQ=2, B=2, Nq=32, Nd=180, d=128, dtype="bf16", train=True),
        # Distillation: 32 queries, each with its own 8 documents, of odd token counts.
        dict(name="maxsim train 32 own 8", op="maxsim", own_docs=True, nQ=32, B=8, Nq=29, Nd=171, d=128, dtype="fp16", train=True),
        # Validation: scores without a gradient, odd sizes, the narrower embedding.
        dict(name="maxsim scores 37x501", op="maxsim", own_docs=False, nQ=37, B=501, Nq=32, Nd=300, d=96, dtype="bf16", train=False),
        # In-batch negatives: 64 queries against the 64 documents of each of them.
        dict(name="maxsim train 64x4096", op="maxsim", own_docs=False, nQ=64, B=4096, Nq=32, Nd=180, d=128, dtype="fp16", train=True),
        # Cross entropy. Latency: the loss of one token (a probe of a model while it is served).
        dict(name="ce 1 token", op="ce", N=1, V=32000, d=768, dtype="bf16", train=False, contrastive=False, reduction="mean"),
        # One vector a text: 1024 queries against 16,384 passages, every other one a negative.
        dict(name="ce contrastive 1024x16384", op="ce", N=1024, V=16384, d=128, dtype="fp16", train=True, contrastive=True, reduction="mean"),
        # Masked tokens of a batch against a word-piece vocabulary, odd counts of both.
        dict(name="ce 1229x30011", op="ce", N=1229, V=30011, d=768, dtype="bf16", train=True, contrastive=False, reduction="mean"),
        # The same loss in fp32, weighted by row.
        dict(name="ce fp32 500x8000", op="ce", N=500, V=8000, d=256, dtype="fp32", train=True, contrastive=False, reduction="none"),
        # A whole batch of tokens against a large multilingual vocabulary.
        dict(name="ce 8192x131072", op="ce", N=8192, V=131072, d=768, dtype="bf16", train=True, contrastive=False, reduction="mean"),
        # Clipping. Latency: the parameters of a projection head alone.
        dict(name="clip head", op="clip", layers=0, d=768, V=128, dtype="fp32", out="fp32", clips=True),
        # An encoder's bf16 gradients into the fp32 ones that the optimizer reads, odd vocabulary.
        dict(name="clip encoder bf16", op="clip", layers=12, d=768, V=30011, dtype="bf16", out="fp32", clips=True),
        # A larger encoder in fp32 throughout.
        dict(name="clip encoder fp32", op="clip", layers=24, d=1024, V=32000, dtype="fp32", out="fp32", clips=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["maxsim", "maxsim", "ce", "ce", "clip"])
    if op == "maxsim":
        own_docs = rng.random() < 0.35
        dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
        nQ, Nq, Nd = _log(rng, 1, 64), rng.randint(1, 64), _log(rng, 1, 512)
        d = rng.choice([32, 64, 77, 96, 128, 128, 128])
        pairs = 64 * 4096 * 32 * 180 // 2
        if dtype == "fp32":
            pairs //= 6
        most = pairs // (nQ * Nq * Nd)
        B = max(1, min(_log(rng, 1, 4096), most))
        if own_docs:
            B = min(B, 64)
        return dict(op=op, own_docs=own_docs, nQ=nQ, B=B, Nq=Nq, Nd=Nd, d=d, dtype=dtype, train=rng.random() < 0.75)
    if op == "ce":
        dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "bf16", "fp32"])
        N, V = _log(rng, 1, 8192), _log(rng, 2, 131072)
        d = rng.choice([32, 77, 96, 128, 128, 256, 384, 512, 768, 768])
        most = 8192 * 131072 * 768 // (6 if dtype != "fp32" else 60)
        V = max(2, min(V, most // (N * d)))
        return dict(op=op, N=N, V=V, d=d, dtype=dtype, train=rng.random() < 0.75, contrastive=rng.random() < 0.4,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]))
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return dict(op=op, layers=rng.randint(0, 12), d=rng.choice([96, 256, 384, 513, 768, 1024]), V=_log(rng, 100, 32000),
                dtype=dtype, out=rng.choice(["fp32", dtype]), clips=rng.random() < 0.8)


# ---------------------------------------------------------------- inputs

def _units(g, *shape):
    """Unit token embeddings on the grid of 2^-11. Dot products of such vectors are exact in
    fp32 whatever the order of the sum, so the position of a maximum is the same for all."""
    x = torch.randn(shape, generator=g, device=DEV)
    x /= x.square().sum(-1, keepdim=True).sqrt()
    return (x * 2048).round_().div_(2048)


def _shapes(layers, d, V):
    """The parameters of an encoder of `layers` layers: embeddings, attention, feed-forward,
    norms, and the projection to 128 dimensions."""
    shapes = [(V, d), (512, d), (d,), (d,)] if layers else [(V, d)]
    for _ in range(layers):
        shapes += [(d, d), (d,)] * 4 + [(4 * d, d), (4 * d,), (d, 4 * d), (d,)] + [(d,)] * 4
    return shapes + [(128, d), (128,)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    dt = DTYPES[c["dtype"]]
    if c["op"] == "maxsim":
        docs = (c["nQ"], c["B"]) if c["own_docs"] else (c["B"],)
        n = math.prod(docs)
        Q = _units(g, c["nQ"], c["Nq"], c["d"]).to(dt)
        D = _units(g, n, c["Nd"], c["d"])
        # relevant documents repeat some of their query's tokens
        rel = torch.arange(n, device=DEV)
        rel = rel // c["B"] if c["own_docs"] else rel % c["nQ"]
        at = torch.randint(0, c["Nd"], (n, 1), generator=g, device=DEV) + torch.arange(min(4, c["Nq"], c["Nd"]), device=DEV)
        at %= c["Nd"]
        D[torch.arange(n, device=DEV)[:, None], at] = Q[rel[:, None], torch.arange(at.shape[1], device=DEV)].float()
        D = D.to(dt)
        # padded batches: documents end anywhere; a text that came out empty
        lens = torch.randint((c["Nd"] + 2) // 3, c["Nd"] + 1, (n,), generator=g, device=DEV)
        if n >= 16:
            lens[n // 2] = 0
        mask = torch.arange(c["Nd"], device=DEV) < lens[:, None]
        qlens = torch.randint((c["Nq"] + 1) // 2, c["Nq"] + 1, (c["nQ"],), generator=g, device=DEV)
        qmask = torch.arange(c["Nq"], device=DEV) < qlens[:, None]
        # what a contrastive loss sends back: softmax over the documents less the relevant one
        G = torch.softmax(2 * torch.randn(c["nQ"], c["B"], generator=g, device=DEV), -1)
        G[torch.arange(c["nQ"], device=DEV), torch.arange(c["nQ"], device=DEV) % c["B"]] -= 1
        G /= c["nQ"]
        D, mask = D.view(*docs, c["Nd"], c["d"]), mask.view(*docs, c["Nd"])
        if c["train"]:
            Q.requires_grad_(True)
            D.requires_grad_(True)
        return dict(c=c, Q=Q, D=D, mask=mask, qmask=qmask, G=G)
    if c["op"] == "ce":
        N, V, d = c["N"], c["V"], c["d"]
        W = torch.randn(V, d, generator=g, device=DEV)
        t = torch.randint(0, V, (N,), generator=g, device=DEV)
        if c["contrastive"]:  # unit vectors; a query lies near its passage
            W /= W.square().sum(-1, keepdim=True).sqrt()
            H = W[t] + 1.5 / math.sqrt(d) * torch.randn(N, d, generator=g, device=DEV)
            H /= H.square().sum(-1, keepdim=True).sqrt()
            scale = 20.0
        else:  # normalised hidden states; some rows are padding
            W *= 2 / math.sqrt(d)
            H = torch.randn(N, d, generator=g, device=DEV)
            scale = 1.0
            if N > 1:
                t[torch.rand(N, generator=g, device=DEV) < 0.1] = IGNORE
                t[0] = int(seed) % V
        G = torch.rand(N, generator=g, device=DEV) + 0.5 if c["reduction"] == "none" else torch.ones((), device=DEV)
        H, W = H.to(dt), W.to(dt)
        if c["train"]:
            H.requires_grad_(True)
            W.requires_grad_(True)
        return dict(c=c, H=H, W=W, t=t, G=G, scale=scale)
    grads, total = [], 0.0
    for i, s in enumerate(_shapes(c["layers"], c["d"], c["V"])):
        std = 1e-3 * (1 + i % 7)
        grads.append((std * torch.randn(s, generator=g, device=DEV)).to(dt))
        total += std * std * math.prod(s)
    # the optimizer's gradients: one flat buffer, each parameter's a view of it
    flat = torch.zeros(sum(x.numel() for x in grads), dtype=DTYPES[c["out"]], device=DEV)
    out = [o.view_as(x) for o, x in zip(flat.split([x.numel() for x in grads]), grads)]
    return dict(c=c, grads=grads, out=out, flat=flat, most=math.sqrt(total) * (0.3 if c["clips"] else 2.0))


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["c"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        if c["op"] == "maxsim":
            return _plain_maxsim(s, c)
        if c["op"] == "ce":
            return _plain_ce(s, c)
        return _plain_clip(s)


def _run_own(s, c):
    import tilemaxsim_amd as tms
    if c["op"] == "maxsim":
        scores = tms.maxsim_pairs(s["Q"], s["D"], s["mask"], s["qmask"])
        if not c["train"]:
            return {"scores": scores}
        dQ, dD = torch.autograd.grad(scores, (s["Q"], s["D"]), s["G"])
        return {"scores": scores.detach(), "dQ": dQ, "dD": dD}
    if c["op"] == "ce":
        loss = tms.linear_cross_entropy(s["H"], s["W"], s["t"], scale=s["scale"], ignore_index=IGNORE, reduction=c["reduction"])
        if not c["train"]:
            return {"loss": loss}
        dH, dW = torch.autograd.grad(loss, (s["H"], s["W"]), s["G"])
        return {"loss": loss.detach(), "dH": dH, "dW": dW}
    return {"norm": tms.clip_grad_norm_(s["grads"], s["most"], out=s["out"]), "out": s["flat"]}


def _plain_maxsim(s, c):
    Q, D, mask, qmask = s["Q"].float(), s["D"].float(), s["mask"], s["qmask"]
    nQ, Nq, d = Q.shape
    Nd = c["Nd"]
    if c["own_docs"]:
        B = c["B"]
        sims = torch.matmul(Q, D.view(nQ, B * Nd, d).transpose(1, 2).contiguous()).view(nQ, Nq, B, Nd)
        sims = sims.masked_fill(~mask.view(nQ, 1, B, Nd), -math.inf)
    else:
        B = c["B"]
        sims = (Q.view(nQ * Nq, d) @ D.view(B * Nd, d).t()).view(nQ, Nq, B, Nd)
        sims = sims.masked_fill(~mask.view(1, 1, B, Nd), -math.inf)
    top = sims.amax(-1)
    empty = ~mask.any(-1)
    empty = empty if c["own_docs"] else empty[None, :].expand(nQ, B)
    scores = torch.where(qmask[:, :, None], top, torch.zeros_like(top)).sum(1)
    scores = torch.where(empty, torch.full_like(scores, -math.inf), scores)
    if not c["train"]:
        return {"scores": scores}
    # the first of equal maxima takes the gradient
    place = torch.arange(Nd, device=DEV, dtype=torch.int32)
    first = torch.where(sims == top[..., None], place, Nd).amin(-1, keepdim=True)
    g = torch.where(empty, torch.zeros_like(s["G"]), s["G"])[:, None, :] * qmask[:, :, None]
    hot = torch.where(place == first, g[..., None], torch.zeros_like(g[..., None]))
    if c["own_docs"]:
        hot = hot.view(nQ, Nq, B * Nd)
        dQ = torch.matmul(hot, D.view(nQ, B * Nd, d))
        dD = torch.matmul(hot.transpose(1, 2).contiguous(), Q).view(nQ, B, Nd, d)
    else:
        hot = hot.view(nQ * Nq, B * Nd)
        dQ = (hot @ D.view(B * Nd, d)).view(nQ, Nq, d)
        dD = (hot.t() @ Q.view(nQ * Nq, d)).view(B, Nd, d)
    return {"scores": scores, "dQ": dQ.to(s["Q"].dtype), "dD": dD.to(s["D"].dtype)}


def _plain_ce(s, c):
    H, W, t = s["H"].float(), s["W"].float(), s["t"]
    N = H.shape[0]
    logits = s["scale"] * (H @ W.t())
    top = logits.amax(1, keepdim=True)
    z = torch.exp(logits - top).sum(1, keepdim=True)
    kept = t != IGNORE
    at = torch.where(kept, t, torch.zeros_like(t))[:, None]
    row = torch.where(kept, (top + torch.log(z) - logits.gather(1, at))[:, 0], torch.zeros_like(z[:, 0]))
    if c["reduction"] == "none":
        loss, g = row, s["G"] * kept
    elif c["reduction"] == "sum":
        loss, g = row.sum(), s["G"] * kept
    else:
        loss, g = row.sum() / kept.sum(), s["G"] * kept / kept.sum()
    if not c["train"]:
        return {"loss": loss}
    P = torch.exp(logits - top) / z
    P[torch.arange(N, device=DEV), at[:, 0]] -= 1
    P *= (g * s["scale"])[:, None]
    return {"loss": loss, "dH": (P @ W).to(s["H"].dtype), "dW": (P.t() @ H).to(s["W"].dtype)}


def _plain_clip(s):
    parts = torch.stack([x.float().square().sum() for x in s["grads"]])
    norm = parts.sum().sqrt()
    coef = torch.clamp(s["most"] / (norm + 1e-6), max=1.0)
    for x, o in zip(s["grads"], s["out"]):
        o.copy_(x.float() * coef)
    return {"norm": norm, "out": s["flat"]}


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "maxsim":
        docs = c["B"] * (c["nQ"] if c["own_docs"] else 1)
        pairs = c["nQ"] * c["B"]
        inputs = (c["nQ"] * c["Nq"] + docs * c["Nd"]) * c["d"] * size + docs * c["Nd"] + c["nQ"] * c["Nq"]
        flops = 2 * pairs * c["Nq"] * c["Nd"] * c["d"]
        if not c["train"]:
            return {"bytes": inputs + 4 * pairs, "flops": flops}
        # the gradients add one document token to a query token's and the reverse, for each maximum
        grads = (c["nQ"] * c["Nq"] + docs * c["Nd"]) * c["d"] * size
        return {"bytes": inputs + grads + 8 * pairs, "flops": flops + 4 * pairs * c["Nq"] * c["d"]}
    if c["op"] == "ce":
        N, V, d = c["N"], c["V"], c["d"]
        nbytes = (N + V) * d * size + 8 * N + 4 * (N if c["reduction"] == "none" else 1)
        if not c["train"]:
            return {"bytes": nbytes, "flops": 2 * N * V * d}
        return {"bytes": nbytes + (N + V) * d * size, "flops": 6 * N * V * d}
    n = sum(math.prod(x) for x in _shapes(c["layers"], c["d"], c["V"]))
    return {"bytes": n * (size + DTYPES[c["out"]].itemsize), "flops": 3 * n}


# ---------------------------------------------------------------- 64 bits

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "maxsim":
        return _exact_maxsim(s, c)
    if c["op"] == "ce":
        return _exact_ce(s, c)
    norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in s["grads"]))
    k = min(1.0, s["most"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "out": torch.cat([x.double().flatten() * k for x in s["grads"]])}


def _exact_maxsim(s, c):
    Q, D = s["Q"].double(), s["D"].double()
    nQ, Nq, d = Q.shape
    scores = torch.zeros(nQ, c["B"], dtype=torch.float64, device=DEV)
    dQ, dD = torch.zeros_like(Q), torch.zeros_like(D)
    for q in range(nQ):  # one query at a time against its documents
        docs, live = (D[q], s["mask"][q]) if c["own_docs"] else (D, s["mask"])
        some = live.any(1)
        sim = docs @ Q[q].t()  # (B, Nd, Nq)
        sim.masked_fill_(~live[:, :, None], -math.inf)
        order = torch.sort(sim, dim=1, descending=True, stable=True)
        best, which = order.values[:, 0], order.indices[:, 0]  # (B, Nq)
        best = torch.where(s["qmask"][q][None, :], best, torch.zeros_like(best))
        scores[q] = torch.where(some, best.sum(1), torch.full_like(best[:, 0], -math.inf))
        if not c["train"]:
            continue
        w = (s["G"][q].double() * some)[:, None] * s["qmask"][q][None, :].double()  # (B, Nq)
        rows = torch.gather(docs, 1, which[:, :, None].expand(-1, -1, d))
        dQ[q] = (rows * w[:, :, None]).sum(0)
        into = dD[q] if c["own_docs"] else dD
        into.scatter_add_(1, which[:, :, None].expand(-1, -1, d), w[:, :, None] * Q[q][None])
    return {"scores": scores, "dQ": dQ, "dD": dD} if c["train"] else {"scores": scores}


def _exact_ce(s, c):
    H, W, t = s["H"].double(), s["W"].double(), s["t"]
    N = H.shape[0]
    count = int((t != IGNORE).sum())
    rows = torch.zeros(N, dtype=torch.float64, device=DEV)
    dH, dW = torch.zeros_like(H), torch.zeros_like(W)
    for a in range(0, N, 1024):  # some rows at a time
        h, tt = H[a:a + 1024], t[a:a + 1024]
        live = (tt != IGNORE).double()
        logp = torch.log_softmax(s["scale"] * h @ W.t(), dim=1)
        rows[a:a + 1024] = -logp.gather(1, tt.clamp(min=0)[:, None])[:, 0] * live
        if not c["train"]:
            continue
        up = s["G"].double() / (count if c["reduction"] == "mean" else 1)
        up = (up[a:a + 1024] if c["reduction"] == "none" else up.expand(len(tt))) * live
        p = logp.exp_()
        p.scatter_add_(1, tt.clamp(min=0)[:, None], torch.full((len(tt), 1), -1.0, dtype=torch.float64, device=DEV))
        p *= (up * s["scale"])[:, None]
        dH[a:a + 1024] = p @ W
        dW += p.t() @ h
    loss = rows if c["reduction"] == "none" else rows.sum() / (count if c["reduction"] == "mean" else 1)
    return {"loss": loss, "dH": dH, "dW": dW} if c["train"] else {"loss": loss}
