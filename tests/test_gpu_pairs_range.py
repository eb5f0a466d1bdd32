"""``maxsim_pairs`` at the ends of its range: the longest documents, the most documents, queries
with no documents of their own; and fp32 embeddings whose 24 bits all count."""
import math

import numpy as np
import pytest
import torch
from test_gpu_pairs import DT, ROUND, TINY, _grid

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype,Nd", [("bf16", 65535), ("fp16", 65281), ("bf16", 65280), ("fp32", 65535), ("fp32", 65409)])
def test_longest_documents(cuda, dtype, Nd):
    """The query gradient that shares documents, whose last stage ends where the mark of a
    maximum without a token would lie: masked query tokens and a document without a real token
    give exactly nothing, with NaN at masked document tokens."""
    import tilemaxsim_amd as tms
    nQ, Nq, B, d = 512, 2, 17, 32
    assert nQ * B > 8192
    rng = np.random.default_rng(Nd)
    dt = DT[dtype]
    Q, D = _grid(rng, nQ, Nq, d).to(dt).cuda(), _grid(rng, B, Nd, d).to(dt).cuda()
    qmask = torch.from_numpy(rng.random((nQ, Nq)) < 0.7).cuda()
    dmask = torch.from_numpy(rng.random((B, Nd)) < 0.9).cuda()
    dmask[3] = False
    step = 128 if dtype == "fp32" else 256
    for last in range(step - 1, Nd, step):  # the last token of every stage
        dmask[:, last] = False
    D[~dmask] = math.nan
    G = torch.from_numpy(rng.standard_normal((nQ, B)).astype(np.float32)).cuda()
    print(f"pairs of long documents {dtype} Nd={Nd}", flush=True)
    Qg, Dg = Q.clone().requires_grad_(True), D.clone().requires_grad_(True)
    s = tms.maxsim_pairs(Qg, Dg, dmask, qmask)
    gQ, gD = torch.autograd.grad(s, (Qg, Dg), G)
    q = Q.double().view(nQ * Nq, d)
    on = qmask.view(nQ * Nq, 1)
    dQ, aQ = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        w = (G[:, b].double()[:, None].expand(nQ, Nq).reshape(-1, 1) * on) if b != 3 else torch.zeros_like(q[:, :1])
        rows = torch.nan_to_num(D[b].double())
        sim = (q @ rows.t()).masked_fill_(~dmask[b][None], -math.inf)
        top = sim.amax(1, keepdim=True)
        place = torch.arange(Nd, device="cuda")
        at = torch.where(sim == top, place, Nd).amin(1) if b != 3 else torch.zeros(nQ * Nq, dtype=torch.int64, device="cuda")
        dQ += w * rows[at]
        aQ += (w * rows[at]).abs()
        dD, aD = torch.zeros_like(rows), torch.zeros_like(rows)
        dD.index_add_(0, at, w * q)
        aD.index_add_(0, at, (w * q).abs())
        lim = (nQ * Nq + 2) * 2.0 ** -24 * aD
        lim = lim + ROUND[dtype] * (dD.abs() + lim) + TINY[dtype]
        assert bool(((gD[b].double() - dD).abs() <= lim).all()), f"dD of document {b}"
    assert bool((gQ.view(nQ * Nq, d)[~on[:, 0]] == 0).all()), "masked query tokens take a gradient"
    lim = (B + 2) * 2.0 ** -24 * aQ
    lim = lim + ROUND[dtype] * (dQ.abs() + lim) + TINY[dtype]
    assert bool(((gQ.view(nQ * Nq, d).double() - dQ).abs() <= lim).all())


@gpu
def test_most_documents(cuda):
    """More than 2^24 documents with a workgroup each: a launch's threads along one axis end at
    2^32. One token a document, so the scores are dot products on the grid, exact in fp32."""
    import tilemaxsim_amd as tms
    B, d = (1 << 24) + 77, 32
    rng = np.random.default_rng(2)
    Q = _grid(rng, 1, 1, d).half().cuda().requires_grad_(True)
    D = _grid(rng, 4096, d).half().cuda().repeat(-(-B // 4096), 1)[:B].view(B, 1, d).contiguous()
    D[-1] = D[0] + D[1]  # the last one unlike the others
    D.requires_grad_(True)
    print(f"pairs of {B} documents", flush=True)
    s = tms.maxsim_pairs(Q, D)
    with torch.no_grad():
        want = (D[:, 0].float() * Q[0, 0].float()).sum(1)  # (a matrix product of so many rows ends at the same 2^32)
        G = torch.zeros(1, B, device="cuda")
        G[0, ::1001] = 0.5
        G[0, -3:] = -2.0
    assert torch.equal(s[0].detach(), want)
    gQ, gD = torch.autograd.grad(s, (Q, D), G)
    assert torch.equal(gD[:, 0], (G[0, :, None] * Q[0, 0].float()).half())
    terms = G[0, :, None].double() * D[:, 0].double()
    ref, sums = terms.sum(0), terms.abs().sum(0)
    lim = (B / 1001 + 600) * 2.0 ** -24 * sums
    assert bool(((gQ[0, 0].double() - ref).abs() <= lim + ROUND["fp16"] * (ref.abs() + lim)).all())


@gpu
@pytest.mark.parametrize("nQ", [0, 3])
def test_no_own_documents(cuda, nQ):
    """Queries with none of their own documents: no scores, and backward gives zeros."""
    import tilemaxsim_amd as tms
    Q = torch.ones(nQ, 4, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    D = torch.ones(nQ, 0, 7, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    s = tms.maxsim_pairs(Q, D)
    assert s.shape == (nQ, 0) and s.dtype == torch.float32
    dQ, dD = torch.autograd.grad(s, (Q, D), torch.ones_like(s))
    assert dQ.shape == Q.shape and bool((dQ == 0).all()) and dD.shape == D.shape
    assert tms.maxsim_pairs(Q.detach(), D.detach()).shape == (nQ, 0)


def _terms(x):
    """A float32 as three bf16 terms, largest first, in float64."""
    out, left = [], torch.from_numpy(x)
    for _ in range(3):
        t = left.bfloat16().float()
        out.append(t.double().numpy())
        left = left - t
    return out


def _hot(rng, rows, d, spread):
    """Rows with one element that is not zero, of 24 random bits, at places in turn; and the places."""
    at = (np.arange(rows) * 13 + spread) % d  # every place: 13 divides no d here
    x = np.zeros((rows, d), dtype=np.float32)
    x[np.arange(rows), at] = (1 + rng.random(rows)).astype(np.float32)
    return x, at


# A product of two such rows is the product of two numbers: six products of terms, in fp32. The
# three that are left out are below 2^-24 of it together, and the six sums round 2^-24 each.
PRODUCT = 2.0 ** -21


def test_the_bound_sees_every_term():
    """In float64: the six products of terms lie within the bound, any five that lack one with a
    third term do not."""
    rng = np.random.default_rng(0)
    a, b = ((1 + rng.random(500)).astype(np.float32) for _ in range(2))
    ta, tb = _terms(a), _terms(b)
    exact = a.astype(np.float64) * b.astype(np.float64)
    six = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]

    def off(pairs):
        return np.abs(sum(ta[i] * tb[j] for i, j in pairs) - exact) / exact
    assert (off(six) < PRODUCT / 4).all()
    for gone in six:
        assert (off([p for p in six if p != gone]) > PRODUCT).mean() > 0.3, gone


@gpu
@pytest.mark.parametrize("nQ,Nq,B,Nd,d,own", [(2, 3, 3, 140, 32, False), (2, 5, 2, 200, 64, False), (1, 4, 5, 300, 96, True), (3, 2, 4, 400, 128, False),
                                              (2, 3, 3, 260, 77, False), (2, 3, 2, 620, 200, False), (9, 5, 100, 200, 64, False),
                                              (20, 3, 60, 400, 128, False), (40, 2, 50, 310, 77, False)])
def test_all_bits_of_fp32(cuda, nQ, Nq, B, Nd, d, own):
    """Scores and gradients of embeddings of 24 bits, in every form of the kernels."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(nQ + B + d)
    docs = nQ * B if own else B
    q, qat = _hot(rng, nQ * Nq, d, 1)
    x, xat = _hot(rng, docs * Nd, d, 0)
    live = rng.random(docs * Nd) < 0.98
    G = rng.standard_normal((nQ, B)).astype(np.float32)
    scores = np.zeros((nQ, B))
    dQ, dD = np.zeros(q.shape), np.zeros(x.shape)
    q64, x64 = q.astype(np.float64), x.astype(np.float64)
    for i in range(nQ):
        for b in range(B):
            rows = np.arange(Nd) + (i * B + b if own else b) * Nd
            for k in range(i * Nq, (i + 1) * Nq):
                sim = np.where(live[rows], np.where(xat[rows] == qat[k], x64[rows, qat[k]] * q64[k, qat[k]], 0.0), -np.inf)
                best = rows[int(np.argmax(sim))]
                second = np.partition(sim, -2)[-2]
                assert sim.max() > 0 and second < sim.max() * (1 - 4 * PRODUCT)  # which one wins is not in doubt
                scores[i, b] += sim.max()
                dQ[k] += G[i, b].astype(np.float64) * x64[best]
                dD[best] += G[i, b].astype(np.float64) * q64[k]
    shape = (nQ, B, Nd) if own else (B, Nd)
    print(f"pairs of 24 bits nQ={nQ} Nq={Nq} B={B} Nd={Nd} d={d} own={own}", flush=True)
    Q, D = (torch.from_numpy(v).cuda().requires_grad_(True) for v in (q.reshape(nQ, Nq, d), x.reshape(*shape, d)))
    mask = torch.from_numpy(live.reshape(shape)).cuda()
    s = tms.maxsim_pairs(Q, D, mask)
    assert torch.equal(s.detach(), tms.maxsim_pairs(Q.detach(), D.detach(), mask))
    gQ, gD = torch.autograd.grad(s, (Q, D), torch.from_numpy(G).cuda())
    far = np.abs(s.detach().cpu().double().numpy() - scores) / scores
    assert far.max() <= PRODUCT + Nq * 2.0 ** -24, far.max()
    n = np.abs(G).max()
    for name, got, ref, terms in (("dQ", gQ, dQ, B), ("dD", gD, dD, nQ * Nq)):
        lim = (terms + 4) * 2.0 ** -24 * terms * n * 2
        got = got.cpu().double().numpy().reshape(ref.shape)
        assert ((got != 0) <= (ref != 0)).all() and np.abs(got - ref).max() <= lim, name
