"""``maxsim_pairs`` at the ends of its range: the longest documents, the most documents, queries
with no documents of their own."""
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
