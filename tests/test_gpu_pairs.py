"""MaxSim of query and document batches with gradients (``maxsim_pairs``) against the
definition in float64, at the sizes and masks where a kernel's tiles, blocks and splits end.

Tolerances. Scores: fp32 accumulation of d products and Nq maxima, (d + Nq) 2^-23 of the same
sum over absolute values; fp32 rows take six products of bf16 terms, 6 d of them. Gradients:
the embeddings lie on a grid on which dot products are exact, so every maximum's position is
the definition's; what is left is an fp32 sum of n terms, (n + 2) 2^-24 of the sum of their
absolute values (each term is one rounded product), and one rounding to the inputs' type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ROUND = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}  # half of the smallest step


def _grid(rng, *shape):
    """Unit rows on multiples of 2^-11: dot products are whole multiples of 2^-22 below 2^24
    of them, so exact in fp32 in any order (rounding to 8 bits keeps a multiple one)."""
    x = rng.standard_normal(shape)
    x /= np.maximum(np.linalg.norm(x, axis=-1, keepdims=True), 1e-9)
    return torch.from_numpy(np.round(x * 2048) / 2048)


def reference(Q, D, dmask, qmask, G):
    """scores, their bound's sum, dQ, dD and both gradients' sums of absolute values, in float64
    on the CPU; D is (nQ, nway, Nd, d) or (B, Nd, d)."""
    nQ, Nq, d = Q.shape
    own = D.dim() == 4
    B, Nd = D.shape[-3], D.shape[-2]
    docs = D if own else D[None].expand(nQ, B, Nd, d)
    live = (dmask if own else dmask[None].expand(nQ, B, Nd))[:, None]  # (nQ, 1, B, Nd)
    rows = torch.einsum("qid,qbjd->qibj" if own else "qid,bjd->qibj", Q, D)
    mags = torch.einsum("qid,qbjd->qibj" if own else "qid,bjd->qibj", Q.abs(), D.abs()).masked_fill(~live, 0)
    sim = rows.masked_fill(~live, -math.inf).numpy()
    at = torch.from_numpy(np.argmax(sim, -1))  # the first of equal ones
    top = torch.from_numpy(np.max(sim, -1))
    on = qmask[:, :, None]  # (nQ, Nq, 1)
    some = live.any(-1)[:, 0]  # (nQ, B)
    scores = torch.where(on, top, torch.zeros_like(top)).sum(1).masked_fill(~some, -math.inf)
    bound = torch.where(on, mags.amax(-1), torch.zeros_like(top)).sum(1)
    w = torch.where(on & some[:, None], G.double()[:, None].expand(nQ, Nq, B), torch.zeros_like(top))
    won = docs[torch.arange(nQ)[:, None, None], torch.arange(B)[None, None], at]  # (nQ, Nq, B, d)
    dQ, aQ = (w[..., None] * won).sum(2), (w[..., None] * won).abs().sum(2)
    doc = torch.arange(nQ * B).view(nQ, 1, B) if own else torch.arange(B).view(1, 1, B)
    into = (doc * Nd + at).flatten()
    add = (w[..., None] * Q[:, :, None]).reshape(-1, d)
    dD = torch.zeros(D.numel() // d, d, dtype=torch.float64).index_add_(0, into, add).view(D.shape)
    aD = torch.zeros(D.numel() // d, d, dtype=torch.float64).index_add_(0, into, add.abs()).view(D.shape)
    return scores, bound, dQ, dD, aQ, aD


def check(nQ, Nq, B, Nd, d, dtype, own=False, seed=0, masks=True, edit=None):
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(seed)
    docs = (nQ, B) if own else (B,)
    dt = DT[dtype]
    Q, D = _grid(rng, nQ, Nq, d).to(dt), _grid(rng, *docs, Nd, d).to(dt)
    dmask = torch.from_numpy(rng.random((*docs, Nd)) < 0.7) if masks else torch.ones(*docs, Nd, dtype=torch.bool)
    qmask = torch.from_numpy(rng.random((nQ, Nq)) < 0.8) if masks else torch.ones(nQ, Nq, dtype=torch.bool)
    if edit is not None:
        edit(Q, D, dmask, qmask)
    G = torch.from_numpy(rng.standard_normal((nQ, B)).astype(np.float32))
    Qr, Dr = torch.nan_to_num(Q.double()), torch.nan_to_num(D.double())  # NaN stands only where it is masked
    scores, bound, dQ, dD, aQ, aD = reference(Qr, Dr, dmask, qmask, G)
    Qc, Dc = Q.cuda().requires_grad_(True), D.cuda().requires_grad_(True)
    given = (dmask.cuda(), qmask.cuda()) if masks or edit is not None else (None, None)
    print(f"pairs nQ={nQ} Nq={Nq} B={B} Nd={Nd} d={d} {dtype} own={own}", flush=True)
    got = tms.maxsim_pairs(Qc, Dc, *given)
    with torch.no_grad():
        again = tms.maxsim_pairs(Qc, Dc, *given)
    gQ, gD = torch.autograd.grad(got, (Qc, Dc), G.cuda())
    torch.cuda.synchronize()
    assert torch.equal(got.detach(), again), "scores with and without gradients"
    s = got.detach().cpu().double()
    assert torch.equal(torch.isinf(s), torch.isinf(scores))
    fine = torch.isfinite(scores)
    lim = (d * (6 if dtype == "fp32" else 1) + Nq) * 2.0 ** -23 * bound + 1e-30
    assert bool(((s - scores).abs()[fine] <= lim[fine]).all()), float(((s - scores).abs() / lim)[fine].max())
    for name, x, ref, mags, n in (("dQ", gQ, dQ, aQ, B), ("dD", gD, dD, aD, (1 if own else nQ) * Nq)):
        assert x.dtype == dt and x.shape == ref.shape
        lim = (n + 2) * 2.0 ** -24 * mags
        lim = lim + ROUND[dtype] * (ref.abs() + lim) + TINY[dtype]
        off = (x.cpu().double() - ref).abs()
        assert bool((off <= lim).all()), f"{name}: {float((off - lim).max())}"


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(1, 1, 1, 1, 32), (2, 32, 2, 180, 128), (3, 7, 5, 17, 96), (1, 33, 4, 16, 64),
                                          (2, 65, 3, 65, 128), (4, 5, 3, 33, 77), (2, 9, 2, 20, 8), (1, 3, 2, 9, 1),
                                          (2, 16, 3, 40, 256), (3, 100, 2, 31, 32), (2, 4, 2, 1030, 64)])
def test_direct(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ + Nq + B + Nd + d)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(5, 32, 8, 37, 128), (3, 3, 64, 5, 32), (2, 40, 3, 64, 96), (4, 1, 1, 100, 64)])
def test_own_documents(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, own=True, seed=nQ + Nq + B)


# every form of the shared kernel: 1, 2 and 4 blocks a wave, several groups, queries of 1 to 4 blocks
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(4, 32, 700, 3, 128), (8, 5, 300, 20, 64), (9, 32, 257, 70, 96), (16, 17, 150, 33, 32),
                                          (17, 32, 130, 66, 128), (33, 8, 70, 9, 128), (7, 40, 310, 12, 128), (9, 50, 250, 21, 64),
                                          (5, 70, 450, 10, 128), (6, 128, 400, 7, 96), (40, 20, 60, 1, 77), (5, 130, 430, 4, 128)])
def test_shared(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ * 3 + Nq + B)


# many queries and documents: the gradients' forms that share documents, whose tokens come in
# one stage or several, in 16-byte pieces or (odd widths) element by element
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(8, 32, 70, 270, 40), (16, 20, 65, 30, 77), (9, 33, 64, 17, 136), (12, 32, 100, 130, 33),
                                          (20, 3, 300, 65, 160)])
def test_many(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ * 3 + Nq + B)


# more than 128 blocks of 32 query tokens: a document's maxima are sorted in two and three runs
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(150, 5, 30, 20, 64), (130, 3, 70, 300, 33), (95, 40, 8, 17, 136)])
def test_runs(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ)


def test_one_token_wins_all(cuda):
    """Every maximum at one token, the first, a middle or the last one."""
    def at(j):
        def edit(Q, D, dmask, qmask):
            D.zero_()
            Q.abs_()
            D[:, j] = 0.125
            dmask[:] = True
        return edit
    for j in (0, 77, 149):
        check(70, 32, 9, 150, 64, "fp16", edit=at(j))


def test_no_masks(cuda):
    check(5, 32, 500, 47, 128, "fp16", masks=False)
    check(2, 20, 6, 100, 128, "bf16", masks=False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("own,nQ,B", [(False, 3, 6), (False, 9, 300), (True, 4, 5)])
def test_empty_rows_and_masked_values(cuda, own, nQ, B, dtype):
    """Documents and queries that their mask leaves nothing of; NaN and infinities behind masks;
    a document whose only real token is its last one."""
    def edit(Q, D, dmask, qmask):
        docs = dmask.view(-1, dmask.shape[-1])
        docs[0] = False
        docs[-1] = False
        docs[1] = False
        docs[1, -1] = True
        docs[2, :64] = False  # a whole stage of padding in front
        docs[2, 64:] = True
        qmask[1] = False
        qmask[0] = True
        D[~dmask] = float("nan")
        D.view(-1, *D.shape[-2:])[0, 0] = float("inf")
        Q[~qmask] = float("nan")
    check(nQ, 12, B, 90, 64, dtype, own=own, edit=edit)


def test_equal_maxima_go_to_the_first(cuda):
    """Repeated tokens: the gradient goes to the lowest index, across tiles, stages and waves."""
    import tilemaxsim_amd as tms
    for B, nQ in ((2, 3), (600, 4)):
        Q = torch.zeros(nQ, 4, 64)
        Q[..., 0] = 1
        D = torch.zeros(B, 150, 64)
        first = torch.arange(B) % 150
        for b in range(B):
            D[b, first[b]:, 0] = 1  # equal from here on
        Q, D = Q.half().cuda().requires_grad_(True), D.half().cuda().requires_grad_(True)
        s = tms.maxsim_pairs(Q, D)
        assert bool((s == 4).all())
        _, dD = torch.autograd.grad(s, (Q, D), torch.ones_like(s))
        want = torch.zeros(B, 150)
        want[torch.arange(B), first] = 4 * nQ
        assert torch.equal(dD[..., 0].float().cpu(), want) and bool((dD[..., 1:] == 0).all())


def test_differences(cuda):
    """The gradients against differences of the definition in float64: linear pieces, so a
    step that moves no maximum gives the slope up to rounding."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(5)
    Q, D = torch.from_numpy(rng.standard_normal((3, 5, 24))), torch.from_numpy(rng.standard_normal((4, 9, 24)))
    Q, D = Q.float().double(), D.float().double()
    G = torch.from_numpy(rng.standard_normal((3, 4)))

    def f(q, x):
        return float((torch.einsum("qid,bjd->qbij", q, x).amax(-1).sum(-1) * G.float().double()).sum())
    Qc, Dc = Q.float().cuda().requires_grad_(True), D.float().cuda().requires_grad_(True)
    dQ, dD = torch.autograd.grad(tms.maxsim_pairs(Qc, Dc), (Qc, Dc), G.float().cuda())
    h = 1e-6
    for _ in range(20):
        for x, dx, at in ((Q, dQ, 0), (D, dD, 1)):
            k = tuple(int(rng.integers(n)) for n in x.shape)
            up, down = x.clone(), x.clone()
            up[k] += h
            down[k] -= h
            slope = ((f(up, D) - f(down, D)) if at == 0 else (f(Q, up) - f(Q, down))) / (2 * h)
            # 2h differences of a sum of about 60 products of a few units: 1e-13 / 1e-6
            assert abs(slope - float(dx[k])) <= 1e-5 + 1e-6 * abs(slope), (k, slope, float(dx[k]))


def test_layouts_streams_and_one_sided_gradients(cuda):
    """Strided and misaligned inputs, integer masks, a side stream, gradients of one side, and
    the same bits from every run."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(1)
    Q, D = _grid(rng, 6, 10, 64).half().cuda(), _grid(rng, 50, 21, 64).half().cuda()
    m = torch.from_numpy(rng.random((50, 21)) < 0.6).cuda()
    m[:, 0] = True
    base = tms.maxsim_pairs(Q, D, m)
    flat = torch.empty(Q.numel() + 3, dtype=Q.dtype, device="cuda")[3:]
    odd = flat.copy_(Q.flatten()).view(Q.shape)  # 6 bytes off
    assert odd.data_ptr() % 16 == 6
    wide = torch.empty(50, 21, 128, dtype=D.dtype, device="cuda")[..., :64].copy_(D)
    back = D.transpose(0, 1).contiguous().transpose(0, 1)
    for q, x in ((odd, D), (Q, wide), (Q, back)):
        assert torch.equal(tms.maxsim_pairs(q, x, m), base)
    for dt in (torch.uint8, torch.int8, torch.int64):
        assert torch.equal(tms.maxsim_pairs(Q, D, m.to(dt) * 3), base)
    G = torch.randn(6, 50, device="cuda")
    Qg, Dg = Q.clone().requires_grad_(True), D.clone().requires_grad_(True)
    both = torch.autograd.grad(tms.maxsim_pairs(Qg, Dg, m), (Qg, Dg), G)
    assert torch.equal(torch.autograd.grad(tms.maxsim_pairs(Qg, D, m), Qg, G)[0], both[0])
    assert torch.equal(torch.autograd.grad(tms.maxsim_pairs(Q, Dg, m), Dg, G)[0], both[1])
    assert torch.equal(torch.autograd.grad(tms.maxsim_pairs(Qg, Dg, m), Dg, G.t().contiguous().t())[0], both[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = tms.maxsim_pairs(Qg, Dg, m)
        again = torch.autograd.grad(s, (Qg, Dg), G)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(s.detach(), base) and all(torch.equal(a, b) for a, b in zip(again, both))


@pytest.mark.parametrize("nQ,Nq,B,Nd", [(0, 3, 4, 5), (3, 0, 4, 5), (3, 4, 0, 5), (3, 4, 5, 0)])
def test_nothing(cuda, nQ, Nq, B, Nd):
    import tilemaxsim_amd as tms
    Q = torch.ones(nQ, Nq, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    D = torch.ones(B, Nd, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    s = tms.maxsim_pairs(Q, D)
    assert s.shape == (nQ, B)
    if s.numel():
        assert bool((s == (-math.inf if Nd == 0 else 0)).all())
    dQ, dD = torch.autograd.grad(s, (Q, D), torch.ones_like(s))
    assert bool((dQ == 0).all()) and bool((dD == 0).all())
    own = torch.ones(nQ, 2, Nd, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    s = tms.maxsim_pairs(Q, own)
    dQ, dD = torch.autograd.grad(s, (Q, own), torch.ones_like(s))
    if Nd == 0 or Nq == 0:
        assert bool((dQ == 0).all()) and bool((dD == 0).all())


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,B,d", [(2, 5, 64), (3, 6, 77), (9, 300, 64), (9, 300, 77), (5, 700, 128), (3, 6, 200)])
def test_nan_at_a_real_token_reaches_the_scores(cuda, dt, nQ, B, d):
    """A NaN or infinity at a real token (of a text of its own) makes that text's scores NaN, at
    a masked one nothing, with and without positions; and the two forms' scores are the same bits."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(d)
    Q, D = _grid(rng, nQ, 7, d).to(DT[dt]).cuda(), _grid(rng, B, 37, d).to(DT[dt]).cuda()
    qmask, dmask = torch.ones(nQ, 7, dtype=torch.bool, device="cuda"), torch.ones(B, 37, dtype=torch.bool, device="cuda")
    qmask[0, 6] = dmask[4, 20] = dmask[0, 36] = False
    dmask[2] = False
    clean = tms.maxsim_pairs(Q, D, dmask, qmask)
    Q[0, 6, d - 1] = D[4, 20, 3] = D[2, 5, 0] = math.nan
    D[0, 36] = math.inf
    assert torch.equal(tms.maxsim_pairs(Q, D, dmask, qmask), clean)
    Q[1, 2, d - 1] = math.nan
    D[3, 36, 0] = math.nan
    D[B - 1, 0] = math.inf  # inf - inf over a row of both signs
    want = torch.zeros(nQ, B, dtype=torch.bool, device="cuda")
    want[1] = want[:, 3] = want[:, B - 1] = True
    want[:, 2] = False
    scores = tms.maxsim_pairs(Q, D, dmask, qmask)
    assert torch.equal(torch.isnan(scores), want)
    assert torch.equal(scores[~want], clean[~want])
    kept = tms.maxsim_pairs(Q.requires_grad_(True), D, dmask, qmask).detach()
    assert torch.equal(torch.isnan(kept), want) and torch.equal(kept[~want], clean[~want])


@pytest.mark.parametrize("nQ,B,Nd", [(3, 6, 20), (9, 300, 70)])
def test_graph(cuda, nQ, B, Nd):
    """Captured scores with both gradients follow their inputs from replay to replay."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(B)
    Q, D = (_grid(rng, *s).half().cuda().requires_grad_(True) for s in ((nQ, 10, 64), (B, Nd, 64)))
    dmask = torch.ones(B, Nd, dtype=torch.bool, device="cuda")
    G = torch.ones(nQ, B, device="cuda")

    def step():
        s = tms.maxsim_pairs(Q, D, dmask)
        return (s.detach(), *torch.autograd.grad(s, (Q, D), G))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for replay in range(4):
        with torch.no_grad():
            Q.copy_(_grid(rng, *Q.shape).half())
            D.copy_(_grid(rng, *D.shape).half())
            dmask.copy_(torch.from_numpy(rng.random((B, Nd)) < 0.7))
            G.copy_(torch.from_numpy(rng.standard_normal((nQ, B)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in kept]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), replay
        torch.cuda.synchronize()


# four blocks a wave: queries of one and of two blocks, the last group of waves full and not
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(27, 32, 90, 70, 128), (30, 7, 80, 33, 64), (14, 40, 160, 66, 96), (64, 32, 40, 37, 128),
                                          (32, 20, 70, 130, 32)])
def test_four_blocks_a_wave(cuda, nQ, Nq, B, Nd, d, dtype):
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ * 3 + Nq + B)


# enough query tokens and documents for the query gradient that shares documents: tokens in one
# stage or several, rows in 16-byte pieces or element by element, last groups of waves partly empty
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("nQ,Nq,B,Nd,d", [(60, 5, 140, 270, 40), (65, 3, 130, 30, 77), (30, 33, 140, 17, 136), (70, 4, 120, 130, 33),
                                          (5, 30, 1700, 9, 128), (17, 32, 500, 20, 64)])
def test_shared_documents_in_the_query_gradient(cuda, nQ, Nq, B, Nd, d, dtype):
    assert nQ * -(-Nq // 32) * B > 8192
    check(nQ, Nq, B, Nd, d, dtype, seed=nQ * 3 + Nq + B)


@pytest.mark.parametrize("nQ,B", [(6, 40), (60, 140)])
def test_infinite_gradient_stays_where_it_belongs(cuda, nQ, B):
    """An infinite gradient of one score: query tokens and documents without a maximum in that
    pair keep the gradients that they have without it."""
    import tilemaxsim_amd as tms
    rng = np.random.default_rng(B)
    Q, D = (_grid(rng, *s).half().cuda().requires_grad_(True) for s in ((nQ, 9, 64), (B, 30, 64)))
    qmask, dmask = torch.ones(nQ, 9, dtype=torch.bool, device="cuda"), torch.ones(B, 30, dtype=torch.bool, device="cuda")
    qmask[2, 4:] = False
    dmask[5, 20:] = False
    scores = tms.maxsim_pairs(Q, D, dmask, qmask)
    G = torch.randn(nQ, B, device="cuda")
    G[2, 5] = 0
    dQ, dD = torch.autograd.grad(scores, (Q, D), G, retain_graph=True)
    G[2, 5] = math.inf
    eQ, eD = torch.autograd.grad(scores, (Q, D), G)
    hit = torch.zeros(nQ, 9, dtype=torch.bool, device="cuda")
    hit[2, :4] = True
    assert torch.equal(dQ[~hit], eQ[~hit]) and not bool(torch.isfinite(eQ[hit]).any())
    others = torch.arange(B, device="cuda") != 5
    assert torch.equal(dD[others], eD[others]) and bool((eD[5, 20:] == 0).all())
    won = ~torch.isfinite(eD[5]).all(-1)
    assert 1 <= int(won.sum()) <= 4 and torch.equal(dD[5][~won], eD[5][~won])
