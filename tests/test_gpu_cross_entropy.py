"""``linear_cross_entropy`` and its gradients against the definition in float64, at the sizes
where tiles, blocks of the vocabulary, pieces and splits end.

Tolerances. A logit is an fp32 sum of d products: D = scale (d + 2) 2^-24 sum |h| |w| off at
most (fp32 rows: 6 d products of bf16 terms), and what exp2 and log2 take and give adds
2^-21 (|x| + |lse| + 2). The loss is two such values off. An element of the softmax is 2 D
off relative to itself, and rounded to the type it is held in (fp16: at least 2^-40 steps of
1); the gradients are fp32 sums of n of them times the other operand, (n + 8) 2^-24 of the
sum of absolute values, and one rounding to the inputs' type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ROUND = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}


def data(N, V, d, dtype, seed, std=2.0, ignored=0.15):
    rng = np.random.default_rng(seed)
    H = torch.from_numpy(rng.standard_normal((N, d))).to(DT[dtype])
    W = torch.from_numpy(rng.standard_normal((V, d)) * std / math.sqrt(max(d, 1))).to(DT[dtype])
    t = torch.from_numpy(rng.integers(0, V, N))
    if N > 1:
        t[torch.from_numpy(rng.random(N) < ignored)] = -100
        t[N // 2] = V - 1
    return H, W, t


def reference(H, W, t, scale, ignore, reduction, G):
    """loss, dH, dW and their bounds, in float64 on the GPU; `G` is what comes back for the loss."""
    H, W = H.double().cuda(), W.double().cuda()
    t, G = t.cuda(), G.double().cuda()
    N, d = H.shape
    kept = t != ignore
    at = torch.where(kept, t, torch.zeros_like(t))
    H = torch.where(kept[:, None], H, torch.zeros_like(H))
    x = scale * (H @ W.t())
    lse = torch.logsumexp(x, 1)
    rows = torch.where(kept, lse - x[torch.arange(N), at], torch.zeros_like(lse))
    n = kept.sum()
    loss = rows if reduction == "none" else rows.sum() / (n if reduction == "mean" else 1)
    g = (G if reduction == "none" else G.expand(N) / (n if reduction == "mean" else 1)) * kept
    soft = torch.exp(x - lse[:, None])
    P = soft.clone()
    P[torch.arange(N), at] -= 1
    P = torch.where(kept[:, None], P * (g * scale)[:, None], torch.zeros_like(P))
    soft = soft * (g * scale).abs()[:, None]
    near = (scale * (H.abs() @ W.abs().t())).amax(1), x.abs().amax(1) + lse.abs() + 2  # per row
    return dict(loss=loss, rows=rows, dH=P @ W, dW=P.t() @ H, aH=P.abs() @ W.abs(), aW=P.abs().t() @ H.abs(),
                eH=soft @ W.abs(), eW=soft.t() @ H.abs(),
                sW=W.abs().sum(0), sH=H.abs().sum(0), near=near, top=float((g * scale).abs().max()) if N else 0.0)


def check(N, V, d, dtype, scale=1.0, reduction="mean", seed=0, ignore=-100, std=2.0, given=None, up=None):
    import tilemaxsim_amd as tms
    H, W, t = given if given is not None else data(N, V, d, dtype, seed, std)
    rng = np.random.default_rng(seed + 1)
    G = torch.from_numpy((rng.random(N) + 0.1).astype(np.float32)) if reduction == "none" else torch.tensor(0.7)
    if up is not None:
        G = up
    r = reference(torch.nan_to_num(H), W, t, scale, ignore, reduction, G)
    print(f"ce N={N} V={V} d={d} {dtype} scale={scale} {reduction}", flush=True)
    Hc, Wc, tc = H.cuda().requires_grad_(True), W.cuda().requires_grad_(True), t.cuda()
    loss = tms.linear_cross_entropy(Hc, Wc, tc, scale=scale, ignore_index=ignore, reduction=reduction)
    with torch.no_grad():
        assert torch.equal(tms.linear_cross_entropy(Hc, Wc, tc, scale=scale, ignore_index=ignore, reduction=reduction), loss)
    dH, dW = torch.autograd.grad(loss, (Hc, Wc), G.cuda())
    torch.cuda.synchronize()
    assert loss.dtype == torch.float32 and dH.dtype == H.dtype and dW.dtype == W.dtype
    terms = 6 if dtype == "fp32" else 1
    off = (terms * d + 2) * 2.0 ** -24 * r["near"][0] + 2.0 ** -21 * r["near"][1]
    lim = 2 * off
    if reduction != "none":
        lim = lim.sum() / (max(int((t != ignore).sum()), 1) if reduction == "mean" else 1) + 2.0 ** -23 * abs(r["loss"])
    assert bool(((loss.double() - r["loss"]).abs() <= lim + 1e-30).all()), (loss, r["loss"])
    rel = ROUND[dtype] + 2.0 ** -22
    for name, x, n, other in (("dH", dH, V, r["sW"]), ("dW", dW, N, r["sH"])):
        sums, ref = r["a" + name[1]], r[name]
        lim = 2 * float(off.max()) * r["e" + name[1]] + (rel + (terms * n + 8) * 2.0 ** -24) * sums + 2.0 ** -40 * r["top"] * other
        lim = lim + ROUND[dtype] * (ref.abs() + lim) + TINY[dtype]
        bad = (x.double() - ref).abs() - lim
        assert bool((bad <= 0).all()), f"{name}: {float(bad.max())} beyond the bound, of {float(ref.abs().max())}"
    return loss, dH, dW


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("N,V,d", [(1, 1, 8), (1, 2, 1), (1, 1000, 64), (2, 63, 32), (3, 65, 77), (64, 129, 96), (65, 1, 128),
                                   (65, 257, 40), (17, 5000, 128), (256, 256, 64), (257, 513, 136), (300, 1000, 768),
                                   (5, 20000, 256), (700, 100, 33), (130, 3001, 520)])
def test_sizes(cuda, N, V, d, dtype):
    check(N, V, d, dtype, seed=N + V + d)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("N,V,d,scale", [(70, 900, 128, 20.0), (10, 333, 64, 0.3)])
def test_reductions_and_scales(cuda, N, V, d, scale, dtype, reduction):
    check(N, V, d, dtype, scale=scale, reduction=reduction, std=1.0, seed=3)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_pieces(cuda, dtype):
    """A vocabulary of several pieces, a short last one among them."""
    check(2000, 40000, 8, dtype, seed=1)  # 2048 rows x 40,000: pieces of 131,072 columns at most: one
    check(9000, 33000, 16, dtype, seed=2)  # 9216 rows: two pieces


def test_unequal_row_weights(cuda):
    """Weights over many powers of two: the largest rows' accuracy holds for the smallest."""
    for dtype in ("fp16", "bf16", "fp32"):
        up = torch.logspace(-6, 3, 80)
        up[7] = -2.5
        up[9] = 0
        H, W, t = data(80, 700, 64, dtype, 4)
        _, dH, _ = check(80, 700, 64, dtype, reduction="none", given=(H, W, t), up=up)
        assert bool((dH[9] == 0).all())


def test_ignored_rows(cuda):
    """Rows that are ignored hold NaN and take no part; other ignore indices; none left."""
    import tilemaxsim_amd as tms
    for N in (40, 300):
        H, W, t = data(N, 500, 64, "bf16", 9, ignored=0.4)
        H[t == -100] = float("nan")
        _, dH, _ = check(N, 500, 64, "bf16", given=(H, W, t))
        assert bool((dH[(t == -100).cuda()] == 0).all())
    H, W, t = data(30, 50, 32, "fp16", 2)
    t = torch.where(t == -100, torch.full_like(t, 7), t)
    check(30, 50, 32, "fp16", ignore=7, given=(H, W, t))
    gone = torch.full((30,), -100, device="cuda")
    Hc, Wc = H.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    for reduction in ("mean", "sum", "none"):
        loss = tms.linear_cross_entropy(Hc, Wc, gone, reduction=reduction)
        if reduction == "mean":
            assert math.isnan(float(loss))
        else:
            assert bool((loss == 0).all())
            dH, dW = torch.autograd.grad(loss, (Hc, Wc), torch.ones_like(loss))
            assert bool((dH == 0).all()) and bool((dW == 0).all())


def test_targets_outside_and_non_finite(cuda):
    import tilemaxsim_amd as tms
    H, W, t = (x.cuda() for x in data(20, 50, 32, "fp16", 2, ignored=0))
    good = tms.linear_cross_entropy(H, W, t, reduction="none")
    for bad in (50, -1, 1 << 40):
        t2 = t.clone()
        t2[3] = bad
        Hg = H.clone().requires_grad_(True)
        rows = tms.linear_cross_entropy(Hg, W, t2, reduction="none")
        assert math.isnan(float(rows[3]))
        rest = torch.arange(20, device="cuda") != 3
        assert torch.equal(rows[rest], good[rest])
        dH, = torch.autograd.grad(rows, Hg, torch.ones_like(rows))
        assert bool(torch.isnan(dH[3]).all()) and bool(torch.isfinite(dH[rest]).all())
    H2 = H.clone()
    H2[5] = float("nan")
    rows = tms.linear_cross_entropy(H2, W, t, reduction="none")
    assert math.isnan(float(rows[5])) and bool(torch.isfinite(rows[torch.arange(20, device="cuda") != 5]).all())
    # a vocabulary row that is never chosen: its logits are -inf
    H3, W3 = H.abs() + 0.01, W.clone()
    W3[11] = float("-inf")
    t3 = torch.where(t == 11, torch.zeros_like(t), t)
    keep = [v for v in range(50) if v != 11]
    rows = tms.linear_cross_entropy(H3, W3, t3, reduction="none")
    want = torch.nn.functional.cross_entropy(H3.double() @ W[keep].double().t(), t3 - (t3 > 11).long(), reduction="none")
    assert bool(((rows.double() - want).abs() <= 1e-5 * (1 + want)).all())


def test_large_logits(cuda):
    """Logits of hundreds, and a softmax that is 1 at the target."""
    for dtype in ("fp16", "bf16", "fp32"):
        check(50, 400, 128, dtype, scale=30.0, std=5.0, seed=6)
        H, W, t = data(40, 100, 64, dtype, 8, ignored=0)
        H = (W[t].double() * 8).to(DT[dtype])
        check(40, 100, 64, dtype, scale=50.0, given=(H, W, t))


def test_differences(cuda):
    """The gradients against differences of the definition in float64: third derivatives times
    h^2 (1e-8) and rounding of the difference (1e-16 / 1e-4) stay below 1e-6."""
    rng = np.random.default_rng(3)
    H, W, t = data(6, 30, 24, "fp32", 5)
    _, dH, dW = check(6, 30, 24, "fp32", given=(H, W, t), up=torch.tensor(1.0))
    H, W = H.double(), W.double()
    kept = t != -100

    def f(h, w):
        return float(torch.nn.functional.cross_entropy(h @ w.t(), t, ignore_index=-100))
    assert int(kept.sum()) > 2
    h = 1e-4
    for _ in range(15):
        for x, dx, at in ((H, dH, 0), (W, dW, 1)):
            k = tuple(int(rng.integers(n)) for n in x.shape)
            up, down = x.clone(), x.clone()
            up[k] += h
            down[k] -= h
            slope = ((f(up, W) - f(down, W)) if at == 0 else (f(H, up) - f(H, down))) / (2 * h)
            assert abs(slope - float(dx[k])) <= 1e-6 + 1e-5 * abs(slope), (k, slope, float(dx[k]))


def test_layouts_streams_and_one_sided_gradients(cuda):
    import tilemaxsim_amd as tms
    H, W, t = (x.cuda() for x in data(96, 300, 64, "bf16", 1))
    Hg, Wg = H.clone().requires_grad_(True), W.clone().requires_grad_(True)
    base = tms.linear_cross_entropy(Hg, Wg, t)
    both = torch.autograd.grad(base, (Hg, Wg))
    H3 = H.view(4, 24, 64).clone().requires_grad_(True)
    l3 = tms.linear_cross_entropy(H3, W, t.view(4, 24).int())
    assert torch.equal(l3, base)
    assert torch.equal(torch.autograd.grad(l3, H3)[0].view(96, 64), both[0])
    assert tms.linear_cross_entropy(H3, W, t.view(4, 24), reduction="none").shape == (4, 24)
    assert torch.equal(torch.autograd.grad(tms.linear_cross_entropy(H, Wg, t), Wg)[0], both[1])
    odd = torch.empty(W.numel() + 1, dtype=W.dtype, device="cuda")[1:].copy_(W.flatten()).view(W.shape)
    assert torch.equal(tms.linear_cross_entropy(H.t().contiguous().t(), odd, t), base)
    tied = W.clone().requires_grad_(True)  # one tensor on both sides
    h = tied[:96]
    g, = torch.autograd.grad(tms.linear_cross_entropy(h, tied, t), tied)
    x = W[:96].clone().requires_grad_(True)
    a, b = torch.autograd.grad(tms.linear_cross_entropy(x, Wg, t), (x, Wg))
    want = b.float()
    want[:96] += a.float()
    assert torch.equal(g, want.bfloat16())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = tms.linear_cross_entropy(Hg, Wg, t)
        again = torch.autograd.grad(loss, (Hg, Wg))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, base) and all(torch.equal(x, y) for x, y in zip(again, both))


def test_nothing(cuda):
    import tilemaxsim_amd as tms
    W = torch.ones(5, 16, device="cuda", requires_grad=True)
    H = torch.ones(0, 16, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert tms.linear_cross_entropy(H, W, t, reduction="none").shape == (0,)
    loss = tms.linear_cross_entropy(H, W, t, reduction="sum")
    assert float(loss) == 0 and math.isnan(float(tms.linear_cross_entropy(H, W, t)))
    dH, dW = torch.autograd.grad(loss, (H, W))
    assert dH.shape == (0, 16) and bool((dW == 0).all())
    z = tms.linear_cross_entropy(torch.ones(3, 0, device="cuda"), torch.ones(4, 0, device="cuda"), torch.tensor([0, 1, 3], device="cuda"))
    assert abs(float(z) - math.log(4)) < 1e-6


def test_graph(cuda):
    """A captured loss with its gradients follows its inputs from replay to replay."""
    import tilemaxsim_amd as tms
    H, W, t = (x.cuda() for x in data(100, 400, 64, "fp16", 1))
    Hg, Wg = H.clone().requires_grad_(True), W.clone().requires_grad_(True)

    def step():
        loss = tms.linear_cross_entropy(Hg, Wg, t)
        return (loss.detach(), *torch.autograd.grad(loss, (Hg, Wg)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            Hg.mul_(1.1)
            Wg.add_(0.01)
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
