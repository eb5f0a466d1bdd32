"""``linear_cross_entropy`` where a row is nearly right: losses of 1e-2 down to 1e-9, with logits
of a few units up to a thousand, keep their digits in the loss and in both gradients.

Embeddings lie on a grid on which dot products are exact, so the logits' own rounding has no
part. Tolerances, relative to the loss or to an element of P (the softmax less the target's 1):
a term exp2(y) takes y as two products and a difference, each rounded at y's size, 3 |y| 2^-24
ln 2 relative to the term, and 2^-20 for exp2 and for sums of a row (32 terms a lane, 64 joined);
the target's element of P is such a sum of the others. log1p adds 2^-22. Gradients are sums of n
terms, (n + 8) 2^-24 of their absolute values (six products a term in fp32), P is rounded to the
type it is held in (fp16: times 2^15 and half a weight or more, so to steps of 2^-39 at least), and
the result once to the inputs' type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ROUND = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}


def _check(H, W, t, scale, dtype, up):
    """H and W in float64 with exact products; `up` is what comes back for each row's loss."""
    import tilemaxsim_amd as tms
    N, V = len(t), W.shape[0]
    row = torch.arange(N)
    x = scale * (H @ W.t())  # 2^-53 of it: nothing beside the tolerances
    y = (x - x[row, t][:, None]).abs() * math.log2(math.e)
    others = torch.exp(x - x[row, t][:, None])
    others[row, t] = 0
    rest = others.sum(1)
    loss = torch.log1p(rest)
    away = 3 * 2.0 ** -24 * math.log(2) * (y + y.amax(1, keepdim=True) * (rest[:, None] > 1)) + 2.0 ** -20  # of each term
    lim = (others * away).sum(1) / (1 + rest) + 2.0 ** -22 * loss
    P = others / (1 + rest)[:, None]
    off = P * (away + (others * away).sum(1, keepdim=True) / (1 + rest)[:, None])
    P[row, t] = -rest / (1 + rest)
    off[row, t] = (others * away).sum(1) / (1 + rest)
    off += (ROUND[dtype] + 2.0 ** -22) * P.abs() + (2.0 ** -39 if dtype == "fp16" else 0.0)
    dH, dW = up * scale * (P @ W), up * scale * (P.t() @ H)
    Hc, Wc = H.to(DT[dtype]).cuda().requires_grad_(True), W.to(DT[dtype]).cuda().requires_grad_(True)
    assert torch.equal(Hc.detach().cpu().double(), H) and torch.equal(Wc.detach().cpu().double(), W)
    got = tms.linear_cross_entropy(Hc, Wc, t.cuda(), scale=scale, reduction="none")
    gH, gW = torch.autograd.grad(got, (Hc, Wc), torch.full((N,), up, device="cuda"))
    got = got.detach().cpu().double()
    assert bool((got >= 0).all())
    bad = (got - loss).abs() / lim.clamp(min=1e-300)
    assert bool(((got - loss).abs() <= lim).all()), f"loss {float(got[bad.argmax()])} for {float(loss[bad.argmax()])}"
    terms = 6 if dtype == "fp32" else 1
    for name, g, ref, sums, wide, n in (("dH", gH, dH, P.abs() @ W.abs(), off @ W.abs(), V), ("dW", gW, dW, P.abs().t() @ H.abs(), off.t() @ H.abs(), N)):
        lim = up * scale * (wide + (terms * n + 8) * 2.0 ** -24 * sums)
        lim = lim + (ROUND[dtype] + 2.0 ** -22) * (ref.abs() + lim) + TINY[dtype]
        far = (g.cpu().double() - ref).abs()
        if dtype == "fp16":  # a gradient past the type's range is an infinity
            past = (ref.abs() - lim >= 65520) & (g.cpu().double() == torch.sign(ref) * math.inf)
            far = torch.where(past, torch.zeros_like(far), far)
        assert bool((far <= lim).all()), f"{name}: {float((far / lim.clamp(min=1e-300)).max())} times the bound"
    return loss


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scale,gap,base", [(1.0, 8, 4), (1.0, 12, 16), (1.0, 20, 256), (1.0, 16, 1024), (20.0, 0.5, 1), (20.0, 1, 4),
                                            (1 / 0.07, 1, 8), (1 / 0.07, 1.5, 64)])
def test_rows_that_are_nearly_right(cuda, dtype, scale, gap, base):
    """48 classes, each with a coordinate of its own; `base` is added to every dot product."""
    rng = np.random.default_rng(7)
    N, V, d = 40, 48, 64
    t = torch.from_numpy(rng.integers(0, V, N))
    W, H = torch.zeros(V, d, dtype=torch.float64), torch.zeros(N, d, dtype=torch.float64)
    W[torch.arange(V), torch.arange(V)] = gap
    H[torch.arange(N), t] = 1
    W[:, 63], H[:, 63] = base / 4, 4
    W[:, 48:62] = torch.from_numpy(rng.integers(-2, 3, (V, 14))) / 8 / min(scale, 4.0).__ceil__()
    H[:, 48:62] = torch.from_numpy(rng.integers(-2, 3, (N, 14))) / 4
    print(f"near zero {dtype} scale={scale} gap={gap} base={base}", flush=True)
    loss = _check(H, W, t, scale, dtype, 4096.0)
    assert float(loss.min()) < 0.1


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("N,V,many", [(30, 5000, 1.0), (70, 3000, 1.5), (3, 20011, 2.0), (2000, 700, 1.0)])
def test_targets_in_every_block(cuda, dtype, N, V, many):
    """A row near its target's among thousands, the nearest other one deciding the loss; one
    target first and one last, and rows that are wrong beside them."""
    rng = np.random.default_rng(N + V)
    W = torch.from_numpy(rng.integers(-4, 5, (V, 64)) / 4.0)
    t = torch.from_numpy(rng.integers(0, V, N))
    t[0], t[1] = 0, V - 1
    H = many * W[t]
    H[2:N:7] = torch.from_numpy(rng.integers(-4, 5, H[2:N:7].shape) / 4.0)
    print(f"near zero {dtype} N={N} V={V} many={many}", flush=True)
    loss = _check(H, W, t, 1.0, dtype, 256.0)
    assert float(loss.min()) < 1e-3 and float(loss.max()) > 1


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_one_class(cuda, dtype):
    """A vocabulary of one: the loss and both gradients are exactly zero."""
    import tilemaxsim_amd as tms
    H = (torch.randn(9, 72, device="cuda") * 3).to(DT[dtype]).requires_grad_(True)
    W = torch.randn(1, 72, device="cuda").to(DT[dtype]).requires_grad_(True)
    loss = tms.linear_cross_entropy(H, W, torch.zeros(9, dtype=torch.int64, device="cuda"), scale=31.0, reduction="none")
    assert bool((loss == 0).all())
    for g in torch.autograd.grad(loss, (H, W), torch.ones_like(loss)):
        assert bool((g == 0).all())
