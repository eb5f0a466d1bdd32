"""The gated projection against float64.

Tolerances, for each element, from the arithmetic. E = 2^-23 for a rounding of an fp32 sum; fp32
inputs' products of three bf16 terms each are off by as much again.
 * g, u: E (d + 4) <|x|, |w|>. The activations' slopes are at most 1.13, their second derivatives at
   most 0.8 (gelu: 2 phi(0)); the functions themselves are formed to 2^-20 of |a| (an exponential, a
   reciprocal or erfc and three products), slopes to 2^-20 (1 + |g|).
 * h: |u| (1.13 eg + 2^-20 |a|) + |a| eu, and half a step of its type (u).
 * dg: |dh| (|a'| eu + |u| (0.8 eg + 2^-20 (1 + |g|))), du: |dh| (1.13 eg + 2^-20 |a|); both u of
   themselves more when they are rounded (16 bits; up to 64 tokens to two terms, u^2), in fp16 at least 2^-25 of the largest |dh|.
 * The products of those: their errors with the other operand's magnitude, E (n + 4) of the sum of magnitudes
   over n, u of the result, and half of the type's smallest number.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -140}
E = 2.0 ** -23
DT = [torch.bfloat16, torch.float16, torch.float32]


def make(N, d, F, dt, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, d, generator=g, device="cuda").to(dt)
    wg, wu = ((torch.randn(F, d, generator=g, device="cuda") * 2 / math.sqrt(d)).to(dt) for _ in range(2))
    G = (torch.randn(N, F, generator=g, device="cuda") * size).to(dt)
    return [t.requires_grad_(True) for t in (x, wg, wu)], G


def functions(g, act):
    """An activation's values and slopes in 64 bits."""
    g = g.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")
        slope = torch.autograd.grad(a.sum(), g)[0]
    return a.detach(), slope


@torch.no_grad()
def reference(x, wg, wu, G, act):
    dt = x.dtype
    u_, tiny = U[dt], TINY[dt]
    held = 0.0 if dt == torch.float32 else u_ if x.shape[0] > 64 else u_ * u_
    x, wg, wu, G = (t.detach().double() for t in (x, wg, wu, G))
    (N, d), F = x.shape, wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = E * (d + 4) * (x.abs() @ wg.abs().T), E * (d + 4) * (x.abs() @ wu.abs().T)
    a, slope = functions(g, act)
    ea = 1.13 * eg + 2.0 ** -20 * a.abs()
    h = a * u
    eh = u.abs() * ea + a.abs() * eu
    dg, du = G * u * slope, G * a
    floor = 2.0 ** -25 * float(G.abs().max()) if dt == torch.float16 and G.numel() else 0.0
    edg = G.abs() * (slope.abs() * eu + u.abs() * (0.8 * eg + 2.0 ** -20 * (1 + g.abs()))) + held * dg.abs() + floor
    edu = G.abs() * ea + held * du.abs() + floor
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + E * (2 * F + 4) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    dwg, dwu = dg.T @ x, du.T @ x
    edwg = edg.T @ x.abs() + E * (N + 4) * (dg.abs().T @ x.abs())
    edwu = edu.T @ x.abs() + E * (N + 4) * (du.abs().T @ x.abs())
    return [(r, e + u_ * r.abs() + tiny) for r, e in ((h, eh), (dx, edx), (dwg, edwg), (dwu, edwu))]


def close(got, want, what):
    for x, (y, o), name in zip(got, want, ("h", "dx", "dw_gate", "dw_up")):
        assert x.shape == y.shape and not torch.isnan(x).any(), f"{what}: {name}"
        beyond = y.abs() > torch.finfo(x.dtype).max * (1 + U[x.dtype])  # rounds to infinity
        assert torch.equal(x[beyond].double(), torch.sign(y[beyond]) * math.inf), f"{what}: {name} beyond its type's range"
        x, y, o = x[~beyond], y[~beyond], o[~beyond]
        over = float(((x.double() - y).abs() / o.clamp(min=1e-300)).max()) if x.numel() else 0.0
        assert over <= 1.0, f"{what}: {name} is {over:.3g} times its bound off"


def check(N, d, F, dt, act, seed=0, size=1.0):
    import tilemaxsim_amd as tms
    what = f"{N} x {d} x {F} {dt} {act}"
    print(what, flush=True)
    (x, wg, wu), G = make(N, d, F, dt, seed, size)
    h = tms.gated_linear(x, wg, wu, act)
    grads = torch.autograd.grad(h, (x, wg, wu), G)
    assert h.dtype == dt and all(t.dtype == dt for t in grads)
    close((h.detach(), *grads), reference(x, wg, wu, G, act), what)
    with torch.no_grad():
        assert torch.equal(tms.gated_linear(x, wg, wu, act), h)
    again = torch.autograd.grad(tms.gated_linear(x, wg, wu, act), (x, wg, wu), G)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "a run's bits differ"


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_activations(cuda, act, dt):
    check(100, 64, 130, dt, act, seed=1)
    check(9, 64, 130, dt, act, seed=2)


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("N,d,F", [
    (1, 8, 1), (1, 1, 1), (1, 768, 2048), (2, 77, 33), (15, 256, 17), (16, 40, 8), (17, 256, 64), (33, 33, 100), (63, 128, 9), (64, 264, 70),
    (65, 64, 31), (65, 1, 16), (128, 77, 64), (129, 200, 65), (257, 96, 127), (300, 264, 129), (64, 64, 300), (1000, 72, 40)])
def test_sizes(cuda, N, d, F, dt):
    check(N, d, F, dt, "silu", seed=N + d + F)


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("N,d,F", [(1229, 768, 2043), (2048, 512, 1024), (4500, 128, 1500), (700, 1032, 2500)])
def test_large_tiles(cuda, N, d, F, dt):
    check(N, d, F, dt, "gelu", seed=3)


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("N,d,F", [(1, 4096, 8193), (9, 4096, 8193), (16, 2048, 8200), (16, 2048, 8190), (17, 2048, 8190), (32, 1024, 2040),
                                   (33, 1024, 2040), (32, 1024, 2050), (64, 1020, 2050), (65, 1020, 2050), (128, 96, 33)])
def test_few_tokens(cuda, N, d, F, dt):
    """Both sides of where the kernel of few tokens ends."""
    check(N, d, F, dt, "silu", seed=5)


@pytest.mark.parametrize("N", [3, 200])
@pytest.mark.parametrize("dt", DT, ids=str)
def test_some_gradients(cuda, dt, N):
    """Each gradient by itself, and each pair, has the bits of all three; frozen operands have none."""
    import tilemaxsim_amd as tms
    ts, G = make(N, 72, 50, dt, seed=7)
    want = torch.autograd.grad(tms.gated_linear(*ts), ts, G)
    for some in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        part = [t.detach().requires_grad_(m in some) for m, t in enumerate(ts)]
        h = tms.gated_linear(*part)
        h.backward(G)
        assert all(torch.equal(t.grad, w) if m in some else t.grad is None for m, (t, w) in enumerate(zip(part, want))), some
        got = torch.autograd.grad(tms.gated_linear(*ts), [ts[m] for m in some], G)
        assert all(torch.equal(a, want[m]) for a, m in zip(got, some)), some


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -20, 2.0 ** 9])
def test_gradients_of_any_size(cuda, size):
    """fp16's narrow range: gradients as a mean over many tokens, or a loss's scale, leave them."""
    check(200, 64, 96, torch.float16, "silu", seed=4, size=size)


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_gradients_of_few_tokens(cuda, dt, size):
    """Two terms of dg and du: zeros, one large row among small ones, and infinities that stay where they are."""
    import tilemaxsim_amd as tms
    for N in (1, 40, 64):
        check(N, 64, 96, dt, "gelu", seed=6, size=size)
    ts, G = make(40, 72, 50, dt, seed=8, size=size)
    with torch.no_grad():
        G[1:] *= 2.0 ** -8
        G[5] = 0
    grads = torch.autograd.grad(tms.gated_linear(*ts), ts, G)
    close((tms.gated_linear(*ts).detach(), *grads), reference(*ts, G, "silu"), f"one large row {dt}")
    with torch.no_grad():
        G[7, 3] = math.inf
    again = torch.autograd.grad(tms.gated_linear(*ts), ts, G)
    keep = torch.arange(50, device="cuda") != 3
    assert not torch.isfinite(again[0][7]).any() and bool(torch.isfinite(again[0][torch.arange(40, device="cuda") != 7]).all())
    assert all(not torch.isfinite(w[3]).any() and bool(torch.isfinite(w[keep]).all()) for w in again[1:])


def test_empty(cuda):
    import tilemaxsim_amd as tms
    for N, F in ((0, 16), (5, 0), (0, 0)):
        x, w = torch.randn(N, 32, device="cuda", requires_grad=True), torch.randn(F, 32, device="cuda", requires_grad=True)
        h = tms.gated_linear(x, w, w * 1)
        dx, dw = torch.autograd.grad(h, (x, w), torch.ones_like(h))
        assert h.shape == (N, F) and not dx.any() and not dw.any() and dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.parametrize("dt", DT, ids=str)
def test_layouts(cuda, dt):
    """Leading dimensions, halves of one tensor, strided and unaligned operands: the contiguous call's bits."""
    import tilemaxsim_amd as tms
    (x, wg, wu), G = make(90, 64, 48, dt)
    want = tms.gated_linear(x, wg, wu)
    grads = torch.autograd.grad(want, (x, wg, wu), G)
    both = torch.cat([wg, wu]).detach().requires_grad_(True)
    h = tms.gated_linear(x.view(9, 10, 64), *both.split(48))
    assert h.shape == (9, 10, 48) and torch.equal(h.view(90, 48), want)
    dx, dw = torch.autograd.grad(h, (x, both), G.view(9, 10, 48))
    assert torch.equal(dx, grads[0]) and torch.equal(dw, torch.cat(grads[1:]))
    with torch.no_grad():
        odd = [torch.empty(t.shape[0] * 64 + 1, device="cuda", dtype=dt)[1:].view(-1, 64).copy_(t).requires_grad_(True) for t in (x, wg, wu)]
        turned = [t.t().contiguous().t().requires_grad_(True) for t in (x, wg, wu)]
    for ts in (odd, turned):
        h = tms.gated_linear(*ts)
        assert torch.equal(h, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, ts, G.t().contiguous().t()), grads))
    one = tms.gated_linear(x[0], wg, wu)
    assert one.shape == (48,)
    # a broadcast gradient, and one weight in both places
    s = torch.autograd.grad(tms.gated_linear(x, wg, wg).sum(), wg)[0]
    a, b = torch.autograd.grad(tms.gated_linear(x, wg, wg * 1).sum(), wg)[0], s
    assert a.shape == b.shape and bool(((a.double() - b.double()).abs() <= 8 * U[dt] * (a.double().abs() + a.double().abs().max())).all())


@pytest.mark.parametrize("dt", DT, ids=str)
def test_values_beyond_the_range(cuda, dt):
    """Large gates saturate without NaN; NaN and infinities stay in their rows and columns."""
    import tilemaxsim_amd as tms
    for act in ("silu", "gelu", "gelu_tanh"):
        x = torch.zeros(70, 8, device="cuda", dtype=dt)
        x[:, 0] = torch.linspace(-200, 200, 70).to(dt)
        wg, wu = torch.zeros(3, 8, device="cuda", dtype=dt), torch.ones(3, 8, device="cuda", dtype=dt)
        wg[0, 0], wg[1, 0], wg[2, 0] = 1, 100, -100
        wu[:, 0] = 0
        x[:, 1] = 0.001
        x, wg, wu = (t.requires_grad_(True) for t in (x, wg, wu))
        h = tms.gated_linear(x, wg, wu, act)
        G = torch.full_like(h, 0.01)
        close((h.detach(), *torch.autograd.grad(h, (x, wg, wu), G)), reference(x, wg, wu, G, act), f"{act} {dt}")
    (x, wg, wu), G = make(80, 64, 40, dt)
    want = tms.gated_linear(x, wg, wu).detach()
    with torch.no_grad():
        y, w = x.clone(), wg.clone()
        y[3], w[7] = math.nan, math.inf
        h = tms.gated_linear(y, w, wu)
        keep = torch.ones_like(h, dtype=torch.bool)
        keep[3], keep[:, 7] = False, False
        assert torch.equal(h[keep], want[keep]) and bool(torch.isnan(h[3]).all())


def test_differences(cuda):
    """fp32 gradients against central differences along random directions: off by the outputs' bounds over
    the step, and by a third of how far the differences at h and 2h are from each other."""
    import tilemaxsim_amd as tms
    for act in ("silu", "gelu", "gelu_tanh"):
        ts, G = make(70, 40, 24, torch.float32, seed=6)
        grads = torch.autograd.grad(tms.gated_linear(*ts, act), ts, G)
        noise = float((reference(*ts, G, act)[0][1] * G.double().abs()).sum())
        with torch.no_grad():
            for m in range(3):
                way = torch.randn_like(ts[m])

                def f(h):
                    y = list(ts)
                    y[m] = ts[m] + h * way
                    return float((tms.gated_linear(*y, act).double() * G).sum())

                h = 2.0 ** -7
                one, two = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
                rounding = float((grads[m].double().abs() * way.abs()).sum()) * 2.0 ** -16
                assert abs(float((grads[m].double() * way).sum()) - one) <= abs(one - two) + noise / h + rounding, (act, m)


def test_streams_and_graphs(cuda):
    """Another stream than the tensors' own; captured passes follow their inputs, replay by replay."""
    import tilemaxsim_amd as tms
    for dt, N in ((torch.float16, 200), (torch.bfloat16, 3), (torch.float32, 70)):
        (x, wg, wu), G = make(N, 77, 50, dt)

        def step():
            h = tms.gated_linear(x, wg, wu, "gelu")
            return (h, *torch.autograd.grad(h, (x, wg, wu), G))

        want = [t.detach().clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [t.detach().clone() for t in step()]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = [t.detach() for t in step()]
        for i in range(4):
            with torch.no_grad():
                x.mul_(0.9)
                G.mul_(1.3)
            graph.replay()
            got = [t.clone() for t in kept]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b.detach()) for a, b in zip(got, step()))
