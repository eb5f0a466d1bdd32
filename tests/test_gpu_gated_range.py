"""The gated projection's gradients in fp16 where dg and du leave its range, above or below.

Tolerances as in test_gpu_gated.py but for what is below fp16's normal numbers. dg and du of a token are held times a
power of two that brings a bound of them, 1.2 max |dh| |x| max |W| with the norms of the token's row and of the weights'
rows, to 2^14 to 2^15: what is lost is half of fp16's smallest number over that power, 2^-25 2^-14 1.2 max |dh| |x| |W|, less
than 2^-38 of the product. The weights' gradients take x over that power, times one that brings the largest bound times |x| to
2^14 to 2^15: 2^-25 lost of it, over 2^14 2^14 and times up to 2^15 of a bound, 2^-38 1.2 of the largest max |dh| |x|^2 |W| for each token."""
import math

import pytest
import torch

from test_gpu_gated import E, TINY, U, functions, make

pytestmark = pytest.mark.gpu
F16 = torch.float16


@torch.no_grad()
def reference(x, wg, wu, G, act):
    """dx, dWg and dWu in 64 bits, and how far each may be off."""
    dt = x.dtype
    u_ = U[dt]
    held = u_ if x.shape[0] > 64 else u_ * u_
    x, wg, wu, G = (t.detach().double() for t in (x, wg, wu, G))
    (N, d), F = x.shape, wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = E * (d + 4) * (x.abs() @ wg.abs().T), E * (d + 4) * (x.abs() @ wu.abs().T)
    a, slope = functions(g, act)
    ea = 1.13 * eg + 2.0 ** -20 * a.abs()
    dg, du = G * u * slope, G * a
    most = G.abs().amax(1, keepdim=True) * x.norm(dim=1, keepdim=True) * max(float(wg.norm(dim=1).max()), float(wu.norm(dim=1).max()))
    floor = 2.0 ** -38 * most
    edg = G.abs() * (slope.abs() * eu + u.abs() * (0.8 * eg + 2.0 ** -20 * (1 + g.abs()))) + held * dg.abs() + floor
    edu = G.abs() * ea + held * du.abs() + floor
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + E * (2 * F + 4) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    low = N * 2.0 ** -37 * float((most * x.norm(dim=1, keepdim=True)).max())
    dwg, dwu = dg.T @ x, du.T @ x
    edwg = edg.T @ x.abs() + E * (N + 4) * (dg.abs().T @ x.abs()) + low
    edwu = edu.T @ x.abs() + E * (N + 4) * (du.abs().T @ x.abs()) + low
    return [(r, e + u_ * r.abs() + TINY[dt]) for r, e in ((dx, edx), (dwg, edwg), (dwu, edwu))]


def check(ts, G, act, what, names=("dx", "dw_gate", "dw_up")):
    import tilemaxsim_amd as tms
    print(what, flush=True)
    grads = torch.autograd.grad(tms.gated_linear(*ts, act), ts, G)
    for got, (want, off), name in zip(grads, reference(*ts, G, act), ("dx", "dw_gate", "dw_up")):
        if name not in names:
            continue
        assert float(want.abs().max()) < 65504, "a case of finite gradients"
        assert bool(torch.isfinite(got).all()), f"{what}: {name} is not finite"
        over = float(((got.double() - want).abs() / off).max())
        assert over <= 1.0, f"{what}: {name} is {over:.3g} times its bound off"
    return grads


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("N,d,F", [(3, 64, 96), (64, 72, 50), (200, 64, 96), (200, 77, 50), (300, 264, 600)])
def test_large_factors(cuda, N, d, F, act):
    """|u| up to 120,000, beyond fp16's range as h is there, with gradients that are not."""
    ts, G = make(N, d, F, F16, seed=N + d, size=2.0 ** -14)
    x, wg, wu = ts
    with torch.no_grad():
        x[:, 0], wg[:, 0] = 200, 0
        wu[:, 0] = torch.linspace(-600, 600, F, device="cuda").to(F16)
    check(ts, G, act, f"u of 120,000, {N} x {d} x {F} {act}")
    with torch.no_grad():  # dg itself beyond the range, its products with small weights not
        wg.mul_(2.0 ** -8)
        G.mul_(2.0 ** 14)
    check(ts, G, act, f"dg of 120,000, {N} x {d} x {F} {act}", names=("dx",))
    with torch.no_grad():  # the same of g: both factors change places
        x[:, 0], wu[:, 0] = 200, 0
        wg[:, 0] = torch.linspace(-600, 600, F, device="cuda").to(F16)
        G.mul_(2.0 ** -14)
    check(ts, G, act, f"g of 120,000, {N} x {d} x {F} {act}")


@pytest.mark.parametrize("N,d,F", [(3, 64, 96), (40, 64, 96), (64, 77, 50), (200, 64, 96), (200, 77, 50), (300, 264, 600)])
@pytest.mark.parametrize("below", [2.0 ** -14, 2.0 ** -18, 2.0 ** -22])
@pytest.mark.parametrize("size", [2.0 ** 5, 1.0, 2.0 ** -4])
def test_rows_far_below_others(cuda, size, below, N, d, F):
    """Tokens whose gradients are far below the largest: each row's own gradient keeps its digits."""
    ts, G = make(N, d, F, F16, seed=5, size=size)
    with torch.no_grad():
        G[1::3] *= below
        G[2::3] *= math.sqrt(below)
        if N > 3:
            G[5] = 0
    check(ts, G, "silu", f"rows of {below} below {size}, {N} x {d} x {F}")


@pytest.mark.parametrize("N", [40, 200])
def test_values_of_any_size(cuda, N):
    """Small and large inputs and weights, rows and columns of zeros; a row that is not finite stays by itself."""
    import tilemaxsim_amd as tms
    for xs, ws in ((2.0 ** -10, 1.0), (1.0, 2.0 ** -10), (2.0 ** -12, 2.0 ** -10), (2.0 ** 6, 2.0 ** -2)):
        ts, G = make(N, 72, 50, F16, seed=8, size=2.0 ** -6)
        with torch.no_grad():
            ts[0].mul_(xs)
            ts[1].mul_(ws)
            ts[2].mul_(ws)
            ts[0][3], ts[1][7], ts[2][9] = 0, 0, 0
        check(ts, G, "gelu", f"x of {xs}, weights of {ws}, {N}")
    ts, G = make(N, 72, 50, F16, seed=8)
    with torch.no_grad():
        G[6] = 0
        G[6, 3] = math.inf  # the row's only gradient
        ts[0][11, 4] = math.nan
    dx, dwg, dwu = torch.autograd.grad(tms.gated_linear(*ts), ts, G)
    rows = torch.ones(N, dtype=torch.bool, device="cuda")
    rows[6] = rows[11] = False
    assert bool(torch.isfinite(dx[rows]).all()) and not torch.isfinite(dx[6]).any() and bool(torch.isnan(dx[11]).all())
    assert bool(torch.isnan(dwg).all()) and bool(torch.isnan(dwu).all())
    with torch.no_grad():
        clean = ts[0].clone()
        clean[11, 4] = 0.5
    ts = [clean.detach().requires_grad_(True), *ts[1:]]
    dx, dwg, dwu = torch.autograd.grad(tms.gated_linear(*ts), ts, G)
    columns = torch.arange(50, device="cuda") != 3
    assert bool(torch.isfinite(dwg[columns]).all()) and bool(torch.isfinite(dwu[columns]).all())
    assert not torch.isfinite(dwg[3]).any() and not torch.isfinite(dwu[3]).any()
