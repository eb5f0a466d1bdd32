"""The global gradient norm and clipping against float64.

Tolerances. The norm: squares are added in 64 bits, so what is left is the rounding of the
root to fp32, 2^-24 of it, doubled for the fp64 sum. A clipped value: the factor is one fp32
division of rounded operands (4 roundings with the norm's and the 1e-6's), the product one
more, 6 * 2^-24 of the value in all, and a rounding to its type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16, torch.float16]
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def _norm(ts, p=2.0):
    if p == math.inf:
        return max([float(t.double().abs().max()) for t in ts if t.numel()], default=0.0)
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def _close(got, ref, dt):
    off = (got.double() - ref).abs()
    lim = (6 * 2.0 ** -24 + ROUND[dt]) * ref.abs() + TINY[dt] + 1e-40
    return bool((off <= lim).all())


def _tensors(sizes, seed=0, dts=DT):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * (0.1 + i % 5)).to(dts[i % len(dts)]) for i, s in enumerate(sizes)]


SIZES = {
    "one": [(1,)],
    "vector ends": [(7,), (8,), (9,), (2047,), (2049,), (3, 5)],
    "chunk ends": [(16384,), (16383,), (16385,), (49153,), (0,), (4, 0, 3)],
    "many": [(1 + (i * 37) % 1000,) for i in range(1000)],  # several launches
    "large": [(3000, 1001), (1 << 22,)],
}


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("kind", list(SIZES))
def test_norm_and_clip(cuda, kind, p):
    import tilemaxsim_amd as tms
    print(f"clip {kind} p={p}", flush=True)
    ts = _tensors(SIZES[kind], seed=len(kind))
    want = _norm(ts, p)
    got = tms.grad_norm(ts, p)
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    assert abs(float(got) - want) <= 2 * 2.0 ** -24 * want
    for most in (want * 0.3, want * 1.5):
        k = min(1.0, most / (want + 1e-6))
        refs = [t.double() * k for t in ts]
        out = [torch.full(t.shape, 7.0, device="cuda", dtype=DT[(i + 1) % 3]) for i, t in enumerate(ts)]
        before = [t.clone() for t in ts]
        n = tms.clip_grad_norm_(ts, most, p, out=out)
        assert torch.equal(n, got)
        assert all(torch.equal(a, b) for a, b in zip(ts, before)), "gradients changed beside out"
        assert all(_close(o, r, o.dtype) for o, r in zip(out, refs))
        mine = [t.clone() for t in ts]
        assert torch.equal(tms.clip_grad_norm_(mine, most, p), got)
        if k == 1.0:
            assert all(torch.equal(a, b) for a, b in zip(mine, ts))
        assert all(_close(o, r, o.dtype) for o, r in zip(mine, refs))


def test_views_at_any_address(cuda):
    """Gradients that are pieces of one buffer, at every alignment; nothing beside them changes."""
    import tilemaxsim_amd as tms
    for dt in DT:
        flat = torch.randn(9000, device="cuda").to(dt)
        keep = flat.clone()
        cuts = [(1, 8), (10, 523), (524, 525), (530, 2700), (2703, 8999)]
        views = [flat[a:b] for a, b in cuts]
        want = _norm(views)
        assert abs(float(tms.grad_norm(views)) - want) <= 2 * 2.0 ** -24 * want
        tms.clip_grad_norm_(views, want / 2)
        for a, b in cuts:
            assert _close(flat[a:b], keep[a:b].double() * (want / 2 / (want + 1e-6)), dt)
        beside = torch.ones(9000, dtype=torch.bool)
        for a, b in cuts:
            beside[a:b] = False
        assert torch.equal(flat[beside.cuda()], keep[beside.cuda()])


def test_range(cuda):
    """Squares that fp32 cannot hold, and norms that are zero, NaN or infinite."""
    import tilemaxsim_amd as tms
    big, small = torch.full((1000,), 1e30, device="cuda"), torch.full((1000,), 1e-30, device="cuda")
    for t in (big, small):
        want = _norm([t])
        assert abs(float(tms.grad_norm(t)) - want) <= 2 * 2.0 ** -24 * want
    x = big.clone()
    tms.clip_grad_norm_(x, 1.0)
    assert _close(x, big.double() / _norm([big]), torch.float32)
    zero = torch.zeros(5, device="cuda")
    assert float(tms.clip_grad_norm_(zero, 1.0)) == 0 and bool((zero == 0).all())
    for bad in (math.nan, math.inf, -math.inf):
        for p in (2.0, math.inf):
            t = torch.ones(70_000, device="cuda")
            t[65_000] = bad
            other = torch.ones(3, device="cuda")
            with pytest.raises(RuntimeError, match="norm of the gradients"):
                tms.clip_grad_norm_([other, t], 1.0, p, error_if_nonfinite=True)
            assert bool((other == 1).all())
            n = tms.clip_grad_norm_([other, t], 1.0, p)
            assert math.isnan(float(n)) if math.isnan(bad) else math.isinf(float(n))
            assert bool(torch.isnan(other).all()) if math.isnan(bad) else bool((other == 0).all())
            assert math.isnan(float(t[65_000]))  # infinity times 0


def test_lists(cuda):
    """None entries, strided gradients, nothing at all, and every run's bits alike."""
    import tilemaxsim_amd as tms
    a, b = torch.randn(300, 200, device="cuda"), torch.randn(64, 64, device="cuda").half()
    want = _norm([a, b])
    assert abs(float(tms.grad_norm([None, a, None, b])) - want) <= 2 * 2.0 ** -24 * want
    wide = torch.randn(300, 400, device="cuda")
    view = wide[:, ::2]
    view.copy_(a)
    rest = wide[:, 1::2].clone()
    tms.clip_grad_norm_([view.t(), None, b], want / 4)
    assert _close(view, a.double() * (want / 4 / (want + 1e-6)), torch.float32)
    assert torch.equal(wide[:, 1::2], rest)
    into = torch.empty(200, 300, device="cuda").t()
    tms.clip_grad_norm_(a, 1.0, out=into)
    assert _close(into, a.double() / (_norm([a]) + 1e-6), torch.float32)
    assert float(tms.grad_norm([])) == 0 and float(tms.clip_grad_norm_([None], 1.0)) == 0
    runs = {float(tms.grad_norm(_tensors(SIZES["many"]))) for _ in range(5)}
    assert len(runs) == 1


def test_graph(cuda):
    """A captured clip follows its gradients from replay to replay."""
    import tilemaxsim_amd as tms
    ts = _tensors([(1000,), (33, 77), (20_000,)])
    out = [torch.empty_like(t) for t in ts]
    tms.clip_grad_norm_(ts, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = tms.clip_grad_norm_(ts, 1.0, out=out)
    for i in range(4):
        for t in ts:
            t.mul_(1.7)
        graph.replay()
        got, kept = norm.clone(), [o.clone() for o in out]
        torch.cuda.synchronize()
        assert torch.equal(got, tms.clip_grad_norm_(ts, 1.0, out=out))
        assert all(torch.equal(a, b) for a, b in zip(kept, out))
