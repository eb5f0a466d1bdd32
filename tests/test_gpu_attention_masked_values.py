"""Attention under prefix masks with NaN and infinities in tokens of the same text that a row does not see: they take no
part in its output or gradients. Bounds are those of test_gpu_attention.py."""
import math

import pytest
import torch

from test_gpu_attention import DT, make, reference

pytestmark = pytest.mark.gpu


def poisoned(ts, G, rows, value, which):
    """Copies with `value` in some elements of the given tokens of q, k, v or the gradient."""
    ts = [t.detach().clone() for t in ts]
    G = G.clone()
    for name, t in zip("qkvG", (*ts, G)):
        if name in which:
            t[rows, :, 3::7] = value
            t[rows[-1:]] = value
    return [t.requires_grad_(True) for t in ts], G


def agree(got, want, off, keep, what):
    for x, y, o, name in zip(got, want, off, ("out", "dq", "dk", "dv")):
        x, y, o = x[keep[name]], y[keep[name]], o[keep[name]]
        assert bool(torch.isfinite(x).all()), f"{what}: {name} is not finite"
        over = float(((x.double() - y).abs() / o.clamp(min=1e-300)).max()) if x.numel() else 0.0
        assert over <= 1.0, f"{what}: {name} is {over:.3g} times its bound off"


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("lens,H,KV,D,how", [
    ([70, 9, 200], 2, 1, 64, {}), ([70, 9, 200], 4, 2, 32, dict(cap=5.0)), ([33] * 20, 2, 2, 96, {}), ([16] * 30, 1, 1, 128, dict(slopes=0.1)),
    ([1500, 1300], 24, 24, 64, {}), ([1300, 1500], 24, 24, 128, dict(cap=30.0)), ([2500], 24, 24, 64, dict(slopes=0.02)), ([130, 600], 12, 1, 32, dict(slopes=0.0))])
@pytest.mark.parametrize("prefix", [0, 7])
def test_unseen_tokens_take_no_part(cuda, lens, H, KV, D, how, prefix, dt):
    """The last tokens of each text are bad. Rows before them do not see their keys and values; their own keys get gradients
    from rows that are bad, and from none before."""
    import tilemaxsim_amd as tms
    ts, offsets, G = make(lens, H, KV, D, dt, seed=D)
    how = {**how, "prefix": prefix}
    if "slopes" in how:
        how["slopes"] = torch.full((H,), how["slopes"], device="cuda")
    bad = [n - max(1, n // 5) for n in lens]  # from here on
    rows = torch.cat([torch.arange(o + b, o + n) for o, b, n in zip(offsets.tolist(), bad, lens)]).cuda()
    seen = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    seen[rows] = True
    # what the rows before the bad ones give, by themselves
    cut = torch.cat([torch.arange(o, o + b) for o, b in zip(offsets.tolist(), bad)]).cuda()
    short = torch.tensor([0, *bad]).cumsum(0)
    part = [t.detach()[cut].requires_grad_(True) for t in ts]
    want, off = reference(*part, short, G[cut], **how)
    for value in (math.nan, math.inf):
        # keys and values: outputs and dq of the rows before
        print(lens, H, D, dt, how, value, flush=True)
        xs, g = poisoned(ts, G, rows, value, "kv")
        out = tms.packed_attention(*xs, offsets, **how)
        grads = torch.autograd.grad(out, xs, g)
        whole = [torch.zeros_like(t, dtype=torch.float64) for t in (out, *xs)]
        bounds = [torch.zeros_like(t) for t in whole]
        for w, b, x, o in zip(whole, bounds, want, off):
            w[cut], b[cut] = x, o
        keep = dict(out=~seen, dq=~seen, dk=rows[:0], dv=rows[:0])
        agree((out.detach(), *grads), whole, bounds, keep, f"bad keys and values, {value}")
    # queries and gradients of tokens behind the prefix: keys behind those do not get any of them
    first = [min(prefix, n - 1) for n in lens]
    ends = [min(n - 1, f + max(1, n // 5)) for f, n in zip(first, lens)]
    rows = torch.cat([torch.arange(o + f, o + e) for o, f, e in zip(offsets.tolist(), first, ends)]).cuda()
    if rows.numel() == 0:
        return
    behind = torch.cat([torch.arange(o + e, o + n) for o, e, n in zip(offsets.tolist(), ends, lens)]).cuda()
    clean = [t.detach().clone() for t in ts]
    zero = G.clone()
    zero[rows] = 0  # rows that a key does not see give it nothing, whatever they are
    want, off = reference(*clean, offsets, zero, **how)
    for value in (math.nan, math.inf):
        xs, g = poisoned(ts, G, rows, value, "qG")
        out = tms.packed_attention(*xs, offsets, **how)
        grads = torch.autograd.grad(out, xs, g)
        agree((out.detach(), *grads), want, off, dict(out=behind, dq=behind, dk=behind, dv=behind), f"bad queries and gradients, {value}")


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [0, 5, 40, 100, 130])
def test_one_token_anywhere(cuda, prefix, D, dt):
    """A single bad token at any place of a tile, and prefixes that end in one."""
    import tilemaxsim_amd as tms
    n = 300
    ts, offsets, G = make([n], 2, 1, D, dt, seed=prefix)
    want, off = reference(*ts, offsets, G, prefix=prefix)
    none = torch.arange(0, device="cuda")
    for b in (prefix, prefix + 1, prefix + 20, 63 + prefix // 64 * 64, 127 + prefix // 128 * 64, 255, 298):
        print(prefix, D, dt, b, flush=True)
        rows, before, behind = torch.tensor([b], device="cuda"), torch.arange(b, device="cuda"), torch.arange(b + 1, n, device="cuda")
        for which in ("k", "v"):
            xs, g = poisoned(ts, G, rows, math.nan, which)
            out = tms.packed_attention(*xs, offsets, prefix=prefix)
            grads = torch.autograd.grad(out, xs, g)
            agree((out.detach(), *grads), want, off, dict(out=before, dq=before, dk=none, dv=none), f"bad {which} of {b}")
        g0 = G.clone()
        g0[b] = 0
        want0, off0 = reference(*ts, offsets, g0, prefix=prefix)
        for which in ("q", "G"):
            xs, g = poisoned(ts, G, rows, math.nan, which)
            out = tms.packed_attention(*xs, offsets, prefix=prefix)
            grads = torch.autograd.grad(out, xs, g)
            others = torch.cat([before, behind])
            agree((out.detach(), *grads), want0, off0, dict(out=others, dq=others, dk=behind, dv=behind), f"bad {which} of {b}")


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("H,KV,D", [(1, 1, 64), (4, 2, 32), (2, 1, 128), (24, 24, 96)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_seen_and_unseen(cuda, H, KV, D, value, dt):
    """A bad value that a row sees, in one column, and another that it does not, in another column next to it."""
    import tilemaxsim_amd as tms
    n = 3001 if H == 24 else 300
    ts, offsets, G = make([n], H, KV, D, dt, seed=H)
    q, k, v = ts
    want, off = reference(*ts, offsets, G, prefix=0)
    with torch.no_grad():
        v2 = v.clone()
        v2[10, :, 3], v2[120, :, 5] = value, value
    out = tms.packed_attention(q, k, v2, offsets, prefix=0)
    fine = torch.ones_like(out, dtype=torch.bool)
    fine[10:, :, 3] = fine[120:, :, 5] = False
    agree((out.detach(),), want[:1], off[:1], dict(out=fine), f"values {D} {dt}")
    assert not torch.isfinite(out[10:, :, 3]).any() and not torch.isfinite(out[120:, :, 5]).any()
    with torch.no_grad():
        g = G.clone()
        g[120, :, 3], g[70, :, 5] = value, value
    grads = torch.autograd.grad(tms.packed_attention(q, k, v, offsets, prefix=0), ts, g)
    # rows 70 and 120 reach the keys up to them, in their own columns of dv, and in all of dk
    fine = torch.ones_like(v, dtype=torch.bool)
    fine[:121, :, 3] = fine[:71, :, 5] = False
    g0 = G.clone()
    g0[120], g0[70] = 0, 0
    without, off0 = reference(*ts, offsets, g0, prefix=0)
    behind = torch.arange(121, n, device="cuda")
    agree((out.detach(), *grads), without, off0, dict(out=behind[:0], dq=behind, dk=behind, dv=behind), f"gradients {D} {dt}")
    agree((grads[2],), [want[3]], [off[3]], dict(out=fine), f"gradients, dv {D} {dt}")
    assert not torch.isfinite(grads[2][:121, :, 3]).any() and not torch.isfinite(grads[2][:71, :, 5]).any() and not torch.isfinite(grads[1][:121]).any()


@pytest.mark.parametrize("dt", DT, ids=str)
def test_seen_tokens_do(cuda, dt):
    """A value that a row sees reaches it where it stands: in its column of the output, infinite with its sign."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([50], 1, 1, 64, dt, seed=3)
    want, off = reference(q, k, v, offsets, G, prefix=0)
    with torch.no_grad():
        v2 = v.clone()
        v2[20, 0, 5], v2[30, 0, 6], v2[30, 0, 7] = math.nan, math.inf, -math.inf
    out = tms.packed_attention(q, k, v2, offsets, prefix=0).detach()
    assert bool(torch.isnan(out[20:, 0, 5]).all()) and bool((out[30:, 0, 6] == math.inf).all()) and bool((out[30:, 0, 7] == -math.inf).all())
    expect = torch.ones(50, 1, 64, dtype=torch.bool, device="cuda")
    expect[20:, 0, 5] = expect[30:, 0, 6] = expect[30:, 0, 7] = False
    agree((out,), want[:1], off[:1], dict(out=expect), f"seen {dt}")
