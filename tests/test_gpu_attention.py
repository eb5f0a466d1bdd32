"""Attention over packed texts against float64, text by text and head by head.

Tolerances, for each element, from the arithmetic. u is half a step of the inputs' type (fp32:
nothing is rounded between the products), e = 2^-23 for a rounding of an fp32 sum (twice half a step).
 * A score: sums of D products, 3 roundings more, in natural units: ex = e (D + 6) scale <|q|, |k|> +
   3 e |x|, and under a cap what tanh is off by, cap 2^-20 (16-bit kernels: from an exponential and a
   reciprocal of 2^-22 each; fp32: 2^-21); of |x| and not of the cap in caps above 64, 2^-16 of it (where it is formed so, |x| is
   at least 2^-4 of the cap; below, it is off by 2^-22 of itself). P is then off by rp = 2 max ex + e (n + 4) of itself (its sum is, too), and by u more when
   it is rounded; in fp16 also by 2^-25 of the row's largest P, where it is below fp16's normal numbers.
 * out: (u + rp) sum P |v| + u |out|, and dv likewise with |do| in the place of |v|.
 * dP: e (D + 1) <|do|, |v|>. delta: from an out before its rounding, (u + rp + u^2) sum P <|do|, |v|> + e (D + 1) of that.
   dS: P (both) + (2 rp + u + 6 e) P (|dP| + |delta|), and under a cap P (|dP| + |delta|) 2^-19 for 1 - tanh^2.
 * dq, dk: the products of those with |k|, |q| times scale, e (n + 1) sum |dS| |k| scale, and u of the result.
 * What is below the type's normal numbers: half of its smallest one.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
LAST = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -140}
E = 2.0 ** -23


def make(lens, H, KV, D, dt, seed=0, front=0, behind=0, fused=False, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = front + sum(lens) + behind
    x = torch.randn(T, H + 2 * KV, D, generator=g, device="cuda")
    x[:, :H] *= 1.5 * scale
    x = x.to(dt)
    q, k, v = x.split([H, KV, KV], 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    offsets = torch.tensor([0] + list(lens)).cumsum(0) + front
    G = torch.randn(T, H, D, generator=g, device="cuda").to(dt)
    return [t.detach().requires_grad_(True) for t in (q, k, v)], offsets, G


@torch.no_grad()
def reference(q, k, v, offsets, G, prefix=None, scale=None, cap=None, slopes=None):
    """Outputs, gradients, and how far each may be off."""
    T, H, D = q.shape
    many = H // k.shape[1]
    dt = q.dtype
    u, last, tiny = U[dt], LAST[dt], TINY[dt]
    scale = 1 / math.sqrt(D) if scale is None else scale
    Q, K, V, G = (t.detach().double() for t in (q, k, v, G))
    res = [torch.zeros_like(t) for t in (Q, Q, K, V)]
    off = [torch.zeros_like(t) for t in (Q, Q, K, V)]
    for b in range(offsets.numel() - 1):
        lo, hi = int(offsets[b]), int(offsets[b + 1])
        n = hi - lo
        if n <= 0:
            continue
        a = slice(lo, hi)
        i = torch.arange(n, device="cuda")
        sees = torch.ones(n, n, dtype=torch.bool, device="cuda")
        if prefix is not None:
            sees = (i[None, :] <= i[:, None]) | (i[None, :] < (prefix if isinstance(prefix, int) else int(prefix[b])))
        for h in range(H):
            kv = h // many
            qh, kh, vh, gh = Q[a, h], K[a, kv], V[a, kv], G[a, h]
            x = scale * qh @ kh.T
            ex = E * (D + 6) * scale * (qh.abs() @ kh.abs().T)
            slope = torch.ones_like(x)
            if cap:
                t = torch.tanh(x / cap)
                x, slope = cap * t, 1 - t * t
                ex = ex + (x.abs() * 2.0 ** -16 if cap > 64 else cap * 2.0 ** (-21 if dt == torch.float32 else -20))
            if slopes is not None:
                x = x - float(slopes[h]) * (i[:, None] - i[None, :]).abs()
            ex = torch.where(sees, ex + 3 * E * x.abs(), 0.0)
            P = torch.softmax(x.masked_fill(~sees, -math.inf), 1)
            rp = 2 * ex.amax(1, keepdim=True) + E * (n + 4)
            low = 2.0 ** -25 * P.amax(1, keepdim=True) if dt == torch.float16 else 0.0
            eP = ((u + rp) * P + low) * sees
            o = P @ vh
            res[0][a, h] = o
            off[0][a, h] = eP @ vh.abs() + last * o.abs() + tiny
            dP, both = gh @ vh.T, gh.abs() @ vh.abs().T
            delta = (P * dP).sum(1, keepdim=True)
            eD = ((eP + u * u * P) * both).sum(1, keepdim=True) + E * (D + 1) * (P * both).sum(1, keepdim=True)
            S = P * (dP - delta)
            eS = P * (E * (D + 1) * both + eD) + (2 * rp + u + 6 * E) * P * (dP.abs() + delta.abs())
            eS = eS * slope + (P * (dP.abs() + delta.abs()) * 2.0 ** -19 if cap else 0.0)
            S = S * slope
            res[1][a, h] = scale * S @ kh
            res[2][a, kv] += scale * S.T @ qh
            res[3][a, kv] += P.T @ gh
            off[1][a, h] = scale * (eS + E * (n + 1) * S.abs()) @ kh.abs()
            off[2][a, kv] += scale * (eS + E * (n * many + 1) * S.abs()).T @ qh.abs()
            off[3][a, kv] += (eP + E * (n * many + 1) * P).T @ gh.abs()
        for m in (1, 2, 3):
            off[m][a] += last * res[m][a].abs() + tiny
    return res, off


def close(got, want, off, what):
    for x, y, o, name in zip(got, want, off, ("out", "dq", "dk", "dv")):
        assert not torch.isnan(x).any(), f"{what}: NaN in {name}"
        d = (x.double() - y).abs()
        over = float((d / o.clamp(min=1e-300)).max()) if x.numel() else 0.0
        assert over <= 1.0, f"{what}: {name} is {over:.3g} times its bound off"


def check(q, k, v, offsets, G, what, **how):
    import tilemaxsim_amd as tms
    print(what, flush=True)
    out = tms.packed_attention(q, k, v, offsets, **how)
    grads = torch.autograd.grad(out, (q, k, v), G)
    assert out.dtype == q.dtype and [g.dtype for g in grads] == [q.dtype] * 3
    want, off = reference(q, k, v, offsets, G, **how)
    close((out.detach(), *grads), want, off, what)
    with torch.no_grad():
        assert torch.equal(tms.packed_attention(q, k, v, offsets, **how), out)
    again = torch.autograd.grad(tms.packed_attention(q, k, v, offsets, **how), (q, k, v), G)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "a run's bits differ"
    return out.detach(), grads


DT = [torch.bfloat16, torch.float16, torch.float32]
LENS = {
    "one token": [1],
    "short": [3, 1, 0, 2, 17, 0, 0, 16, 15],
    "tile ends": [63, 64, 65, 31, 32, 33, 127, 128, 129],
    "long": [700, 5, 321],
    "many": [(i * 37) % 41 for i in range(130)],
}


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lens", list(LENS))
def test_texts(cuda, lens, D, dt):
    qkv, offsets, G = make(LENS[lens], 3, 3, D, dt, seed=D)
    check(*qkv, offsets, G, f"texts {lens} {D} {dt}")


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["causal", "prefix", "cap", "bias", "all"])
def test_masks_and_scores(cuda, kind, D, dt):
    lens = [70, 1, 0, 129, 200, 33]
    qkv, offsets, G = make(lens, 4, 4, D, dt, seed=len(kind), scale=3.0)
    how = {}
    if kind == "causal":
        how["prefix"] = 0
    if kind in ("prefix", "all"):
        how["prefix"] = torch.tensor([20, 0, 3, 65, 200, 1000])
    if kind in ("cap", "all"):
        how["cap"] = 4.0
    if kind in ("bias", "all"):
        how["slopes"] = torch.tensor([0.5, 0.0, 2.0 ** -8, 8.0], device="cuda")
    if kind == "causal":
        out, _ = check(*qkv, offsets, G, f"{kind} {D} {dt}", prefix=torch.zeros(6, dtype=torch.int32, device="cuda"))
        import tilemaxsim_amd as tms
        assert torch.equal(out, tms.packed_attention(*qkv, offsets, prefix=0))
    else:
        check(*qkv, offsets, G, f"{kind} {D} {dt}", **how)


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("H,KV", [(4, 1), (6, 2), (12, 12), (1, 1)])
def test_shared_heads_of_one_projection(cuda, H, KV, dt):
    qkv, offsets, G = make([90, 200, 0, 7], H, KV, 64, dt, fused=True, front=3, behind=6)
    check(*qkv, offsets, G, f"shared {H} {KV} {dt}", prefix=torch.tensor([0, 100, 0, 7]), slopes=torch.full((H,), 0.1, device="cuda"))


@pytest.mark.parametrize("dt", DT, ids=str)
def test_layouts(cuda, dt):
    """Heads outside tokens, odd strides, addresses off 16 bytes, expanded heads: the contiguous call's bits."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([50, 80], 4, 2, 64, dt)
    want = tms.packed_attention(q, k, v, offsets)
    grads = torch.autograd.grad(want, (q, k, v), G)
    with torch.no_grad():
        heads_out = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
        odd = [torch.empty(130, x.shape[1], 67, device="cuda", dtype=dt)[..., 1:65].copy_(x) for x in (q, k, v)]
        wide = [torch.empty(130, x.shape[1], 128, device="cuda", dtype=dt)[..., ::2].copy_(x) for x in (q, k, v)]
    for name, xs in (("heads outside", heads_out), ("odd", odd), ("every other", wide)):
        xs = [x.detach().requires_grad_(True) for x in xs]
        out = tms.packed_attention(*xs, offsets.cuda())
        assert torch.equal(out, want), name
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, xs, G.transpose(0, 1).contiguous().transpose(0, 1)), grads)), name
    one = [x[:, :1].detach().requires_grad_(True) for x in (k, v)]
    out = tms.packed_attention(q, one[0].expand(-1, 2, -1), one[1].expand(-1, 2, -1), offsets)
    two = tms.packed_attention(q, *one, offsets)
    assert torch.equal(out, two)
    dk = torch.autograd.grad(out, one, G)
    want, off = reference(q, *one, offsets, G)
    u = LAST[dt]  # both heads' gradients are rounded, and so is their sum
    for got, w, o in zip(dk, want[2:], off[2:]):
        assert bool(((got.double() - w).abs() <= 2 * o + 4 * u * o.amax() + u * w.abs() * 4).all())


@pytest.mark.parametrize("dt", DT, ids=str)
def test_nothing_of_other_texts_is_seen(cuda, dt):
    """NaN and infinities in one text, and in rows of none, stay there."""
    import tilemaxsim_amd as tms
    lens = [70, 40, 100]
    (q, k, v), offsets, G = make(lens, 2, 1, 64, dt, front=2, behind=9)
    want = tms.packed_attention(q, k, v, offsets)
    grads = torch.autograd.grad(want, (q, k, v), G)
    bad = torch.ones(221, dtype=torch.bool, device="cuda")
    bad[2:72] = bad[112:212] = False
    for value in (math.nan, math.inf):
        xs = [torch.where(bad[:, None, None], value, x).to(dt).detach().requires_grad_(True) for x in (q, k, v)]
        out = tms.packed_attention(*xs, offsets)
        got = torch.autograd.grad(out, xs, torch.where(bad[:, None, None], value, G).to(dt))
        for a, b in zip((out, *got), (want, *grads)):
            assert torch.equal(a[~bad], b[~bad])
        for a in (out, *got):
            assert bool((a[:2] == 0).all()) and bool((a[212:] == 0).all())
            assert not bool(torch.isfinite(a[72:112]).all())


def test_no_tokens_and_no_texts(cuda):
    import tilemaxsim_amd as tms
    for T, offsets in ((0, [0]), (0, [0, 0, 0]), (5, [0]), (5, [5, 5]), (5, [3])):
        q, k = (torch.randn(T, h, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (2, 1))
        out = tms.packed_attention(q, k, k * 2, torch.tensor(offsets))
        dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
        assert out.shape == q.shape and not out.any() and not dq.any() and not dk.any() and dk.shape == k.shape


def test_offsets_that_descend_stay_inside(cuda):
    """Offsets on the GPU are not looked over: bad ones give some result, within the tensors."""
    import tilemaxsim_amd as tms
    big = torch.full((300 + 64, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    for offsets in ([0, 200, 100, 300], [-50, 20, 4000], [300, 0], [5, 1 << 40, -(1 << 40), 9]):
        print(offsets, flush=True)
        q = torch.randn(300, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        o = torch.tensor(offsets, device="cuda")
        out = tms.packed_attention(q, q * 1, q * 1, o, prefix=torch.full((len(offsets) - 1,), -7, device="cuda"))
        torch.autograd.grad(out, q, torch.ones_like(out))
    torch.cuda.synchronize()
    assert bool((big == 7).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=str)
def test_gradients_of_any_size(cuda, dt):
    """fp16's narrow range: gradients of 2^-14 and 2^9 and one row far above the others."""
    (q, k, v), offsets, G = make([300], 1, 1, 64, dt, seed=3)
    for size in (2.0 ** -14, 1.0, 2.0 ** 9):
        g = G * size
        check(q, k, v, offsets, g, f"sized {size} {dt}")
        h = G * size * 2.0 ** -6
        h[130] = g[130]
        check(q, k, v, offsets, h, f"one row {size} {dt}")


def test_differences(cuda):
    """fp32 gradients against differences of the outputs along a random direction. f = sum(out G) is off by
    its outputs' bounds, and a central difference of step h by h^2 / 6 of the third derivative: the
    difference of the differences at h and 2h, a third of which it is, bounds that."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([40, 1, 90], 4, 2, 32, torch.float32, seed=5)
    how = dict(prefix=torch.tensor([10, 0, 90]), cap=5.0, slopes=torch.tensor([0.1, 0.0, 0.3, 0.02], device="cuda"))
    grads = torch.autograd.grad(tms.packed_attention(q, k, v, offsets, **how), (q, k, v), G)
    _, off = reference(q, k, v, offsets, G, **how)
    noise = float((off[0] * G.double().abs()).sum())
    with torch.no_grad():
        for m in range(3):
            x = [q, k, v]
            way = torch.randn_like(x[m])

            def f(h):
                y = list(x)
                y[m] = x[m] + h * way
                return float((tms.packed_attention(*y, offsets, **how).double() * G).sum())

            h = 2.0 ** -7
            one, two = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
            rounding = float((grads[m].double().abs() * way.abs()).sum()) * 2.0 ** -16  # of x + h way: 2^-24 of x, over h
            got = float((grads[m].double() * way).sum())
            assert abs(got - one) <= abs(one - two) + noise / h + rounding, m


def test_long_text(cuda):
    """Many tiles of keys, rows far from the last maximum."""
    for dt in (torch.bfloat16, torch.float16):
        qkv, offsets, G = make([3001], 2, 1, 128, dt, scale=2.0)
        check(*qkv, offsets, G, f"long {dt}", prefix=0)


@pytest.mark.parametrize("D,dt", [(32, torch.bfloat16), (64, torch.bfloat16), (64, torch.float16), (96, torch.float16), (128, torch.bfloat16)],
                         ids=str)
@pytest.mark.parametrize("kind", ["plain", "prefix", "bias", "cap"])
def test_tiles_of_128(cuda, kind, D, dt):
    """Texts and heads enough for a wave to take 32 rows; a steep bias lets tokens see a part of their text only."""
    H = 24
    qkv, offsets, G = make([2901, 60, 37], H, H, D, dt, seed=9, behind=2)
    how = {}
    if kind in ("prefix", "cap"):
        how["prefix"] = torch.tensor([700, 0, 37])
    if kind == "bias":
        how["slopes"] = torch.exp2(3 - torch.arange(H, device="cuda") / 2.0)
        qkv, offsets, G = make([2901], H, H, D, dt, seed=9, behind=2)
    if kind == "cap":
        how["cap"] = 6.0
    check(*qkv, offsets, G, f"wide {kind} {D} {dt}", **how)


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("cap", [0.5, 64.0, 65.0, 300.0, 1e5, 1e12])
def test_caps(cuda, cap, dt):
    """A cap far above the scores changes nothing, one below flattens them."""
    (q, k, v), offsets, G = make([90, 33], 2, 2, 64, dt, seed=4, scale=4.0)
    out, _ = check(q, k, v, offsets, G, f"cap {cap} {dt}", cap=cap)


@pytest.mark.parametrize("slope", [0.0, -0.01, 1.0, math.inf])
def test_reach(cuda, slope):
    """A bias of any slope over a long text; norms that are not finite leave nothing out. An infinite
    slope makes a token's own distance a NaN, as 0 times infinity is."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([2100], 2, 1, 64, torch.bfloat16, seed=2, behind=3)
    slopes = torch.tensor([slope, 0.3], device="cuda")
    if math.isinf(slope):
        out = tms.packed_attention(q, k, v, offsets, slopes=slopes)
        assert bool(torch.isnan(out[:2100, 0]).all())
        return
    check(q, k, v, offsets, G, f"slope {slope}", slopes=slopes)
    want = tms.packed_attention(q, k, v, offsets, slopes=slopes)
    with torch.no_grad():
        k2 = k.clone()
        k2[2101:] = math.nan  # in rows of no text
        want, off = reference(q, k, v, offsets, G, slopes=slopes)
        close([tms.packed_attention(q, k2, v, offsets, slopes=slopes)], want, off, "NaN norms")


@pytest.mark.parametrize("H,KV", [(12, 1), (10, 2), (7, 1)])
@pytest.mark.parametrize("dt", DT, ids=str)
def test_heads_shared_by_workgroups(cuda, H, KV, dt):
    """Few tiles of keys with many heads each: their sums come in parts."""
    qkv, offsets, G = make([130, 600, 1], H, KV, 32, dt, seed=H)
    check(*qkv, offsets, G, f"parts {H} {KV} {dt}", prefix=0)
    qkv, offsets, G = make([64] * 90, H, KV, 32, dt, seed=H)
    check(*qkv, offsets, G, f"fewer parts {H} {KV} {dt}", slopes=torch.linspace(0, 1, H, device="cuda"))


@pytest.mark.parametrize("lens", ["short", "long"])
@pytest.mark.parametrize("dt", DT, ids=str)
def test_some_gradients(cuda, dt, lens):
    """Each gradient by itself, and each pair, has the bits of all three; frozen operands have none."""
    import tilemaxsim_amd as tms
    ts, offsets, G = make(LENS[lens], 6, 2, 64, dt, seed=8)
    how = dict(prefix=4, cap=20.0, slopes=torch.linspace(0, 0.5, 6, device="cuda"))
    want = torch.autograd.grad(tms.packed_attention(*ts, offsets, **how), ts, G)
    for some in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        part = [t.detach().requires_grad_(m in some) for m, t in enumerate(ts)]
        tms.packed_attention(*part, offsets, **how).backward(G)
        assert all(torch.equal(t.grad, w) if m in some else t.grad is None for m, (t, w) in enumerate(zip(part, want))), some
        got = torch.autograd.grad(tms.packed_attention(*ts, offsets, **how), [ts[m] for m in some], G)
        assert all(torch.equal(a, want[m]) for a, m in zip(got, some)), some


def test_one_tensor_three_times(cuda):
    """Queries, keys and values that are the same tensor: its gradient is the three gradients' sum."""
    import tilemaxsim_amd as tms
    (x, _, _), offsets, G = make([33, 1, 70], 4, 4, 64, torch.float32, seed=9)
    parts = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    a, b, c = torch.autograd.grad(tms.packed_attention(*parts, offsets), parts, G)
    out = tms.packed_attention(x, x, x, offsets)
    grad = torch.autograd.grad(out, x, G)[0].double()
    a, b, c = (t.double() for t in (a, b, c))
    # two sums of three addends in either order: two roundings each of at most the sum of magnitudes
    assert bool(((grad - (a + b + c)).abs() <= 4 * 2.0 ** -24 * (a.abs() + b.abs() + c.abs())).all())


def test_streams_and_graphs(cuda):
    """Another stream than the tensors' own; a captured forward and backward pass follows its inputs, replay by replay."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([50, 200, 3], 4, 2, 64, torch.bfloat16)
    offsets = offsets.cuda()
    prefix = torch.tensor([5, 0, 3], device="cuda")

    def step():
        out = tms.packed_attention(q, k, v, offsets, prefix=prefix)
        return (out, *torch.autograd.grad(out, (q, k, v), G))

    want = [x.detach().clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [x.detach().clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [x.detach() for x in step()]
    for i in range(4):
        with torch.no_grad():
            q.mul_(0.9)
            offsets[1] += 3
            prefix[1] += 40
        graph.replay()
        got = [x.clone() for x in kept]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.detach()) for a, b in zip(got, step()))
