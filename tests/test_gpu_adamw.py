"""AdamW steps against float64, and 8-bit states against a restatement of their rounding.

Tolerances, with e = 2^-24 (half a step of fp32). The clip factor: 6 e of itself (the norm's, the constant's,
the sum's and the quotient's roundings). m: each product's rounding and that of its factor, the sum's: 6 e of
the summands' magnitudes, and 6 e more of the gradient's under a clip. v: the same with the gradient's part twice: 10 e, 22 e.
p: its decay and the subtraction: 4 e |p|; the step: m's error and 16 e of m (root, quotient, both
factors, v's error halved), over the denominator. Then half a step of the tensor's own type.
8-bit states are equal to the restatement's, bit for bit: m and v are formed from single roundings.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16, torch.float16]
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}
e = 2.0 ** -24
BLOCK = 128

SIZES = {
    "one": [(1,)],
    "vector ends": [(7,), (8,), (9,), (2047,), (2049,), (3, 5)],
    "block ends": [(127,), (128,), (129,), (255,), (257,), (0,), (4, 0, 3), (1,)],
    "chunk ends": [(8192,), (8191,), (8193,), (24577,), (8192 - 120,), (8192 + 130,)],
    "many": [(1 + (i * 37) % 300,) for i in range(1000)],  # several launches, and counters over one list
    "large": [(1000, 1001), (1 << 20,)],
}


def tensors(sizes, seed, dts, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * (size * (0.1 + i % 5))).to(dts[i % len(dts)]) for i, s in enumerate(sizes)]


def clip_of(gs, norm, most):
    return 1.0 if norm is None else min(1.0, most / (float(norm) + 1e-6))


def expect(p, g, m, v, t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, c=1.0, clipped=False):
    """The new p, m and v in 64 bits, and how far each may be off."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    b1, b2 = betas
    x = c * g
    parts = (b1 * m).abs() + ((1 - b1) * x).abs()
    em = 6 * e * parts + (6 * e * ((1 - b1) * x).abs() if clipped else 0)
    m, v = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    ev = (22 if clipped else 10) * e * v
    step, under = lr / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt() + eps
    move = step * m / under
    new = p * (1 - lr * weight_decay) - move
    ep = 4 * e * (p.abs() + new.abs()) + step * em / under + 32 * e * move.abs()
    return (new, ep), (m, em), (v, ev)


def near(got, want, off, what):
    dt = got.dtype
    off = off + ROUND[dt] * want.abs() + TINY[dt]
    over = float(((got.double() - want).abs() / off).max()) if got.numel() else 0.0
    assert not torch.isnan(got).any() and over <= 1.0, f"{what}: {over:.3g} times its bound off"


# ---------------------------------------------------------------- 8 bits, restated

def numbers(codes, exps, octaves, magnitude):
    k = codes.long() & magnitude
    e_ = exps.long().repeat_interleave(BLOCK) - octaves
    bits = ((k + 8 * e_).clamp(min=0) << 20).to(torch.int32)
    x = bits.view(torch.float32)
    x = torch.where(k == 0, torch.zeros_like(x), x)
    x = torch.where(k == magnitude, torch.full_like(x, math.nan), x)
    return torch.where(codes.long() > magnitude, -x, x)


def mixed(x):
    for s, f in ((16, 0x7feb352d), (15, 0x846ca68b)):
        x = ((x ^ (x >> s)) * f) & 0xffffffff
    return x ^ (x >> 16)


def codes(x, at, t, octaves, magnitude):
    """x's codes and exponents, its first element at place `at`, in the tensor's step t."""
    n = x.numel()
    a = x.abs().view(torch.int32).long()
    exps = torch.where(a < 0x7f800000, a, 0).view(-1, BLOCK).amax(1) >> 23
    base = 8 * (exps.repeat_interleave(BLOCK) - octaves)
    place = torch.arange(at, at + n, device=x.device)
    h = mixed((place & 0xffffffff) ^ mixed((t + (place >> 32) * 0x9e3779b1) & 0xffffffff))
    u = h & 0xffff if magnitude == 127 else h >> 16
    c = ((a + 16 * u) >> 20) - base
    least = ((base + 1).clamp(min=0) << 20).to(torch.int32).view(torch.float32).double()
    under = (x.abs().double() >= u.double() / 65536 * least).long() if magnitude == 127 else torch.ones_like(c)
    c = torch.where(c < 1, under, c)
    c = torch.where(a == 0, 0, c)
    c = torch.where(a >= 0x7f800000, magnitude, c)
    if magnitude == 127:
        c = c + 128 * (x.view(torch.int32) < 0)
    return c.to(torch.uint8), exps.to(torch.uint8)


def moved(g, m, v, c=None):
    """m and v in fp32, operation by operation."""
    g = g.float() if c is None else g.float() * c
    return 0.9 * m + (1 - 0.9) * g, 0.999 * v + (1 - 0.999) * g * g


def padded(state, ts):
    flat = torch.zeros(state.size, device="cuda")
    for view, t in zip(state.views(flat), ts):
        view.copy_(t)
    return flat


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", list(SIZES))
def test_steps(cuda, kind, bits):
    import tilemaxsim_amd as tms
    print(f"adamw {kind} {bits}", flush=True)
    ps = tensors(SIZES[kind], 1, DT, 0.1)
    state = tms.AdamWState(ps, bits=bits)
    copies = [torch.full(p.shape, 7.0, device="cuda", dtype=DT[(i + 2) % 3]) if i % 4 else None for i, p in enumerate(ps)]
    for t in range(1, 4):
        gs = tensors(SIZES[kind], 10 + t, DT[1:] + DT[:1], 1e-2)
        norm = tms.grad_norm(gs) if t > 1 else None
        most = None if norm is None else float(norm) * (0.3 if t == 2 else 2.0)
        c = clip_of(gs, norm, most)
        before = [p.clone() for p in ps]
        m0, v0 = (x.clone() for x in state.moments())
        keep = [g.clone() for g in gs]
        tms.adamw_(ps, gs, state, norm=norm, max_norm=most, copies=copies)
        assert all(torch.equal(a, b) for a, b in zip(gs, keep)), "gradients changed"
        assert state.steps.tolist() == [t] * len(ps)
        m1, v1 = state.moments()
        for i, (p, q, g, m, v, m_, v_) in enumerate(zip(before, ps, gs, *(state.views(x) for x in (m0, v0, m1, v1)))):
            (want, ep), (wm, em), (wv, ev) = expect(p, g, m, v, t, c=c, clipped=norm is not None)
            near(q, want, ep, f"p[{i}]")
            if copies[i] is not None:
                near(copies[i], want, ep, f"copy[{i}]")
            if bits == 32:
                near(m_, wm, em, f"m[{i}]")
                near(v_, wv, ev, f"v[{i}]")
        if bits == 8:
            factor = None if norm is None else torch.clamp(torch.full_like(norm, most) / (norm + 1e-6), max=1.0)
            m, v = moved(padded(state, gs), m0, v0, factor)
            for x, name, octaves, mag in ((m, "m", 14, 127), (v, "v", 30, 255)):
                cs, exps = codes(x, 0, t, octaves, mag)
                assert torch.equal(getattr(state, name), cs) and torch.equal(getattr(state, name + "_exp"), exps), name
                assert torch.equal(numbers(cs, exps, octaves, mag), m1 if name == "m" else v1)
        else:
            assert all(torch.equal(a, b) for a, b in zip(state.moments(), moved(padded(state, gs), m0, v0,
                       None if norm is None else torch.clamp(torch.full_like(norm, most) / (norm + 1e-6), max=1.0))))


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_and_range(cuda, bits):
    """Gradients of zero, of sizes whose squares leave fp32's range, and blocks of one large element."""
    import tilemaxsim_amd as tms
    for size in (0.0, 1e-25, 1e-18, 1e15):
        p, g = torch.full((300,), 0.5, device="cuda"), torch.full((300,), size, device="cuda")
        state = tms.AdamWState(p, bits=bits)
        tms.adamw_(p, g, state, weight_decay=0.0)
        m, _ = state.moments()
        x = float(torch.tensor(size))
        square = float((torch.tensor(0.001) * x) * x)  # as fp32 holds it
        assert bool((m[:300] >= 0).all()) and bool(torch.isfinite(p).all())
        update = 1e-3 * x / (math.sqrt(square / 1e-3) + 1e-8)
        assert bool(((0.5 - p).double() - update).abs().max() <= 2e-3 * abs(update) + 1e-7), size
    p, g = torch.zeros(128, device="cuda"), torch.full((128,), 1e-3, device="cuda")
    g[5] = 1e9
    state = tms.AdamWState(p, bits=bits)
    for _ in range(3):
        tms.adamw_(p, g, state, weight_decay=0.0)
    assert bool(torch.isfinite(p).all()) and float(p.abs().max()) < 4e-3  # no step above lr: v below its range is rounded up


def test_codes_are_right_in_the_mean(cuda):
    """States without new gradients shrink as b^t does. A code's rounding has a standard deviation of at most half a
    step, an eighth of the value: over t steps less than sqrt(t) / 16 of the value, and the mean of n elements sqrt(n) less;
    six of those."""
    import tilemaxsim_amd as tms
    n, steps = 1 << 18, 200
    p, g = torch.zeros(n, device="cuda"), (1 + torch.rand(n, device="cuda"))
    state = tms.AdamWState(p, bits=8)
    tms.adamw_(p, g, state)
    m0, v0 = (x.double().mean() for x in state.moments())
    zero = torch.zeros_like(g)
    for t in range(1, steps + 1):
        tms.adamw_(p, zero, state)
        if t in (10, steps):
            m, v = (x.double().mean() for x in state.moments())
            within = 6 * math.sqrt(t) / 16 / math.sqrt(n)
            if t == 10:
                assert abs(float(m / m0) / 0.9 ** t - 1) <= within
            assert abs(float(v / v0) / 0.999 ** t - 1) <= within


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_gradients(cuda, bits):
    """None: nothing of the parameter changes, and its count stays behind."""
    import tilemaxsim_amd as tms
    ps = tensors([(200,), (300,), (50, 3)], 1, [torch.float32])
    state = tms.AdamWState(ps, bits=bits)
    gs = tensors([(200,), (300,), (50, 3)], 2, [torch.float32])
    tms.adamw_(ps, gs, state)
    before = [p.clone() for p in ps], [x.clone() for x in state.moments()]
    tms.adamw_(ps, [gs[0], None, gs[2]], state)
    assert state.steps.tolist() == [2, 1, 2]
    assert torch.equal(ps[1], before[0][1]) and not torch.equal(ps[0], before[0][0]) and not torch.equal(ps[2], before[0][2])
    for now, was in zip(state.moments(), before[1]):
        assert torch.equal(state.views(now)[1], state.views(was)[1]) and not torch.equal(state.views(now)[2], state.views(was)[2])
    m0, v0 = state.moments()
    m0, v0, p0 = state.views(m0)[1].clone(), state.views(v0)[1].clone(), ps[1].clone()
    tms.adamw_(ps, [None, gs[1], None], state)
    (want, ep), *_ = expect(p0, gs[1], m0, v0, 2)
    near(ps[1], want, ep, "the second step")
    tms.adamw_(ps, [None] * 3, state)
    assert state.steps.tolist() == [2, 2, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_in_the_step(cuda, bits):
    """The same as clip_grad_norm_ first, to the bits of fp32 gradients."""
    import tilemaxsim_amd as tms
    sizes = [(300, 7), (1000,)]
    a, b = tensors(sizes, 1, [torch.float32]), tensors(sizes, 1, [torch.float32])
    one, two = tms.AdamWState(a, bits=bits), tms.AdamWState(b, bits=bits)
    for t in range(3):
        gs = tensors(sizes, 5 + t, [torch.float32])
        tms.adamw_(a, gs, one, norm=tms.grad_norm(gs), max_norm=1.0)
        tms.clip_grad_norm_(gs, 1.0)
        tms.adamw_(b, gs, two)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(x, y) for x, y in zip(one.state_dict().values(), two.state_dict().values()))


def test_layouts(cuda):
    """Views of one buffer at every alignment, with what is beside them left as it is; strided tensors."""
    import tilemaxsim_amd as tms
    for dt in DT:
        flat, gflat, cflat = (torch.randn(9000, device="cuda").to(k) for k in (dt, dt, torch.bfloat16))
        keep, ckeep = flat.clone(), cflat.clone()
        cuts = [(1, 8), (10, 523), (524, 525), (530, 2700), (2703, 8999)]
        ps, gs, cs = ([x[a:b] for a, b in cuts] for x in (flat, gflat, cflat))
        state = tms.AdamWState(ps)
        tms.adamw_(ps, gs, state, copies=cs)
        beside = torch.ones(9000, dtype=torch.bool, device="cuda")
        for a, b in cuts:
            (want, ep), *_ = expect(keep[a:b], gflat[a:b], torch.zeros(b - a, device="cuda"), torch.zeros(b - a, device="cuda"), 1)
            near(flat[a:b], want, ep, "view")
            beside[a:b] = False
        assert torch.equal(flat[beside], keep[beside]) and torch.equal(cflat[beside], ckeep[beside])
    wide = torch.randn(30, 80, device="cuda")
    rest = wide[:, 1::2].clone()
    p, c, g = wide[:, ::2], torch.empty(40, 30, device="cuda").t(), torch.randn(40, 30, device="cuda").t()
    p0 = p.clone()
    state = tms.AdamWState([p])
    tms.adamw_([p], [g], state, copies=[c])
    (want, ep), (wm, em), _ = expect(p0, g, torch.zeros_like(p0), torch.zeros_like(p0), 1)
    near(p, want, ep, "strided")
    assert torch.equal(c, p) and torch.equal(wide[:, 1::2], rest)
    near(state.views(state.m)[0], wm, em, "strided m")


def test_one_element_in_two_places(cuda):
    """Parameters and copies that are expanded, or given twice, are refused, and nothing has changed."""
    import tilemaxsim_amd as tms
    p, q = torch.ones(1, 5, device="cuda"), torch.ones(4, 5, device="cuda")
    for params, copies in (([p.expand(4, 5)], None), ([q], [p.expand(4, 5)]), ([p.expand(4, 5)], [q]), ([q], [q])):
        state = tms.AdamWState(params)
        with pytest.raises(ValueError, match="overlap"):
            tms.adamw_(params, [torch.ones(4, 5, device="cuda")], state, copies=copies)
        assert not state.steps.any() and not state.m.any() and bool((p == 1).all()) and bool((q == 1).all())
    q = torch.ones(4, 5, device="cuda").t()  # rows and columns in the other order are no overlap
    state = tms.AdamWState([q])
    tms.adamw_([q], [p.expand(4, 5).t()], state)
    assert int(state.steps) == 1 and bool((q < 1).all())


def test_views_of_one_buffer(cuda):
    """Strided parameters and copies side by side are stepped as each by itself; where they overlap they are refused, and
    nothing has changed."""
    import tilemaxsim_amd as tms
    g = torch.Generator(device="cuda").manual_seed(7)
    w, grad, c = (torch.randn(30, 80, generator=g, device="cuda") for _ in range(3))
    keep, ckeep = w.clone(), c.clone()
    for params, grads, copies in (([w[:, :50], w[:, 40:]], [grad[:, :50], grad[:, 40:]], None), ([w.t()[:, :3], w[2]], [grad.t()[:, :3], grad[2]], None),
                                  ([w[:, :40]], [grad[:, :40]], [w[:, 39:79]]), ([w[:, :40]], [w[:, 30:70]], None), ([w[5:7].view(160)], [w.view(-1)[300:620:2]], None)):
        state = tms.AdamWState(params)
        with pytest.raises(ValueError, match="overlap"):
            tms.adamw_(params, grads, state, copies=copies)
        assert not state.steps.any() and not state.m.any() and torch.equal(w, keep)
    ps, gs, cs = [w[:, :40], w[:, 40:60:2], w[:, 41:60:2]], [grad[:, :40], grad[:, 40:60:2], grad[:, 41:60:2]], [c[:, 40:], c[:, :10], c[:, 10:20]]
    alone = [p.clone() for p in ps]
    for p, x in zip(alone, gs):
        tms.adamw_(p, x.contiguous(), tms.AdamWState(p))
    tms.adamw_(ps, gs, tms.AdamWState(ps), copies=cs)
    assert all(torch.equal(p, a) and torch.equal(x, a) for p, x, a in zip(ps, cs, alone))
    assert torch.equal(w[:, 60:], keep[:, 60:]) and torch.equal(c[:, 20:40], ckeep[:, 20:40])


def test_some_copies(cuda):
    """Copies of some parameters, of several types, and parameters of inference mode: each as by itself, versions counted."""
    import tilemaxsim_amd as tms
    g = torch.Generator(device="cuda").manual_seed(3)
    ps, gs = ([torch.randn(n, generator=g, device="cuda") for n in (5, 300, 77, 1)] for _ in range(2))
    with torch.inference_mode():
        ps[3] = ps[3].clone()
    alone = [p.clone() for p in ps]
    for p, x in zip(alone, gs):
        tms.adamw_(p, x, tms.AdamWState(p))
    copies = [None, torch.empty(300, device="cuda", dtype=torch.float16), torch.empty(77, device="cuda", dtype=torch.bfloat16), None]
    before = [t._version for t in (*ps[:3], *copies[1:3])]
    tms.adamw_(ps, gs, tms.AdamWState(ps), copies=copies)
    assert all(torch.equal(a, b) for a, b in zip(ps, alone)) and all(torch.equal(c, p.to(c.dtype)) for c, p in zip(copies[1:3], ps[1:3]))
    assert all(t._version > v for t, v in zip((*ps[:3], *copies[1:3]), before))


def test_nonfinite(cuda):
    """A NaN or infinite gradient goes into its own element alone, in 8 bits too; a NaN norm into all."""
    import tilemaxsim_amd as tms
    for bits in (32, 8):
        for bad in (math.nan, math.inf, -math.inf):
            p, q = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
            g = torch.randn(300, device="cuda")
            h = g.clone()
            h[130] = bad
            one, two = tms.AdamWState(p, bits=bits), tms.AdamWState(q, bits=bits)
            for _ in range(2):
                tms.adamw_(p, g, one)
                tms.adamw_(q, h, two)
            here = torch.arange(300, device="cuda") == 130
            assert torch.equal(p[~here], q[~here]) and not bool(torch.isfinite(q[here]).any())
            for a, b in zip(one.moments(), two.moments()):
                a, b = a[:300], b[:300]
                if bits == 32:
                    assert torch.equal(a[~here], b[~here])
                else:  # where the element was its block's largest, the others' range begins lower
                    near_ = (a - b).abs() <= 2 * b.abs() / 8 + a.abs().max() * 2.0 ** -13
                    assert bool(near_[~here].all()) and bool(torch.isnan(b[here]).all())
        p, g = torch.ones(5, device="cuda"), torch.ones(5, device="cuda")
        tms.adamw_(p, g, tms.AdamWState(p, bits=bits), norm=torch.tensor(math.nan, device="cuda"), max_norm=1.0)
        assert bool(torch.isnan(p).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_kept_and_loaded(cuda, bits, tmp_path):
    """A saved state goes on to the same bits; a model's parameters change their version."""
    import tilemaxsim_amd as tms
    ps = [torch.nn.Parameter(t) for t in tensors([(70, 3), (200,)], 1, [torch.float32])]
    gs = tensors([(70, 3), (200,)], 2, [torch.bfloat16])
    state = tms.AdamWState(ps, bits=bits)
    version = ps[0]._version
    tms.adamw_(ps, gs, state)
    assert ps[0]._version > version
    torch.save({k: v for k, v in state.state_dict().items()}, tmp_path / "state.pt")
    qs = [p.detach().clone() for p in ps]
    other = tms.AdamWState(qs, bits=bits)
    other.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    tms.adamw_(ps, gs, state)
    tms.adamw_(qs, gs, other)
    assert all(torch.equal(a, b) for a, b in zip(ps, qs))
    assert all(torch.equal(a, b) for a, b in zip(state.state_dict().values(), other.state_dict().values()))


@pytest.mark.parametrize("bits", [32, 8])
def test_streams_and_graphs(cuda, bits):
    """A captured step counts on, and follows its gradients, norm and lr from replay to replay."""
    import tilemaxsim_amd as tms
    sizes = [(1000,), (33, 77), (20_000,)]
    a, b = tensors(sizes, 1, [torch.float32]), tensors(sizes, 1, [torch.float32])
    gs = tensors(sizes, 2, [torch.bfloat16])
    one, two = tms.AdamWState(a, bits=bits), tms.AdamWState(b, bits=bits)
    lr = torch.tensor(1e-3, device="cuda")

    def step(ps, state):
        tms.adamw_(ps, gs, state, lr=lr, norm=tms.grad_norm(gs), max_norm=5.0)

    step(a, one)
    step(b, two)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, one)
    side = torch.cuda.Stream()
    for i in range(4):
        for g in gs:
            g.mul_(1.5)
        lr.mul_(0.7)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(b, two)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert one.steps.tolist() == [i + 2] * 3
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(x, y) for x, y in zip(one.state_dict().values(), two.state_dict().values()))
