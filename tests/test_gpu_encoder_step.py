"""The training step of ``examples/train_retriever.py`` with attention layers: packed attention, gated
blocks, MaxSim, cross entropy, the norm and AdamW together, against the same model in float64 with
elementary operations on the CPU; and the step captured into a graph."""
import importlib.util
import math
import os

import pytest
import torch
from torch.nn import functional as F

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_retriever", os.path.join(REPO, "examples", "train_retriever.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_layer(example):
    class Plain(example.Layer):
        def attention(self, q, k, v, offsets):
            outs = []
            for a, b in zip(offsets[:-1].tolist(), offsets[1:].tolist()):
                i = torch.arange(b - a)
                x = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) / math.sqrt(q.shape[2])
                x = x - self.slopes[:, None, None] * (i[:, None] - i).abs()
                outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(x, -1), v[a:b]))
            return torch.cat(outs)

        def gated(self, x):
            return F.silu(x @ self.gate.weight.T) * (x @ self.up.weight.T)

    return Plain


def plain_losses(model, queries, docs, masked, targets):
    _, Q, q_real = model(queries)
    _, D, d_real = model(docs)
    sim = torch.einsum("qid,bjd->qbij", Q, D).masked_fill(~d_real[None, :, None], -torch.inf)
    scores = (sim.amax(-1) * q_real[:, None]).sum(-1)
    answer = torch.arange(len(queries))

    def pooled(x, real):
        return F.normalize((x * real[..., None]).sum(1), dim=-1)

    vector = F.cross_entropy(20.0 * pooled(Q, q_real) @ pooled(D, d_real).T, answer)
    states, _, _ = model(masked)
    words = F.cross_entropy((states @ model.words.weight.T).flatten(0, 1), targets.flatten(), ignore_index=-100)
    return F.cross_entropy(scores, answer), vector, words


def test_a_step_is_the_plain_models(cuda, example):
    """fp32 against float64. Tolerance: two layers are some eighty roundings of 2^-24 in a row, of sums of up to
    2,000 terms whose errors add up like their square root, logits up to 20 in the exponent: 80 * 45 * 20 * 2^-24 =
    4.3e-3 of a gradient's largest element, far below what a wrong mask, head or factor makes. A parameter moves by
    lr in its first step whatever its gradient's size, so the step is compared where the gradient is above the
    tolerance: there its sign is known, and with eps = 0 the update is lr sign(g) + lr decay p to 2e-6 of lr."""
    import tilemaxsim_amd as tms
    data = example.batch(torch.Generator().manual_seed(3), 24, 1501)
    torch.manual_seed(4)
    model = example.PackedEncoder(1501, 2)
    with torch.no_grad():
        model.words.weight.mul_(20)  # differing tokens, as training makes them
    exact = example.PackedEncoder(1501, 2, layer=plain_layer(example))
    exact.load_state_dict(model.state_dict())
    exact, model = exact.double(), model.cuda()
    *got, _ = example.losses(model, *(x.cuda() for x in data), dtype=torch.float32)
    want = plain_losses(exact, *data)
    for a, b in zip(got, want):
        assert abs(float(a) - float(b)) <= 4.3e-3 * abs(float(b))
    sum(got).backward()
    sum(want).backward()
    params, grads = list(model.parameters()), [p.grad for p in model.parameters()]
    for (name, p), q in zip(model.named_parameters(), exact.parameters()):
        top = float(q.grad.abs().max())
        assert float((p.grad.cpu().double() - q.grad).abs().max()) <= 4.3e-3 * top, name
    norm = tms.grad_norm(grads)
    total = math.sqrt(sum(float(q.grad.square().sum()) for q in exact.parameters()))
    assert abs(float(norm) - total) <= 4.3e-3 * total
    state = tms.AdamWState(params)
    before = [p.detach().cpu().double() for p in params]
    tms.adamw_(params, grads, state, lr=1e-3, eps=0.0, weight_decay=0.01, norm=norm, max_norm=total / 3)
    for p, b, q in zip(params, before, exact.parameters()):
        sure = q.grad.abs() > 4.3e-3 * float(q.grad.abs().max())
        want = b * (1 - 1e-5) - 1e-3 * torch.sign(q.grad)
        off = (p.detach().cpu().double() - want).abs()
        assert float((off - 2.0 ** -23 * b.abs() - 2e-9)[sure].max()) <= 0


def test_training_runs(cuda, example):
    """bf16 weights with 8-bit states: finite losses, moving weights that are the parameters' roundings."""
    history = example.train(steps=3, texts=8, vocabulary=503, show=None, layers=2)
    assert history.shape == (3, 5) and bool(torch.isfinite(history).all())


def test_weights_are_the_parameters_roundings(cuda, example, monkeypatch):
    """Every step of the example moves its fp32 parameters, and leaves in each 16-bit weight what its parameter rounds to."""
    import tilemaxsim_amd as tms
    step, seen = tms.adamw_, []

    def watched(params, grads, state, copies=None, **how):
        weights = list(copies)
        before = [p.clone() for p in params]
        step(params, grads, state, copies=weights, **how)
        assert all(torch.equal(w.detach(), p.to(w.dtype)) for p, w in zip(params, weights))
        seen.append((sum(int((p != b).sum()) for p, b in zip(params, before)), sum(p.numel() for p in params)))

    monkeypatch.setattr(example.tms, "adamw_", watched)
    example.train(steps=3, texts=8, vocabulary=503, show=None, layers=2)
    assert len(seen) == 3 and all(moved > n // 2 for moved, n in seen)


def test_a_captured_step(cuda, example):
    """Forward, backward and the optimizer's step in one graph, replayed with new batches, against eager steps."""
    import tilemaxsim_amd as tms
    torch.manual_seed(1)
    T, width, heads = 150, 128, 2
    layer = example.Layer(width, heads).cuda().bfloat16()
    weights = list(layer.parameters())

    def make():
        return [p.detach().float() for p in weights]

    start = [p.detach().clone() for p in weights]
    masters, x = make(), torch.randn(T, width, device="cuda").bfloat16()
    offsets, G = torch.tensor([0, 60, 60, 140], device="cuda"), torch.randn(T, width, device="cuda").bfloat16()
    state = tms.AdamWState(masters, bits=8)

    def step(masters, state):
        grads = torch.autograd.grad(layer(x, offsets), weights, G)
        norm = tms.grad_norm(grads)
        tms.adamw_(masters, grads, state, lr=1e-2, norm=norm, max_norm=1.0, copies=weights)
        return norm

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(masters, state)  # warm
    torch.cuda.current_stream().wait_stream(side)

    def reset():
        with torch.no_grad():
            for p, s in zip(weights, start):
                p.copy_(s)
        return make()

    def rounds(run, state):
        g, norms = torch.Generator(device="cuda").manual_seed(5), []
        for i in range(4):
            with torch.no_grad():
                x.copy_(torch.randn(T, width, generator=g, device="cuda"))
                offsets[1] = 60 - 10 * i
            norms.append(run().clone())
        torch.cuda.synchronize()
        return norms, [p.detach().clone() for p in weights], [t.clone() for t in state.state_dict().values()]

    masters = reset()
    state = tms.AdamWState(masters, bits=8)
    eager = rounds(lambda: step(masters, state), state)

    fresh = reset()
    kept = tms.AdamWState(fresh, bits=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(fresh, kept)

    def replay():
        graph.replay()
        return norm

    replayed = rounds(replay, kept)
    for a, b in zip(eager, replayed):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
