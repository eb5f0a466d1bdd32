"""GPU tests of ``examples/train_retriever.py``: one step's losses and gradients against the
same model in float64 with elementary operations on the CPU, and a short training run."""
import importlib.util
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


def plain(model, queries, docs, masked, targets):
    """The example's losses with nothing of the package's."""
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
    """fp32 against float64. Tolerance: some twenty roundings of 2^-24 in a row, of sums of up
    to 2,000 terms whose errors add up like their square root, logits up to 20 in the exponent:
    20 * 45 * 20 * 2^-24 = 1.1e-3 of a gradient's largest element, far below what a wrong
    weight, mask or factor makes. (amax shares a gradient among equal maxima; they are equal
    here where a word repeats in a document, whose states and parameters are the same.)"""
    import tilemaxsim_amd as tms
    g = torch.Generator().manual_seed(3)
    data = example.batch(g, 24, 1501)
    torch.manual_seed(4)
    model = example.Encoder(1501)
    exact = example.Encoder(1501).double()
    exact.load_state_dict(model.state_dict())
    model = model.cuda()
    *got, _ = example.losses(model, *(x.cuda() for x in data), dtype=torch.float32)
    want = plain(exact, *data)
    for a, b in zip(got, want):
        assert abs(float(a) - float(b)) <= 1.1e-3 * abs(float(b))
    sum(got).backward()
    sum(want).backward()
    for (name, p), q in zip(model.named_parameters(), exact.parameters()):
        top = float(q.grad.abs().max())
        assert float((p.grad.double().cpu() - q.grad).abs().max()) <= 1.1e-3 * top, name
    norm = torch.sqrt(sum(q.grad.square().sum() for q in exact.parameters()))
    before = [p.grad.clone() for p in model.parameters()]
    assert abs(float(tms.clip_grad_norm_([p.grad for p in model.parameters()], 0.1)) - float(norm)) <= 1.1e-3 * float(norm)
    c = min(1.0, 0.1 / (float(norm) + 1e-6))
    for p, b in zip(model.parameters(), before):
        assert float((p.grad - c * b).abs().max()) <= 1.2e-3 * c * float(b.abs().max())


def test_training_learns(cuda, example):
    """All three losses of the last ten steps are below those of the first ten, and most
    queries find their document, which one in 32 does by chance."""
    h = example.train(steps=80, show=None)
    assert bool(torch.isfinite(h).all())
    for column in range(3):
        assert float(h[-10:, column].mean()) < float(h[:10, column].mean())
    assert float(h[-10:, 3].mean()) > 0.5
