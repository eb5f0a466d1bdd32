"""Trains a small late-interaction retriever on synthetic text, with the package's training
operators for everything that is large in such a step:

* ``maxsim_pairs``: every query of the batch against every document, both sides' gradients;
* ``linear_cross_entropy``: the masked tokens' loss over the vocabulary, whose weights are
  the token embeddings, and the one-vector loss of the pooled texts against each other;
* ``clip_grad_norm_``: the norm of all gradients, which stays on the GPU.

A document is a bag of words of one topic and some noise, its query a few other words of
the same topic: which words go together has to be learned.

    python examples/train_retriever.py --steps 200
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tilemaxsim_amd as tms  # noqa: E402

PAD, MASK, FIRST_WORD = 0, 1, 2
IGNORED = -100


class Encoder(nn.Module):
    """Token states from a token and the mean of its text; 128-wide unit token embeddings."""

    def __init__(self, vocabulary: int, width: int = 256, out: int = 128):
        super().__init__()
        self.words = nn.Embedding(vocabulary, width)
        self.mix = nn.Linear(2 * width, width)
        self.norm = nn.LayerNorm(width)
        self.out = nn.Linear(width, out, bias=False)
        nn.init.normal_(self.words.weight, std=0.02)

    def forward(self, tokens: torch.Tensor):
        """tokens (n, length) -> states (n, length, width), embeddings (n, length, 128), real (n, length)."""
        real = tokens != PAD
        x = self.words(tokens)
        mean = (x * real[..., None]).sum(1, keepdim=True) / real.sum(1).clamp(min=1)[:, None, None]
        states = self.norm(x + F.gelu(self.mix(torch.cat([x, mean.expand_as(x)], -1))))
        return states, F.normalize(self.out(states), dim=-1), real


def batch(g: torch.Generator, texts: int, words: int, topics: int = 40, query_tokens: int = 8, doc_tokens: int = 60):
    """Queries (texts, query_tokens) and documents (texts, doc_tokens), padded, on the CPU."""
    topic = torch.randperm(topics, generator=g)[:texts, None]
    half = (words - FIRST_WORD) // (2 * topics)  # of a topic's words are in its documents, half in its queries
    docs = FIRST_WORD + 2 * topic * half + torch.randint(0, half, (texts, doc_tokens), generator=g)
    noise = torch.randint(FIRST_WORD, words, docs.shape, generator=g)
    docs = torch.where(torch.rand(docs.shape, generator=g) < 0.3, noise, docs)
    queries = FIRST_WORD + (2 * topic + 1) * half + torch.randint(0, half, (texts, query_tokens), generator=g)
    docs[torch.arange(doc_tokens) >= torch.randint(doc_tokens // 3, doc_tokens + 1, (texts, 1), generator=g)] = PAD
    queries[torch.arange(query_tokens) >= torch.randint(2, query_tokens + 1, (texts, 1), generator=g)] = PAD
    hidden = (torch.rand(docs.shape, generator=g) < 0.15) & (docs != PAD)
    return queries, docs, torch.where(hidden, MASK, docs), torch.where(hidden, docs, IGNORED)


def losses(model: Encoder, queries, docs, masked, targets, dtype=torch.bfloat16):
    """The ranking, one-vector and masked-token losses, and the scores (queries, documents)."""
    _, Q, q_real = model(queries)
    _, D, d_real = model(docs)
    answer = torch.arange(len(queries), device=queries.device)
    scores = tms.maxsim_pairs(Q.to(dtype), D.to(dtype), d_real, q_real)
    rank = F.cross_entropy(scores, answer)

    def pooled(x, real):
        return F.normalize((x * real[..., None]).sum(1), dim=-1).to(dtype)

    vector = tms.linear_cross_entropy(pooled(Q, q_real), pooled(D, d_real), answer, scale=20.0)
    states, _, _ = model(masked)
    words = tms.linear_cross_entropy(states.to(dtype), model.words.weight.to(dtype), targets, ignore_index=IGNORED)
    return rank, vector, words, scores


def train(steps: int = 200, texts: int = 32, vocabulary: int = 2003, seed: int = 0, dtype=torch.bfloat16, show=print):
    """Returns the three losses and the share of queries whose document ranks first, a row a step."""
    torch.manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    model = Encoder(vocabulary).cuda()
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3, weight_decay=0.01)
    history = []
    for step in range(steps):
        queries, docs, masked, targets = (x.cuda() for x in batch(g, texts, vocabulary))
        rank, vector, words, scores = losses(model, queries, docs, masked, targets, dtype)
        optimizer.zero_grad(set_to_none=True)
        (rank + vector + words).backward()
        norm = tms.clip_grad_norm_([p.grad for p in model.parameters()], 1.0)
        optimizer.step()
        first = (scores.argmax(1) == torch.arange(texts, device="cuda")).float().mean()
        history.append(torch.stack([rank, vector, words, first, norm]).detach())
        if show and (step % 20 == 0 or step == steps - 1):
            r, v, w, f, n = history[-1].tolist()  # waits for the step
            show(f"step {step:4d}  ranking {r:.3f}  one vector {v:.3f}  masked tokens {w:.3f}  first {f:.2f}  gradient norm {n:.3f}", flush=True)
    return torch.stack(history).cpu()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--texts", type=int, default=32, help="texts a batch (at most 40)")
    args = parser.parse_args()
    train(args.steps, args.texts)
