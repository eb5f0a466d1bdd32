"""Trains a small late-interaction retriever on synthetic text, with the package's training
operators for everything that is large in such a step:

* ``maxsim_pairs``: every query of the batch against every document, both sides' gradients;
* ``linear_cross_entropy``: the masked tokens' loss over the vocabulary, whose weights are
  the token embeddings, and the one-vector loss of the pooled texts against each other;
* ``clip_grad_norm_``: the norm of all gradients, which stays on the GPU;
* ``adamw_``: the optimizer's step, over all parameters at once.

With ``--layers`` the encoder is a stack of attention layers over the texts without their padding
(``packed_attention``, ``gated_linear``) in bf16, its fp32 parameters have 8-bit optimizer states, and
the step clips and writes the bf16 weights itself.

A document is a bag of words of one topic and some noise, its query a few other words of
the same topic: which words go together has to be learned.

    python examples/train_retriever.py --steps 200
    python examples/train_retriever.py --steps 200 --layers 2
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


class Layer(nn.Module):
    """Attention within each text, nearer tokens first, and a gated feed-forward block."""

    def __init__(self, width: int, heads: int):
        super().__init__()
        inner = (8 * width // 3 + 63) // 64 * 64
        self.heads = heads
        self.before_attention, self.before_block = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv, self.mix = nn.Linear(width, 3 * width, bias=False), nn.Linear(width, width, bias=False)
        self.gate, self.up = (nn.Linear(width, inner, bias=False) for _ in range(2))
        self.down = nn.Linear(inner, width, bias=False)
        self.register_buffer("slopes", 2.0 ** (-8 * torch.arange(1, heads + 1) / heads), persistent=False)

    def attention(self, q, k, v, offsets):
        return tms.packed_attention(q, k, v, offsets, slopes=self.slopes.float())

    def gated(self, x):
        return tms.gated_linear(x, self.gate.weight, self.up.weight)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor):
        qkv = self.qkv(self.before_attention(x)).view(len(x), 3 * self.heads, -1)
        x = x + self.mix(self.attention(*qkv.split(self.heads, 1), offsets).flatten(1))
        return x + self.down(self.gated(self.before_block(x)))


class PackedEncoder(nn.Module):
    """Token states from layers over the texts one behind another; 128-wide unit token embeddings."""

    def __init__(self, vocabulary: int, layers: int, width: int = 256, out: int = 128, layer=Layer):
        super().__init__()
        self.words = nn.Embedding(vocabulary, width)
        self.layers = nn.ModuleList(layer(width, width // 64) for _ in range(layers))
        self.norm = nn.LayerNorm(width)
        self.out = nn.Linear(width, out, bias=False)
        nn.init.normal_(self.words.weight, std=0.02)

    def forward(self, tokens: torch.Tensor):
        """tokens (n, length) -> states (n, length, width), embeddings (n, length, 128), real (n, length)."""
        real = tokens != PAD
        offsets = F.pad(real.sum(1).cumsum(0), (1, 0))
        x = self.words(tokens[real])
        for layer in self.layers:
            x = layer(x, offsets)
        packed = self.norm(x)
        states = packed.new_zeros(*tokens.shape, packed.shape[1]).masked_scatter(real[..., None], packed)
        embeddings = packed.new_zeros(*tokens.shape, self.out.out_features)
        return states, embeddings.masked_scatter(real[..., None], F.normalize(self.out(packed), dim=-1)), real


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


def losses(model: nn.Module, queries, docs, masked, targets, dtype=torch.bfloat16):
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


def train(steps: int = 200, texts: int = 32, vocabulary: int = 2003, seed: int = 0, dtype=torch.bfloat16, show=print, layers: int = 0):
    """Returns the three losses and the share of queries whose document ranks first, a row a step."""
    torch.manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    if layers:  # 16-bit weights, which the step below writes from fp32 parameters
        model = PackedEncoder(vocabulary, layers).cuda().to(dtype)
        parameters = [p.detach().float() for p in model.parameters()]
    else:
        model = Encoder(vocabulary).cuda()
        parameters = list(model.parameters())
    state = tms.AdamWState(parameters, bits=8 if layers else 32)
    history = []
    for step in range(steps):
        queries, docs, masked, targets = (x.cuda() for x in batch(g, texts, vocabulary))
        rank, vector, words, scores = losses(model, queries, docs, masked, targets, dtype)
        model.zero_grad(set_to_none=True)
        (rank + vector + words).backward()
        grads = [p.grad for p in model.parameters()]
        if layers:
            norm = tms.grad_norm(grads)
            tms.adamw_(parameters, grads, state, lr=1e-3, weight_decay=0.01, norm=norm, max_norm=1.0, copies=model.parameters())
        else:
            norm = tms.clip_grad_norm_(grads, 1.0)
            tms.adamw_(parameters, grads, state, lr=2e-3, weight_decay=0.01)
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
    parser.add_argument("--layers", type=int, default=0, help="attention layers of the encoder (0: a mean of the text's words)")
    args = parser.parse_args()
    train(args.steps, args.texts, layers=args.layers)
