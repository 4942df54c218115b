"""Beam search over a KVCache: beams that continue one prompt hold its blocks together, attend
reads them once for all beams, select_beams chooses the best continuations of every prompt, and
fork makes the chosen beams the next step's sequences.

The model is made up: one attention layer with random projections over a small vocabulary.

    python examples/beam_search.py [--prompts 4] [--beams 6] [--steps 24]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import vicinity_amd as va  # noqa: E402


class Model:
    """Token embeddings, their keys, values and queries, and logits of what attention returns."""

    def __init__(self, vocab=1000, heads=4, group=2, dim=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.group, self.dim = heads, group, dim
        width = heads * group * dim

        def matrix(*shape):
            return torch.randn(shape, generator=g, device="cuda") / shape[0] ** 0.5

        self.embed = torch.randn((vocab, width), generator=g, device="cuda")
        self.wk, self.wv = matrix(width, heads * dim), matrix(width, heads * dim)
        self.wq, self.out = matrix(width, width), matrix(width, vocab) * 3.0

    def kv(self, tokens):
        x = self.embed[tokens]
        return [(x @ w).view(-1, self.heads, self.dim).to(torch.bfloat16) for w in (self.wk, self.wv)]

    def queries(self, tokens):
        q = self.embed[tokens] @ self.wq
        return q.view(-1, self.heads * self.group, self.dim).to(torch.bfloat16)

    def logits(self, tokens, attended):
        return (self.embed[tokens] + attended.float().flatten(1)) @ self.out


def search(model, prompts, beams, steps, copy=False):
    """The best `beams` continuations of each prompt by `steps` tokens: tokens [prompts, beams,
    steps] and their log-probabilities.  copy: every beam has blocks of its own."""
    n, rows = len(prompts), len(prompts) * beams
    longest = max(len(p) for p in prompts)
    each = (longest + steps) // 64 + 2
    cache = va.KVCache(rows, model.heads, model.dim, 2 * rows * each)
    # the prompts, in the first beam of each
    first = [i * beams for i in range(n)]
    k, v = model.kv(torch.cat(prompts))
    cache.append(k, v, seqs=first, counts=[len(p) for p in prompts])
    last = torch.stack([p[-1] for p in prompts])
    out = cache.attend(model.queries(last), seqs=first)
    scores, _, tokens = va.select_beams(model.logits(last, out), None, 1, beams)
    cache.fork([i for i in first for _ in range(beams)], range(rows), copy=copy)
    texts = tokens.view(rows, 1)
    for _ in range(steps - 1):
        last = texts[:, -1]
        k, v = model.kv(last)
        cache.append(k, v)
        out = cache.attend(model.queries(last))
        scores, parents, tokens = va.select_beams(model.logits(last, out), scores.view(-1), beams)
        texts = torch.cat([texts[parents.view(-1)], tokens.view(rows, 1)], dim=1)
        cache.fork(parents.view(-1).tolist(), range(rows), copy=copy)
    return texts.view(n, beams, steps), scores, cache


def run(prompts=4, beams=6, steps=24, length=700, seed=0):
    """Texts and scores with shared blocks and with copied ones, and the blocks that each holds."""
    model = Model(seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    texts = [torch.randint(0, 1000, (length - 37 * i,), generator=g, device="cuda") for i in range(prompts)]
    results = []
    for copy in (False, True):
        found, scores, cache = search(model, texts, beams, steps, copy)
        results.append((found, scores, cache.num_blocks - cache.info()["free_blocks"]))
    return results


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--prompts", type=int, default=4)
    p.add_argument("--beams", type=int, default=6)
    p.add_argument("--steps", type=int, default=24)
    a = p.parse_args()
    (texts, scores, shared), (_, _, copied) = run(a.prompts, a.beams, a.steps)
    for i in range(a.prompts):
        print(f"prompt {i}: log-probability {float(scores[i, 0]):.2f}, tokens {texts[i, 0, :8].tolist()} ..")
    print(f"{shared} blocks hold all beams, {copied} when each has its own")


if __name__ == "__main__":
    main()
