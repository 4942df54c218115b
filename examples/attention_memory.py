"""A long conversation on a small cache: what the attention memory forgets goes to a vector
index, and comes back when a query asks for it.

Every token's key and value enter a KVCache in 8 bits; each step attends and adds up the
weight that the cached tokens receive.  When the cache is full, evict keeps the newest
tokens and the heaviest ones, and the others' keys go into one FlatIndex per head, whose
metric "cosine" is 1 - q.k: the score that attention takes softmax of.  At the end a few
queries look for old tokens: the index finds the best forgotten ones, they are appended to a
sequence of their own, and the two attentions are joined by their logarithms.

    python examples/attention_memory.py [--tokens 6000] [--budget 1024]
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import vicinity_amd as va  # noqa: E402


def tokens_of(n: int, heads: int, dim: int, seed: int):
    """Keys and values of a made-up model: tokens lie around a few dozen topics."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    topics = torch.randn((48, heads, dim), generator=g, device="cuda")
    topic = torch.randint(0, 48, (n,), generator=g, device="cuda")
    k = topics[topic] + 0.7 * torch.randn((n, heads, dim), generator=g, device="cuda")
    v = torch.randn((n, heads, dim), generator=g, device="cuda")
    return k.to(torch.bfloat16), v.to(torch.bfloat16), topics


def full_attention(q, k, v):
    """softmax(q k^T / sqrt(d)) v over all tokens, in float64: q [t, heads, d]."""
    s = torch.einsum("thd,nhd->htn", q.double(), k.double()) / math.sqrt(q.shape[2])
    return torch.einsum("htn,nhd->thd", torch.softmax(s, dim=2), v.double())


def run(tokens=6000, budget=1024, recent=256, step=64, heads=4, group=2, dim=64, recall=32,
        queries=16, seed=0):
    """Returns the mean error of the cut cache's attention and of it with what came back."""
    k, v, topics = tokens_of(tokens, heads, dim, seed)
    cache = va.KVCache(1 + queries, heads, dim, 2 * (budget // 64 + 8) + queries * (recall // 64 + 1))
    index = [va.FlatIndex(dim, "cosine") for _ in range(heads)]
    old_k, old_v = [], []
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    for at in range(0, tokens, step):
        # the conversation goes on: new tokens join and attend
        kt, vt = k[at:at + step], v[at:at + step]
        cache.append(kt, vt, seqs=[0])
        q = kt.repeat_interleave(group, dim=1) * 0.5 + 0.5 * torch.randn(
            (kt.shape[0], heads * group, dim), generator=g, device="cuda").to(kt.dtype)
        cache.attend(q, seqs=[0], decay=1.0)
        if cache.lengths[0] >= budget + 4 * step:
            gone = cache.evict(budget, recent, seqs=[0], dropped=True)
            old_k.append(gone["k"][0])
            old_v.append(gone["v"][0])
            for h in range(heads):
                index[h].add(gone["k"][0, :, h].cpu().numpy())
    old_k, old_v = torch.cat(old_k), torch.cat(old_v)

    # queries about topics of long ago, one per query token and head
    about = torch.randint(0, topics.shape[0], (queries,), generator=g, device="cuda")
    q = (2.0 * topics[about]).to(torch.bfloat16)  # [queries, heads, dim]
    want = full_attention(q, k, v)

    # the cache alone; queries do not follow the tokens, so all of them see it all
    out, lse = cache.attend(q, seqs=[0], causal=False, return_lse=True)

    # each head's best forgotten tokens, to a sequence for each query
    ids = torch.stack([index[h].search_device(q[:, h].float().contiguous(), recall)[0]
                       for h in range(heads)], dim=2)  # [queries, recall, heads]
    head = torch.arange(heads, device="cuda")
    seqs = list(range(1, 1 + queries))
    cache.append(old_k[ids, head].reshape(-1, heads, dim), old_v[ids, head].reshape(-1, heads, dim),
                 seqs=seqs, positions=ids.reshape(-1, heads).to(torch.int32).contiguous())
    more, more_lse = cache.attend(q, seqs=seqs, return_lse=True)

    # softmax over both parts: weights by the parts' denominators
    both = torch.logaddexp(lse, more_lse)
    joined = out * torch.exp(lse - both)[..., None] + more * torch.exp(more_lse - both)[..., None]
    err = [(x.double() - want).norm() / want.norm() for x in (out, joined)]
    return float(err[0]), float(err[1]), len(old_k)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--tokens", type=int, default=6000)
    p.add_argument("--budget", type=int, default=1024)
    a = p.parse_args()
    cut, joined, gone = run(tokens=a.tokens, budget=a.budget)
    print(f"{a.tokens} tokens, {a.budget} slots kept, {gone} in the index of each head")
    print(f"error against attention over all tokens: cut cache {cut:.3f}, "
          f"with 32 recalled tokens {joined:.3f}")


if __name__ == "__main__":
    main()
