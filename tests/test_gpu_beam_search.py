"""Beam search with all of it: prompts in a KVCache, beams forked from them, attention over the
shared prefix, select_beams, and forks of the chosen ones, step after step against references
that hold each beam alone."""

import copy
import os
import runpy

import numpy as np
import pytest

import kv_reference as ref
from test_gpu_beams import ERR, reference
from test_gpu_kv import Pair, _check_attend, _np, _rand
from test_gpu_kv_shared import share

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _torch():
    import torch

    return torch


@pytest.mark.parametrize("code,dtype", [("int8", "bfloat16"), ("fp8", "float32")])
def test_steps_of_a_search(code, dtype):
    """Every step's attention, choice and cached values, each beam by itself."""
    torch = _torch()
    import vicinity_amd as va

    groups, beams, heads, group, dim, vocab = 2, 5, 2, 2, 64, 501
    rows = groups * beams
    print(f"[case] beam search {code} {dtype}", flush=True)
    pair = Pair(rows, heads, dim, 32, code, blocks=200)
    share(pair.cache)
    g = torch.Generator().manual_seed(3)
    table = torch.randn((vocab, 2, heads, dim), generator=g).to(getattr(torch, dtype)).to("cuda:0")
    head = torch.randn((heads * group * dim, vocab), generator=g).to("cuda:0") * 0.2
    first, lengths = [0, beams], [300, 411]
    k, v = _rand((sum(lengths), heads, dim), dtype, 1), _rand((sum(lengths), heads, dim), dtype, 2)
    pair.append(k, v, first, lengths)
    pair.cache.fork([i // beams * beams for i in range(rows)], range(rows))
    for i in range(rows):
        pair.k[i], pair.v[i] = copy.deepcopy(pair.k[i // beams * beams]), copy.deepcopy(pair.v[i // beams * beams])
    # the first step goes on from one beam of each prompt
    scores = torch.full((rows,), -torch.inf, device="cuda:0")
    scores[first] = 0.0
    for step in range(6):
        q = _rand((rows, heads * group, dim), dtype, 10 + step)
        _check_attend(pair, q, list(range(rows)), [1] * rows)
        out = pair.cache.attend(q)
        logits = (out.float().flatten(1) @ head).to(getattr(torch, dtype))
        best, parents, tokens = va.select_beams(logits, scores, beams)
        want, wparents, wtokens, _ = reference(logits, scores, beams, beams)
        assert np.abs(_np(best) - want).max() <= ERR + 2.0 ** -24 * np.abs(want).max()
        same = (parents.cpu().numpy() == wparents) & (tokens.cpu().numpy() == wtokens)
        gaps = np.abs(np.diff(want, axis=1)).min()
        assert same.all() or gaps <= 2 * ERR
        order = parents.view(-1).tolist()
        pair.cache.fork(order, range(rows))
        was = [(copy.deepcopy(pair.k[i]), copy.deepcopy(pair.v[i])) for i in order]
        for i in range(rows):
            pair.k[i], pair.v[i] = was[i]
        kv = table[tokens.view(-1)]
        pair.append(kv[:, 0], kv[:, 1], list(range(rows)), [1] * rows)
        pair.check_values()
        scores = best.view(-1)
        if step == 3:
            pair.cache.compact(120)
            pair.check_values()
    pair.cache.truncate([0] * rows)
    assert pair.cache.info()["free_blocks"] == 120


def test_the_example_finds_the_same_with_shared_and_copied_blocks():
    torch = _torch()
    mod = runpy.run_path(os.path.join(ROOT, "examples", "beam_search.py"))
    (texts, scores, shared), (texts2, scores2, copied) = mod["run"](prompts=3, beams=4, steps=12, length=500)
    assert texts.shape == (3, 4, 12) and scores.shape == (3, 4)
    assert (scores[:, 1:] <= scores[:, :-1]).all() and torch.isfinite(scores).all()
    for p in range(3):  # a prompt's beams are different texts
        assert len({tuple(t) for t in texts[p].tolist()}) == 4
    # 12 beams of 8 blocks each, or the prompts' 24 and what the beams wrote
    assert copied >= 12 * 8 - 12 and shared <= 24 + 12 * 2
    assert scores2.shape == scores.shape and texts2.shape == texts.shape
