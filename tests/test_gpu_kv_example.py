"""examples/attention_memory.py: append, attention, eviction and the flat index together."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "attention_memory.py")


def test_recalled_tokens_bring_attention_back():
    print("[case] example: 3000 tokens, 512 slots", flush=True)
    spec = importlib.util.spec_from_file_location("attention_memory", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    cut, joined, gone = example.run(tokens=3000, budget=512, recent=128)
    # 3000 tokens less the 512 kept at the last cut and what came after it
    assert 3000 - 512 - 256 <= gone <= 3000 - 512
    # what is missing after the cut is mostly found again
    assert joined < 0.5 * cut
