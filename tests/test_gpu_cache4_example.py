"""The speculative decoding example over 4-bit caches: it runs, its masses add
up, and a budget keeps the rows that it says."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))

import speculative_decode as example  # noqa: E402
from slimkv_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu


def prompts(model, batch, n):
    gen = torch.Generator(device='cuda').manual_seed(5)
    return torch.randint(0, model.vocab, (batch, n), generator=gen, device='cuda')


def test_it_runs_and_the_masses_are_the_rows_attention():
    model = example.Model()
    prompt = prompts(model, 2, 70)
    tokens, cache = example.generate(model, prompt, 10, four_bit=True)
    again, _ = example.generate(model, prompt, 10, four_bit=True)
    assert _lib.device_status(clear=True) == 0 and tokens == again and cache.k.dtype == torch.uint8
    group = model.heads // model.kv_heads
    for b, length in enumerate(cache.lengths.tolist()):
        assert length == 70 + len(tokens[b]) - 1
        # A row's weights are e^(s - lse) of the same 16-bit products: fp32 exponents, sums of at most a few hundred terms.
        total = cache.mass[:, b, :, :length].double().sum(-1)
        assert (total - length * group).abs().max() < 1e-4 * length * group


def test_a_budget_holds():
    model = example.Model()
    prompt = prompts(model, 3, 70)
    free, _ = example.generate(model, prompt, 30, four_bit=True)
    tokens, cache = example.generate(model, prompt, 30, budget=90, slack=20, sinks=4, recent=40, four_bit=True)
    assert _lib.device_status(clear=True) == 0
    for b, (f, t) in enumerate(zip(free, tokens)):
        # 70 rows and at most 5 a step: nothing leaves in the first 8 steps, which make 8 tokens at least.
        assert t[:9] == f[:9]
        length = int(cache.lengths[b])
        assert 90 <= length <= 115
        for rows in cache.positions[:, b, :, :length].flatten(0, 1).tolist():
            assert rows == sorted(set(rows)) and rows[:4] == [0, 1, 2, 3]
            assert rows[-40:] == list(range(70 + len(t) - 1 - 40, 70 + len(t) - 1))
    assert torch.isfinite(cache.mass).all()
