"""The speculative decoding example: its tokens against a plain 64-bit forward
of the same weights, and its cache under a budget."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))

import speculative_decode as example  # noqa: E402
from slimkv_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu


def plain_logits(model, tokens):
    """Logits ``[n, vocab]`` of one sequence in 64 bits."""
    n, heads, kv_heads, dim = len(tokens), model.heads, model.kv_heads, model.head_dim
    cos, sin = model.cos[:n, None].double(), model.sin[:n, None].double()

    def norm(x):
        return x * (x.pow(2).mean(-1, keepdim=True) + model.eps).rsqrt() * model.norm.double()

    def rope(x):
        return x * cos + torch.cat([-x[..., dim // 2:], x[..., :dim // 2]], -1) * sin

    x = model.embedding[torch.tensor(tokens, device='cuda')].double()
    for l in range(model.layers):
        qkv = (norm(x) @ model.qkv[l].double().T).view(n, heads + 2 * kv_heads, dim)
        q, k, v = rope(qkv[:, :heads]), rope(qkv[:, heads:heads + kv_heads]), qkv[:, heads + kv_heads:]
        k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        s = torch.einsum('qhd,khd->hqk', q, k) * dim ** -0.5
        s = s.masked_fill(torch.ones(n, n, device='cuda', dtype=torch.bool).triu(1), float('-inf')).softmax(-1)
        x = x + torch.einsum('hqk,khd->qhd', s, v).reshape(n, -1) @ model.o[l].double().T
        gate, up = (norm(x) @ model.gate_up[l].double().T).chunk(2, -1)
        x = x + torch.nn.functional.silu(gate) * up @ model.down[l].double().T
    return norm(x) @ model.head.double().T


def prompts(model, batch, n):
    gen = torch.Generator(device='cuda').manual_seed(5)
    return torch.randint(0, model.vocab, (batch, n), generator=gen, device='cuda')


@pytest.mark.parametrize('branches,depth', [(3, 4), (1, 6), (0, 0)])
def test_tokens_are_the_greedy_ones(branches, depth):
    model = example.Model()
    prompt = prompts(model, 3, 70)
    tokens, cache = example.generate(model, prompt, 24, branches=branches, depth=depth)
    assert _lib.device_status(clear=True) == 0
    for p, new, length in zip(prompt.tolist(), tokens, cache.lengths.tolist()):
        assert length == 70 + len(new) - 1 and len(new) >= 25
        # The first 64-bit logit of the new tokens against the largest: some 30 roundings of up to 2^-8 of a unit-size
        # value with random signs are off by 0.02; three times that for each of the two logits.
        logits = plain_logits(model, p + new)[69:-1]
        gap = logits.amax(1) - logits.gather(1, torch.tensor(new, device='cuda')[:, None])[:, 0]
        assert gap.max() < 0.125


def test_a_budget_holds_and_changes_nothing_before_the_first_eviction():
    model = example.Model()
    prompt = prompts(model, 3, 70)
    free, _ = example.generate(model, prompt, 30)
    tokens, cache = example.generate(model, prompt, 30, budget=90, slack=20, sinks=4, recent=40)
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


def test_masses_sum_to_the_rows_attention():
    """Without decay or eviction each accepted row has given every head's weight once."""
    model = example.Model()
    prompt = prompts(model, 2, 50)
    tokens, cache = example.generate(model, prompt, 10)
    for b, length in enumerate(cache.lengths.tolist()):
        total = cache.mass[:, b, :, :length].double().sum(-1)
        group = model.heads // model.kv_heads
        # A row's weights are e^(s - lse) of the same 16-bit products: fp32 exponents, sums of at most a few hundred terms.
        assert (total - length * group).abs().max() < 1e-4 * length * group
