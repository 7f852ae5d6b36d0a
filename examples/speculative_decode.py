"""Greedy decoding with drafted token trees over a cache kept within a budget.

A small decoder with random weights, batched.  Each step:

1. drafts a tree behind the last token from the sequence's own history (the
   continuations of the places where its last token stood before),
2. runs the model once over the tree's nodes: their K/V rows go behind the
   context, ``tree.tree_attention`` attends over context and ancestors,
3. accepts the path that the model would have taken (``tree.tree_accept``) and
   moves its rows next to the context in every layer (``tree.tree_commit``),
4. adds the attention that the accepted rows gave each key to its mass
   (``eviction.key_mass``), and
5. once a cache has outgrown its budget by the slack, keeps the sinks, the
   recent rows and the heaviest others (``eviction.evict``).

While nothing has been evicted the tokens are those of one-token-at-a-time
greedy decoding.  Keys are cached rotated, so the rows that stay need no
change.

    python examples/speculative_decode.py [--steps 64] [--budget 192]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from slimkv_b200 import eviction, kernels, tree  # noqa: E402
from slimkv_b200.rope import rope_tables  # noqa: E402


class Model:
    """Weights of a decoder with grouped K/V heads, RMS norms and gated MLPs (bf16, random)."""

    def __init__(self, vocab=251, hidden=512, layers=3, heads=8, kv_heads=2, head_dim=64, positions=4096, seed=0):
        self.vocab, self.hidden, self.layers = vocab, hidden, layers
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, 1e-5
        gen = torch.Generator(device='cuda').manual_seed(seed)

        def rand(*shape, scale=1.0):
            return (torch.randn(shape, generator=gen, device='cuda') * scale * shape[-1] ** -0.5).to(torch.bfloat16)

        inner = 2 * hidden
        branch = 0.5 * (2 * layers) ** -0.5     # what a layer adds: mild, so that histories repeat and drafts hit
        self.embedding = rand(vocab, hidden) * hidden ** 0.5
        self.qkv = [rand((heads + 2 * kv_heads) * head_dim, hidden) for _ in range(layers)]
        self.o = [rand(hidden, heads * head_dim, scale=branch) for _ in range(layers)]
        self.gate_up = [rand(2 * inner, hidden) for _ in range(layers)]
        self.down = [rand(hidden, inner, scale=branch) for _ in range(layers)]
        self.norm = torch.ones(hidden, dtype=torch.bfloat16, device='cuda')
        self.head = rand(vocab, hidden)
        self.cos, self.sin = rope_tables(head_dim, 10000.0, positions, device='cuda')


class Cache:
    """K, V and masses of all layers; a second set of buffers takes what an eviction keeps."""

    def __init__(self, model, batch, capacity):
        shape = (model.layers, batch, capacity, model.kv_heads, model.head_dim)
        self.k, self.v, self.k2, self.v2 = (torch.zeros(shape, dtype=torch.bfloat16, device='cuda') for _ in range(4))
        self.mass, self.mass2 = (torch.zeros((model.layers, batch, model.kv_heads, capacity), device='cuda')
                                 for _ in range(2))
        # Where each kept row stood in the sequence.
        self.positions = torch.arange(capacity, dtype=torch.int32, device='cuda').expand(self.mass.shape).contiguous()
        self.positions2 = torch.zeros_like(self.positions)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device='cuda')

    def evict(self, keep, sinks, recent):
        for l in range(self.k.shape[0]):
            lengths = eviction.evict(self.k[l], self.v[l], self.mass[l], self.positions[l], self.lengths, keep, sinks,
                                     recent, out=(self.k2[l], self.v2[l], self.mass2[l], self.positions2[l]))[4]
        self.k, self.k2, self.v, self.v2 = self.k2, self.k, self.v2, self.v
        self.mass, self.mass2, self.positions, self.positions2 = self.mass2, self.mass, self.positions2, self.positions
        self.lengths = lengths


def forward(model, cache, tokens, positions, mask=None):
    """Logits ``[B, T, vocab]`` of the nodes, and each layer's ``(q, lse)`` for the masses."""
    batch, t = tokens.shape
    heads, kv_heads, dim = model.heads, model.kv_heads, model.head_dim
    sequences = torch.arange(batch, device='cuda')[:, None]
    rows = cache.lengths[:, None].long() + torch.arange(t, device='cuda')
    x = model.embedding[tokens]
    seen = []
    for l in range(model.layers):
        qkv = (kernels.rms_norm(x, model.norm, model.eps) @ model.qkv[l].T).view(batch, t, heads + 2 * kv_heads, dim)
        q = kernels.rope_rows(qkv[:, :, :heads], positions, model.cos, model.sin)
        cache.k[l, sequences, rows] = kernels.rope_rows(qkv[:, :, heads:heads + kv_heads], positions, model.cos, model.sin)
        cache.v[l, sequences, rows] = qkv[:, :, heads + kv_heads:]
        out, lse = tree.tree_attention(q, cache.k[l], cache.v[l], cache.lengths, dim ** -0.5, mask=mask)
        seen.append((q, lse))
        x = x + out.view(batch, t, heads * dim) @ model.o[l].T
        gate_up = kernels.rms_norm(x, model.norm, model.eps).view(batch * t, -1) @ model.gate_up[l].T
        x = x + (kernels.silu_mul(gate_up) @ model.down[l].T).view_as(x)
    return kernels.rms_norm(x, model.norm, model.eps) @ model.head.T, seen


def add_masses(model, cache, seen, lengths, rows=None, counts=None, decay=1.0):
    for l, (q, lse) in enumerate(seen):
        eviction.key_mass(q, cache.k[l], lse, cache.mass[l], lengths, model.head_dim ** -0.5, rows=rows, counts=counts,
                          decay=decay)


def prefill(model, cache, prompt, chunk=64):
    """The prompt in chains of ``chunk`` nodes (no mask); returns the first token after it."""
    for begin in range(0, prompt.shape[1], chunk):
        tokens = prompt[:, begin:begin + chunk]
        positions = torch.arange(begin, begin + tokens.shape[1], dtype=torch.int32, device='cuda')
        logits, seen = forward(model, cache, tokens, positions.expand(tokens.shape[0], -1).contiguous())
        add_masses(model, cache, seen, cache.lengths)
        cache.lengths = cache.lengths + tokens.shape[1]
    return logits[:, -1].argmax(-1)


def draft(history, branches, depth):
    """Nodes' tokens and parents: node 0 is the last token, behind it the latest
    distinct continuations of its earlier occurrences."""
    tokens, parents, drafted = [history[-1]], [-1], set()
    for at in range(len(history) - 2, -1, -1):
        if len(drafted) == branches:
            break
        if history[at] == history[-1] and history[at + 1] not in drafted:
            drafted.add(history[at + 1])
            for i, token in enumerate(history[at + 1:at + 1 + depth]):
                parents.append(len(tokens) - 1 if i else 0)
                tokens.append(token)
    # Trees of a batch have one size: what is left over hangs at the root.
    while len(tokens) < 1 + branches * depth:
        parents.append(0)
        tokens.append(history[-1])
    return tokens, parents


def generate(model, prompt, steps, budget=None, slack=32, sinks=4, recent=64, branches=3, depth=4, decay=1.0):
    """``steps`` speculative steps behind ``prompt [B, n]``; returns each
    sequence's new tokens, and the cache."""
    batch, n = prompt.shape
    nodes = 1 + branches * depth
    # A step adds up to depth + 1 rows and needs room for the nodes' rows behind the context.
    most = n + steps * (depth + 1) if budget is None else max(n, budget + slack) + depth + 1
    cache = Cache(model, batch, most + nodes)
    first = prefill(model, cache, prompt)
    history = [p + [t] for p, t in zip(prompt.tolist(), first.tolist())]
    length = n
    for _ in range(steps):
        drafts = [draft(h, branches, depth) for h in history]
        tokens = torch.tensor([d[0] for d in drafts], device='cuda')
        parents = torch.tensor([d[1] for d in drafts], dtype=torch.int32, device='cuda')
        deep = [[0] * nodes for _ in drafts]
        for b, (_, ps) in enumerate(drafts):
            for t in range(1, nodes):
                deep[b][t] = deep[b][ps[t]] + 1
        positions = torch.tensor([[len(h) - 1 + d for d in ds] for h, ds in zip(history, deep)], dtype=torch.int32,
                                 device='cuda')
        old = cache.lengths
        logits, seen = forward(model, cache, tokens, positions, tree.tree_masks(parents))
        # The i-th node of any path stands i behind the root.
        behind = torch.arange(nodes, dtype=torch.int32, device='cuda')
        cache.positions[:, torch.arange(batch, device='cuda')[:, None], :, old[:, None].long() + behind] = \
            (positions[:, :1] + behind)[:, :, None, None]
        path, count, following = tree.tree_accept(logits, tokens, parents)
        cache.lengths = tree.tree_commit(cache.k, cache.v, old, path, count)
        add_masses(model, cache, seen, old, rows=path, counts=count, decay=decay)
        for h, nodes_taken, c, token, ts in zip(history, path.tolist(), count.tolist(), following.tolist(), drafts):
            h.extend(ts[0][node] for node in nodes_taken[1:c])
            h.append(token)
        length = length + depth + 1
        if budget is not None and length > budget + slack:      # at most: the lengths stay on the device
            cache.evict(budget, sinks, recent)
            length = budget
    return [h[n:] for h in history], cache


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument('--batch', type=int, default=4)
    parser.add_argument('--prompt', type=int, default=160)
    parser.add_argument('--steps', type=int, default=64)
    parser.add_argument('--budget', type=int, default=192)
    args = parser.parse_args()
    model = Model()
    gen = torch.Generator(device='cuda').manual_seed(1)
    prompt = torch.randint(0, model.vocab, (args.batch, args.prompt), generator=gen, device='cuda')
    tokens, cache = generate(model, prompt, args.steps, budget=args.budget)
    made = sum(map(len, tokens))
    print(f'{made} tokens in {args.steps} steps of {args.batch} sequences '
          f'({made / args.steps / args.batch:.2f} per sequence and step); cache rows {cache.lengths.tolist()}')


if __name__ == '__main__':
    main()
