"""What the speculative-decoding and cache-eviction operators are measured on.

A serving step that drafts a tree of tokens and keeps its cache within a budget calls, in this order,

* ``tree_attention``: the drafted nodes' queries over the cache (context rows, then the nodes' own rows, which
  a node sees when they are its ancestors or itself), dense or in pages, or over the Beacon latents;
* ``tree_accept``: the greedy target token of each node on the accepted path, and that path;
* ``tree_commit``: the accepted nodes' rows moved next to the context, every layer in one call;
* ``key_mass``: the attention weight that the accepted rows gave each key, added to its running mass;
* ``evict``: the cache cut to its budget by that mass (sinks and the recent rows always stay).

Sizes are those of this repository's own configurations: 32 / 8 heads of 128 with latent rank 320 and a
vocabulary of 128256, 40 / 8 heads of 128, 16-token pages, windows of 1024 behind 4 sinks, contexts of about
8.3k rows (and up to 131072 where the cost allows).  ``own`` selects the framework's kernels; the plain form
works in 32 bits whatever the type of the inputs.
"""
import math
import random

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # One chat sequence right after a short prompt, one token at a time: latency.
        dict(name='attention one token', op='tree_attention', batch=1, nodes=1, heads=32, kv_heads=8, dim=128,
             lo=517, hi=517, page=0, context_only=False, dtype='bf16'),
        # A small batch of ragged sequences in the serving engine's 16-token pages, 13 drafted nodes each, 40 heads.
        dict(name='attention paged drafts', op='tree_attention', batch=8, nodes=13, heads=40, kv_heads=8, dim=128,
             lo=301, hi=4099, page=16, context_only=False, dtype='bf16'),
        # Absorbed queries of 8 drafted nodes over the shared Beacon latents (one latent head, rank 320).
        dict(name='attention latents', op='tree_attention', batch=4, nodes=8, heads=32, kv_heads=1, dim=320,
             lo=7900, hi=8700, page=0, context_only=True, dtype='bf16'),
        # A full serving batch with 64-node trees behind 8k tokens of context: the heaviest call.
        dict(name='attention wide trees', op='tree_attention', batch=16, nodes=64, heads=32, kv_heads=8, dim=128,
             lo=7700, hi=8700, page=0, context_only=False, dtype='bf16'),
        # The first accepted token of one sequence, its raw window of sinks + 1024 tokens.
        dict(name='mass one token', op='key_mass', batch=1, nodes=1, heads=32, kv_heads=8, dim=128, lo=1028, hi=1028,
             page=0, context_only=False, dtype='bf16'),
        # The accepted rows of 8-node trees over the latents of a full batch.
        dict(name='mass latents', op='key_mass', batch=16, nodes=8, heads=32, kv_heads=1, dim=320, lo=7900, hi=8700,
             page=0, context_only=True, dtype='bf16'),
        # Two sequences a little over their budget of one window.
        dict(name='evict slack', op='evict', batch=2, kv_heads=8, dim=128, lo=1181, hi=1283, keep=1028, sinks=4,
             recent=128, dtype='bf16'),
        # A full batch of 32k latents cut to a quarter after a long prompt.
        dict(name='evict latents', op='evict', batch=16, kv_heads=1, dim=320, lo=32768, hi=32768, keep=8192, sinks=4,
             recent=256, dtype='bf16'),
        # A chain of 4 drafted tokens of one sequence, fp32 logits.
        dict(name='accept chain', op='tree_accept', batch=1, nodes=5, vocab=128256, depth=4, dtype='fp32'),
        # 64-node trees of a full batch, bf16 logits.
        dict(name='accept wide trees', op='tree_accept', batch=16, nodes=64, vocab=128256, depth=7, dtype='bf16'),
        # One layer of one sequence.
        dict(name='commit one layer', op='tree_commit', layers=1, batch=1, nodes=8, kv_heads=8, dim=128, lo=517,
             hi=517, depth=5, dtype='bf16'),
        # Every layer of a full batch.
        dict(name='commit all layers', op='tree_commit', layers=32, batch=16, nodes=64, kv_heads=8, dim=128, lo=60,
             hi=180, depth=7, dtype='bf16'),
    ]


def _cost(case):
    w = work(case)
    return max(w['bytes'] / 6.4e12, w['flops'] / 1.6e15, 1e-7)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {}
    for c in listed():
        limits[c['op']] = max(limits.get(c['op'], 0.0), _cost(c))
    op = rng.choice(['tree_attention', 'tree_attention', 'key_mass', 'evict', 'tree_accept', 'tree_commit'])
    while True:
        dtype = rng.choice(['bf16', 'bf16', 'fp16'])
        batch = _log(rng, 1, 16)
        if op in ('tree_attention', 'key_mass'):
            heads, kv_heads, dim, latent = rng.choice([(32, 8, 128, False), (40, 8, 128, False), (16, 4, 64, False),
                                                       (8, 8, 64, False), (12, 2, 96, False), (32, 1, 320, True),
                                                       (32, 1, 160, True)])
            hi = _log(rng, 16, 131072)
            case = dict(op=op, batch=batch, nodes=_log(rng, 1, 64), heads=heads, kv_heads=kv_heads, dim=dim,
                        lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi,
                        page=0 if latent else rng.choice([0, 0, 16, 48]), context_only=latent, dtype=dtype)
            if op == 'key_mass':
                case['nodes'] = min(case['nodes'], 16)
        elif op == 'evict':
            kv_heads, dim = rng.choice([(8, 128), (4, 64), (1, 320), (1, 160), (2, 96)])
            hi = _log(rng, 64, 131072)
            keep = max(1, int(hi * rng.uniform(0.1, 0.95)))
            sinks = min(4, keep)
            case = dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, lo=max(1, int(hi * rng.uniform(0.5, 1.0))),
                        hi=hi, keep=keep, sinks=sinks, recent=min(rng.choice([0, 32, 257]), keep - sinks), dtype=dtype)
        elif op == 'tree_accept':
            nodes = _log(rng, 1, 64)
            case = dict(op=op, batch=batch, nodes=nodes, vocab=_log(rng, 1000, 152064),
                        depth=rng.randint(1, min(nodes, 8)), dtype=rng.choice(['bf16', 'fp16', 'fp32']))
        else:
            nodes, hi = _log(rng, 1, 64), _log(rng, 16, 256)
            kv_heads, dim = rng.choice([(8, 128), (4, 64), (1, 320)])
            case = dict(op=op, layers=_log(rng, 1, 32), batch=batch, nodes=nodes, kv_heads=kv_heads, dim=dim,
                        lo=max(1, hi // 2), hi=hi, depth=rng.randint(1, min(nodes, 8)), dtype=dtype)
        if _cost(case) <= limits[op]:
            return case


# ---------------------------------------------------------------- prepare --
def _lengths(case):
    """Context lengths spread evenly over lo..hi: their sum does not depend on the seed."""
    b, lo, hi = case['batch'], case['lo'], case['hi']
    return [lo + (hi - lo) * i // max(b - 1, 1) for i in range(b)]


def _counts(case):
    """Accepted nodes of each sequence, 1..depth in turn."""
    return [1 + (i * 5 + case['depth'] - 1) % case['depth'] for i in range(case['batch'])]


def _mass_counts(case):
    return [1 + (i * 3 + case['nodes'] - 1) % case['nodes'] for i in range(case['batch'])]


def _tree(rng, nodes, depth):
    """Parents (-1: the root; a parent precedes its children) with one chain of `depth` nodes from the root, and it."""
    chain = [0] + sorted(rng.sample(range(1, nodes), depth - 1))
    parents = [-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, nodes)]
    for a, b in zip(chain, chain[1:]):
        parents[b] = a
    return parents, chain


def _ancestor_words(parents):
    """int32 words of each node's row: bit i set when the node sees node i (its ancestors and itself)."""
    words = (len(parents) + 31) // 32
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return [[(r >> 32 * w & 0xffffffff) - (r >> 32 * w & 0x80000000) * 2 for w in range(words)] for r in rows]


def _cache(case, gen, cap, dtype):
    """K and V as a user's cache holds them, and the block tables (None when dense)."""
    b, g, d = case['batch'], case['kv_heads'], case['dim']
    if case.get('page'):
        # The serving engine's raw pages [blocks, page, 2, Hkv, D]; every sequence owns its pages, in any order.
        per = -(-cap // case['page'])
        pages = torch.randn(b * per, case['page'], 2, g, d, generator=gen, device='cuda', dtype=dtype)
        order = torch.randperm(b * per, generator=gen, device='cuda')
        return pages[:, :, 0], pages[:, :, 1], order.view(b, per).to(torch.int32)
    if case.get('context_only'):
        # Latent K rows and V rows as two planes.
        lat = torch.randn(b, 2, cap, d, generator=gen, device='cuda', dtype=dtype)
        return lat[:, 0].unsqueeze(2), lat[:, 1].unsqueeze(2), None
    # Head-major planes seen as [B, rows, Hkv, D].
    kv = torch.randn(2, b, g, cap, d, generator=gen, device='cuda', dtype=dtype)
    return kv[0].transpose(1, 2), kv[1].transpose(1, 2), None


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case['dtype']]
    s = dict(op=case['op'])
    i32 = dict(dtype=torch.int32, device='cuda')
    if case['op'] in ('tree_attention', 'key_mass', 'evict', 'tree_commit'):
        lengths = _lengths(case)
        rng.shuffle(lengths)
        s['lengths'] = torch.tensor(lengths, **i32)
    if case['op'] in ('tree_attention', 'key_mass'):
        b, t, h, d = case['batch'], case['nodes'], case['heads'], case['dim']
        cap = case['hi'] + t
        s['k'], s['v'], s['tables'] = _cache(case, gen, cap, dtype)
        s['q'] = torch.randn(b, t, h, d, generator=gen, device='cuda', dtype=dtype)
        s['scale'], s['context_only'] = d ** -0.5, case['context_only']
    if case['op'] == 'tree_attention':
        trees = [_tree(rng, t, min(t, 6))[0] for _ in range(b)]
        # Without a mask the nodes are a chain: what single tokens and plain drafts use.
        s['mask'] = torch.tensor([_ancestor_words(p) for p in trees], **i32) if t > 1 and not s['context_only'] else None
    elif case['op'] == 'key_mass':
        # Accepted rows: a path of node numbers for each sequence, its count, and the rows' log-sum-exps.
        counts = _mass_counts(case)
        s['rows'] = torch.tensor([sorted(rng.sample(range(t), c)) + [-1] * (t - c) for c in counts], **i32)
        s['counts'], s['decay'] = torch.tensor(counts, **i32), 0.97
        s['lse'] = torch.full((b, t, h), -math.inf, device='cuda')
        scores, seen, at = _mass_scores(s)
        got = scores.masked_fill(~seen, -math.inf).logsumexp(-1)
        got = got.unflatten(2, (h // case['kv_heads'], t)).permute(0, 3, 1, 2).reshape(b, t, h)
        s['lse'].scatter_(1, at[:, :, None].expand(b, t, h), got)
        s['mass'] = torch.rand(b, case['kv_heads'], cap, generator=gen, device='cuda')
    elif case['op'] == 'evict':
        b, g, d, n = case['batch'], case['kv_heads'], case['dim'], case['hi']
        s['k'], s['v'], _ = _cache(dict(case, context_only=g == 1), gen, n, dtype)
        # Running masses spread over decades; a tenth of the keys was never attended to.
        mass = torch.randn(b, g, n, generator=gen, device='cuda').mul_(2).exp_()
        s['mass'] = mass * (torch.rand(b, g, n, generator=gen, device='cuda') > 0.1)
        step = torch.randint(1, 4, (b, g, n), generator=gen, device='cuda')
        s['positions'] = step.cumsum(-1).to(torch.int32)
        s['keep'], s['sinks'], s['recent'] = case['keep'], case['sinks'], case['recent']
    elif case['op'] == 'tree_accept':
        b, t, v = case['batch'], case['nodes'], case['vocab']
        logits = torch.randn(b, t, v, generator=gen, device='cuda', dtype=dtype)
        tokens = torch.randint(0, v, (b, t), generator=gen, device='cuda')
        trees = [_tree(rng, t, case['depth']) for _ in range(b)]
        # The target agrees with the drafts along the first nodes of each sequence's chain.
        hits = [(i, chain[k], chain[k + 1]) for i, ((_, chain), c) in enumerate(zip(trees, _counts(case)))
                for k in range(c - 1)]
        if hits:
            i, at, child = torch.tensor(hits, device='cuda').unbind(1)
            logits[i, at, tokens[i, child]] = 12.0
        s.update(logits=logits, tokens=tokens, parents=torch.tensor([p for p, _ in trees], **i32))
    else:
        n_layers, b, t, g, d = case['layers'], case['batch'], case['nodes'], case['kv_heads'], case['dim']
        cap = case['hi'] + t
        kv = torch.randn(2, n_layers, b, g, cap, d, generator=gen, device='cuda', dtype=dtype)
        s['k'], s['v'] = kv[0].transpose(2, 3), kv[1].transpose(2, 3)
        counts = _counts(case)
        paths = [[0] + sorted(rng.sample(range(1, t), c - 1)) + [-1] * (t - c) for c in counts]
        s['path'], s['count'] = torch.tensor(paths, **i32), torch.tensor(counts, **i32)
    return s


# -------------------------------------------------------------- plain form --
def _dense(x, tables):
    """[B, rows, Hkv, D] of a cache, gathered through its block tables when it is paged."""
    return x if tables is None else x[tables.long()].flatten(1, 2)


def _grouped(q, kv_heads):
    """[B, T, H, D] -> [B, Hkv, G * T, D], rows (head of the group, token)."""
    b, t, h, d = q.shape
    return q.view(b, t, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _plain_attention(s):
    q, k, v = s['q'].float(), _dense(s['k'], s['tables']).float(), _dense(s['v'], s['tables']).float()
    (b, t, h, _), n, g = q.shape, k.shape[1], k.shape[2]
    at = torch.arange(n, device=q.device)
    node = at - s['lengths'][:, None]                                   # [B, N]: which node's row, < 0: context
    seen = (node < 0)[:, None].expand(b, t, n)
    if not s['context_only']:
        i = torch.arange(t, device=q.device)
        if s['mask'] is None:
            bits = (i[:, None] >= i).expand(b, t, t)
        else:
            bits = (s['mask'][:, :, i // 32] >> (i % 32) & 1).bool()
        own_row = bits.gather(2, node.clamp(0, t - 1)[:, None].expand(b, t, n))
        seen = seen | (own_row & ((node >= 0) & (node < t))[:, None])
    scores = _grouped(q, g) @ k.permute(0, 2, 3, 1) * s['scale']
    scores = scores.unflatten(2, (h // g, t)).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isfinite(), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = p.flatten(2, 3) @ v.transpose(1, 2) / total.flatten(2, 3).clamp_min(1e-30)
    out = out.unflatten(2, (h // g, t)).permute(0, 3, 1, 2, 4).reshape(b, t, h, -1)
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, t, h)
    return out.to(s['q'].dtype), lse


def _mass_scores(s):
    """Scores [B, Hkv, G * A, N] of the selected rows, which keys each sees, and the rows' node numbers."""
    t = s['q'].shape[1]
    g = s['k'].shape[2]
    at = s['rows'].long().clamp_min(0)
    q = s['q'].gather(1, at[:, :, None, None].expand(*at.shape, *s['q'].shape[2:])).float()
    k = _dense(s['k'], s['tables']).float()
    scores = _grouped(q, g) @ k.permute(0, 2, 3, 1) * s['scale']
    i = torch.arange(t, device=q.device)
    end = s['lengths'][:, None] + (0 if s['context_only'] else i + 1)
    seen = (torch.arange(k.shape[1], device=q.device) < end.expand(-1, t)[:, :, None]) & (i < s['counts'][:, None])[:, :, None]
    return scores, seen.repeat(1, q.shape[2] // g, 1)[:, None], at


def _plain_mass(s):
    scores, seen, at = _mass_scores(s)
    b, t, h = s['lse'].shape
    g = s['k'].shape[2]
    n = s['mass'].shape[2]
    lse = _grouped(s['lse'].gather(1, at[:, :, None].expand(b, t, h))[..., None], g)
    added = torch.exp(scores - lse).masked_fill(~seen, 0.0).sum(2)[:, :, :n]
    key = torch.arange(n, device=added.device)
    before = key < s['lengths'][:, None, None]
    fresh = (s['lengths'] + (0 if s['context_only'] else s['counts']))[:, None, None]
    new = torch.where(before, s['decay'] * s['mass'], 0.0) + added
    s['mass'].copy_(torch.where(key < fresh, new, s['mass']))
    return s['mass']


def _plain_evict(s):
    b, g, n = s['mass'].shape
    length = s['lengths'].long()[:, None, None]
    at = torch.arange(n, device='cuda')
    stays = (at < s['sinks']) | (at >= length - s['recent'])
    rank = torch.where(stays, math.inf, s['mass']).masked_fill(at >= length, -math.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :s['keep']].sort(-1).values
    live = kept < length

    def rows(x):
        got = x.transpose(1, 2).gather(2, kept[..., None].expand(*kept.shape, x.shape[-1]))
        return torch.where(live[..., None], got, 0).transpose(1, 2)

    return (rows(s['k']), rows(s['v']), torch.where(live, s['mass'].gather(2, kept), 0.0),
            torch.where(live, s['positions'].gather(2, kept), 0), s['lengths'].clamp_max(s['keep']))


def _plain_accept(s):
    logits, tokens, parents = s['logits'].float(), s['tokens'], s['parents'].long()
    b, t, v = logits.shape
    vocab = torch.arange(v, device=logits.device)
    best = torch.where(logits == logits.amax(-1, keepdim=True), vocab, v).amin(-1)       # lowest index of the largest
    i = torch.arange(t, device=logits.device)
    child = parents[:, None] == i[:, None]                                               # [B, parent, child]
    match = child & (tokens[:, None] == best[:, :, None])
    step = (match & (match.long().cumsum(-1) == 1)).float()                              # the first matching child
    reach = torch.linalg.matrix_power(step + torch.eye(t, device=step.device), 16)       # paths of at most 16 steps
    on = reach[:, 0] > 0
    path = torch.where(on, i, t).sort(-1).values
    count = on.sum(-1)
    last = path.gather(1, count[:, None] - 1)
    return torch.where(path < t, path, -1).to(torch.int32), count.to(torch.int32), best.gather(1, last)[:, 0]


def _plain_commit(s):
    n_layers, b, n, g, d = s['k'].shape
    t = s['path'].shape[1]
    i = torch.arange(t, device='cuda')
    dst = s['lengths'].long()[:, None] + i
    src = torch.where(i < s['count'][:, None], s['lengths'].long()[:, None] + s['path'], dst)
    seq = torch.arange(b, device='cuda')[:, None]
    s['k'][:, seq, dst] = s['k'][:, seq, src]
    s['v'][:, seq, dst] = s['v'][:, seq, src]
    return s['k'], s['v'], s['lengths'] + s['count']


PLAIN = dict(tree_attention=_plain_attention, key_mass=_plain_mass, evict=_plain_evict, tree_accept=_plain_accept,
             tree_commit=_plain_commit)


# -------------------------------------------------------------------- run --
def run(state):
    s = state
    if not own:
        return PLAIN[s['op']](s)
    from slimkv_b200 import eviction, tree
    if s['op'] == 'tree_attention':
        return tree.tree_attention(s['q'], s['k'], s['v'], s['lengths'], s['scale'], mask=s['mask'],
                                   block_tables=s['tables'], context_only=s['context_only'])
    if s['op'] == 'key_mass':
        return eviction.key_mass(s['q'], s['k'], s['lse'], s['mass'], s['lengths'], s['scale'], rows=s['rows'],
                                 counts=s['counts'], decay=s['decay'], block_tables=s['tables'],
                                 context_only=s['context_only'])
    if s['op'] == 'evict':
        return eviction.evict(s['k'], s['v'], s['mass'], s['positions'], s['lengths'], s['keep'], sinks=s['sinks'],
                              recent=s['recent'])
    if s['op'] == 'tree_accept':
        return tree.tree_accept(s['logits'], s['tokens'], s['parents'])
    return s['k'], s['v'], tree.tree_commit(s['k'], s['v'], s['lengths'], s['path'], s['count'])


# ------------------------------------------------------------------- work --
def work(case):
    size = torch.empty(0, dtype=TYPES[case['dtype']]).element_size()
    op, b = case['op'], case['batch']
    if op == 'tree_accept':
        rows = sum(_counts(case))                       # only the accepted path's logits are needed
        return dict(bytes=rows * case['vocab'] * size + 12 * b * case['nodes'] + 12 * b, flops=rows * case['vocab'])
    total = sum(_lengths(case))
    if op == 'tree_commit':
        moved = (sum(_counts(case)) - b) * case['layers'] * case['kv_heads'] * case['dim'] * 2 * size
        return dict(bytes=2 * moved + 4 * b * (case['nodes'] + 3), flops=0)
    g, d = case['kv_heads'], case['dim']
    if op == 'evict':
        kept = sum(min(n, case['keep']) for n in _lengths(case)) * g
        return dict(bytes=4 * g * total + kept * (4 * d * size + 4 + 8), flops=g * total)
    t, h = case['nodes'], case['heads']
    if op == 'tree_attention':
        rows = total + (0 if case['context_only'] else b * t)
        return dict(bytes=rows * g * d * 2 * size + b * t * h * (2 * d * size + 4), flops=4 * t * h * d * total)
    picked = sum(_mass_counts(case))
    rows = total + (0 if case['context_only'] else picked)
    flops = sum(2 * c * h * d * n for c, n in zip(_mass_counts(case), _lengths(case)))
    return dict(bytes=rows * g * (d * size + 8) + picked * h * (d * size + 4), flops=flops)


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    if case['op'] == 'tree_accept':
        return None                                     # whole numbers only
    s = prepare(case, seed)
    f64 = torch.float64
    if case['op'] == 'tree_commit':
        k, v = s['k'].to(f64), s['v'].to(f64)
        for b, (n, c) in enumerate(zip(s['lengths'].tolist(), s['count'].tolist())):
            src = (n + s['path'][b, :c]).long()
            k[:, b, n:n + c] = k[:, b].index_select(1, src)
            v[:, b, n:n + c] = v[:, b].index_select(1, src)
        return k, v, None
    if case['op'] == 'evict':
        b, g, n = s['mass'].shape
        keep, d = case['keep'], case['dim']
        k, v = (torch.zeros(b, g, keep, d, dtype=f64, device='cuda') for _ in range(2))
        mass = torch.zeros(b, g, keep, dtype=f64, device='cuda')
        for i, length in enumerate(s['lengths'].tolist()):
            for j in range(g):
                m = s['mass'][i, j, :length].to(f64)
                free = torch.ones(length, dtype=torch.bool, device='cuda')
                free[:case['sinks']] = False
                free[max(0, length - case['recent']):] = False
                order = torch.where(free)[0]
                room = max(0, min(keep, length) - int((~free).sum()))
                order = order[m[order].sort(descending=True, stable=True).indices[:room]]
                idx = torch.cat([torch.where(~free)[0], order]).sort().values
                k[i, j, :len(idx)], v[i, j, :len(idx)] = s['k'][i, idx, j].to(f64), s['v'][i, idx, j].to(f64)
                mass[i, j, :len(idx)] = m[idx]
        return k.transpose(1, 2), v.transpose(1, 2), mass, None, None
    t, h, g = case['nodes'], case['heads'], case['kv_heads']
    lengths = s['lengths'].tolist()
    if case['op'] == 'tree_attention':
        out = torch.zeros(case['batch'], t, h, case['dim'], dtype=f64, device='cuda')
        lse = torch.zeros(case['batch'], t, h, dtype=f64, device='cuda')
    else:
        mass = s['mass'].to(f64)
    for b, n in enumerate(lengths):
        rows = n + (0 if case['context_only'] else t)
        if case['page']:
            flat = s['tables'][b].long()
            k, v = (x[flat].flatten(0, 1)[:rows].to(f64) for x in (s['k'], s['v']))
        else:
            k, v = s['k'][b, :rows].to(f64), s['v'][b, :rows].to(f64)
        if case['op'] == 'tree_attention':
            seen = torch.ones(t, rows, dtype=torch.bool, device='cuda')
            if not case['context_only']:
                if s['mask'] is None:
                    seen[:, n:] = torch.ones(t, t, device='cuda').tril().bool()
                else:
                    words = [[w & 0xffffffff for w in row] for row in s['mask'][b].tolist()]
                    seen[:, n:] = torch.tensor([[bool(row[i // 32] >> i % 32 & 1) for i in range(t)] for row in words],
                                               device='cuda')
            for j in range(h):
                x = (s['q'][b, :, j].to(f64) @ k[:, j * g // h].T * s['scale']).masked_fill(~seen, -math.inf)
                lse[b, :, j] = x.logsumexp(-1)
                out[b, :, j] = x.softmax(-1) @ v[:, j * g // h]
        else:
            count = int(s['counts'][b])
            end = n + (0 if case['context_only'] else count)
            mass[b, :, :n] *= s['decay']
            mass[b, :, n:end] = 0
            for i, r in enumerate(s['rows'][b, :count].tolist()):
                m = n if case['context_only'] else n + i + 1
                for j in range(h):
                    x = k[:m, j * g // h] @ s['q'][b, r, j].to(f64) * s['scale']
                    mass[b, j * g // h, :m] += torch.exp(x - s['lse'][b, r, j].to(f64))
    return (out, lse) if case['op'] == 'tree_attention' else mass
