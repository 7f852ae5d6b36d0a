"""What the operators of the 4-bit cache are measured on.

A serving loop that holds its keys and values in 4 bits calls

* ``cache4.write``: new rows quantised into the cache, dense or in pages, at each sequence's own place, and
  ``cache4.read``: rows of the cache as 16-bit rows;
* ``cache4.attention``: the attention of one token or of a drafted tree over that cache;
* ``cache4.key_mass``: the attention weight that accepted rows gave each of its keys.

A row of D dims (a multiple of 32) is D / 2 bytes of codes, then (scale, minimum) of each group of 32 dims in the
rows' 16-bit type, filled up to a multiple of 16 bytes.  Byte 4w + 2h + i holds the codes of the dims 8w + 4i + h
(low half) and 8w + 4i + 2 + h (high half); a code c stands for ``c * scale + minimum``, rounded to the rows' type.
The minimum is the group's smallest value, the scale (largest - smallest) / 15 in the rows' type, a code the nearest
whole number (ties: the even one) to (value - minimum) / scale; a scale below 2^-126 is 0, and so are its codes.

Sizes are those of this repository's own configurations: 32 / 8 heads of 128 with latent ranks 320 and 160, 40 / 8
heads of 128, 16-token pages, windows of 1024 behind 4 sinks, contexts of about 8.3k rows and up to 131072.  ``own``
selects the framework's kernels; the plain form works in 32 bits (codes at a border in 64) whatever the inputs' type.
"""
import math
import random

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
GROUP = 32


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # One chat sequence right after a short prompt, one token at a time: latency.
        dict(name='attention one token', op='attention', batch=1, nodes=1, heads=32, kv_heads=8, dim=128, lo=517,
             hi=517, page=0, context_only=False, dtype='bf16'),
        # A small batch of ragged sequences in 16-token pages, 5 drafted nodes each, 40 heads.
        dict(name='attention paged drafts', op='attention', batch=8, nodes=5, heads=40, kv_heads=8, dim=128, lo=301,
             hi=4099, page=16, context_only=False, dtype='bf16'),
        # A full serving batch behind 8k tokens of context, one token each: what a decode step does most.
        dict(name='attention full batch', op='attention', batch=16, nodes=1, heads=32, kv_heads=8, dim=128, lo=7700,
             hi=8700, page=0, context_only=False, dtype='bf16'),
        # One long document in pages, fp16: the split over a long axis.
        dict(name='attention long context', op='attention', batch=1, nodes=1, heads=32, kv_heads=8, dim=128, lo=131072,
             hi=131072, page=16, context_only=False, dtype='fp16'),
        # Absorbed queries over the shared Beacon latents (one latent head, rank 320) of a full batch.
        dict(name='attention latents', op='attention', batch=16, nodes=1, heads=32, kv_heads=1, dim=320, lo=7900,
             hi=8700, page=0, context_only=True, dtype='bf16'),
        # The new token of every sequence of a full batch.
        dict(name='write one token', op='write', batch=16, kv_heads=8, dim=128, lo=1, hi=1, behind=8300, page=0,
             dtype='bf16'),
        # Prompt chunks of four sequences into pages, the last ones not full.
        dict(name='write prompt chunk', op='write', batch=4, kv_heads=8, dim=128, lo=4097, hi=5120, behind=1028,
             page=16, dtype='bf16'),
        # A window's Beacon latents of a full batch, fp16.
        dict(name='write latents', op='write', batch=16, kv_heads=1, dim=320, lo=128, hi=257, behind=4096, page=0,
             dtype='fp16'),
        # The open window of one sequence, to rebuild its dense rows.
        dict(name='read open window', op='read', batch=1, kv_heads=8, dim=128, lo=1028, hi=1028, page=0, dtype='bf16'),
        # Latent histories of a full batch out of 48-row pages, before a prompt chunk attends over them.
        dict(name='read latent histories', op='read', batch=16, kv_heads=1, dim=320, lo=7168, hi=8300, page=48,
             dtype='bf16'),
        # The first accepted token of one sequence, its raw window of sinks + 1024 tokens.
        dict(name='mass one token', op='mass', batch=1, nodes=1, heads=32, kv_heads=8, dim=128, lo=1028, hi=1028,
             page=0, context_only=False, dtype='bf16'),
        # The accepted rows of 5-node drafts of a full batch.
        dict(name='mass full batch', op='mass', batch=16, nodes=5, heads=32, kv_heads=8, dim=128, lo=7700, hi=8700,
             page=0, context_only=False, dtype='bf16'),
    ]


def _cost(case):
    w = work(case)
    return max(w['bytes'] / 6.4e12, w['flops'] / 3e14, 1e-7)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {}
    for c in listed():
        limits[c['op']] = max(limits.get(c['op'], 0.0), _cost(c))
    op = rng.choice(['attention', 'attention', 'attention', 'write', 'read', 'mass'])
    while True:
        dtype = rng.choice(['bf16', 'bf16', 'fp16'])
        batch = _log(rng, 1, 16)
        if op in ('attention', 'mass'):
            heads, kv_heads, dim, latent = rng.choice([(32, 8, 128, False), (40, 8, 128, False), (16, 4, 64, False),
                                                       (8, 8, 64, False), (12, 2, 96, False), (32, 1, 320, True),
                                                       (32, 1, 160, True)])
            hi = _log(rng, 16, 131072)
            case = dict(op=op, batch=batch, nodes=_log(rng, 1, 16), heads=heads, kv_heads=kv_heads, dim=dim,
                        lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, page=rng.choice([0, 0, 16, 48]),
                        context_only=latent, dtype=dtype)
        else:
            kv_heads, dim = rng.choice([(8, 128), (8, 128), (4, 64), (2, 96), (1, 320), (1, 160)])
            hi = _log(rng, 1, 131072)
            case = dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, lo=max(1, int(hi * rng.uniform(0.3, 1.0))),
                        hi=hi, page=rng.choice([0, 0, 16, 48]), dtype=dtype)
            if op == 'write':
                case['behind'] = _log(rng, 1, 8300)
        if _cost(case) <= limits[op]:
            return case


# ---------------------------------------------------------------- prepare --
def _row_bytes(dim):
    return -(-(dim // 2 + dim // 8) // 16) * 16


def _lengths(case):
    """Lengths spread evenly over lo..hi: their sum does not depend on the seed."""
    b, lo, hi = case['batch'], case['lo'], case['hi']
    return [lo + (hi - lo) * i // max(b - 1, 1) for i in range(b)]


def _mass_counts(case):
    return [1 + (i * 3 + case['nodes'] - 1) % case['nodes'] for i in range(case['batch'])]


def _ancestor_words(rng, nodes):
    """A drafted tree's int32 mask words: bit i of node t set when t sees i (its ancestors and itself)."""
    rows = []
    for t in range(nodes):
        rows.append((rows[rng.randrange(max(0, t - 4), t)] if t else 0) | 1 << t)
    return [[r - (r >> 31 << 32)] for r in rows]


def _rows(gen, shape, dtype):
    """Keys and values as a model's projections give them: noise around each channel's mean, a few channels large."""
    g, d = shape[-2:]
    mean = torch.randn(g, d, generator=gen, device='cuda')
    mean = mean * torch.where(torch.rand(g, d, generator=gen, device='cuda') < 0.04, 6.0, 0.3)
    return torch.randn(shape, generator=gen, device='cuda', dtype=dtype).add_(mean.to(dtype))


def _pages_of(case, rows, gen):
    """Block tables [B, n] in any order, for caches of `rows` rows a sequence."""
    per = -(-rows // case['page'])
    return torch.randperm(case['batch'] * per, generator=gen, device='cuda').view(case['batch'], per).to(torch.int32)


def _cache(case, rows, gen, dtype):
    """4-bit K and V rows of a full cache, and its block tables (None when dense)."""
    b, g, d = case['batch'], case['kv_heads'], case['dim']
    if case['page']:
        tables = _pages_of(case, rows, gen)
        k, v = (_pack(_rows(gen, (tables.numel(), case['page'], g, d), dtype)) for _ in range(2))
        return k, v, tables
    # Head-major planes seen as [B, rows, Hkv, bytes].
    k, v = (_pack(_rows(gen, (b, rows, g, d), dtype).transpose(1, 2).contiguous()).transpose(1, 2) for _ in range(2))
    return k, v, None


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case['dtype']]
    i32 = dict(dtype=torch.int32, device='cuda')
    b, g, d = case['batch'], case['kv_heads'], case['dim']
    lengths = _lengths(case)
    rng.shuffle(lengths)
    s = dict(op=case['op'], dim=d, dtype=dtype, lengths=torch.tensor(lengths, **i32))
    if case['op'] == 'write':
        n = case['hi']
        s['k'], s['v'] = _rows(gen, (b, n, g, d), dtype), _rows(gen, (b, n, g, d), dtype)
        starts = [max(0, case['behind'] - 7 * i) for i in range(b)]
        s['starts'], s['tables'] = torch.tensor(starts, **i32), None
        capacity, shape = case['behind'] + n, (g, _row_bytes(d))
        if case['page']:
            s['tables'] = _pages_of(case, capacity, gen)
            shape = (s['tables'].numel(), case['page']) + shape
        else:
            shape = (b, capacity) + shape
        s['k4'], s['v4'] = (torch.zeros(shape, dtype=torch.uint8, device='cuda') for _ in range(2))
    elif case['op'] == 'read':
        s['rows'] = case['hi']
        s['k4'], s['v4'], s['tables'] = _cache(case, case['hi'], gen, dtype)
    else:
        t, h = case['nodes'], case['heads']
        s['k4'], s['v4'], s['tables'] = _cache(case, case['hi'] + t, gen, dtype)
        s['q'] = torch.randn(b, t, h, d, generator=gen, device='cuda', dtype=dtype)
        s['scale'], s['context_only'] = 0.5 * d ** -0.5, case['context_only']
        # Without a mask the nodes are a chain: what single tokens and plain drafts use.
        s['mask'] = None
        if t > 1 and not s['context_only'] and case['op'] == 'attention':
            s['mask'] = torch.tensor([_ancestor_words(rng, t) for _ in range(b)], **i32)
    if case['op'] == 'mass':
        # Accepted rows: a path of node numbers for each sequence, its count, and the rows' log-sum-exps.
        counts = _mass_counts(case)
        s['rows'] = torch.tensor([sorted(rng.sample(range(t), c)) + [-1] * (t - c) for c in counts], **i32)
        s['counts'], s['decay'] = torch.tensor(counts, **i32), 0.97
        s['lse'] = torch.full((b, t, h), -math.inf, device='cuda')
        scores, seen, at = _mass_scores(s)
        got = scores.masked_fill(~seen, -math.inf).logsumexp(-1)
        got = got.unflatten(2, (h // g, t)).permute(0, 3, 1, 2).reshape(b, t, h)
        s['lse'].scatter_reduce_(1, at[:, :, None].expand(b, t, h), got, 'amax')        # (-inf where a path has ended)
        s['mass'] = torch.rand(b, g, case['hi'] + t, generator=gen, device='cuda')
    return s


# -------------------------------------------------------------- plain form --
def _codes(x):
    """Codes [..., groups, 32], scales and minima [..., groups, 1] of 16-bit rows, in 32 bits."""
    dtype = x.dtype
    x = x.unflatten(-1, (-1, GROUP)).float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high * 0.5 - low * 0.5) / 7.5).to(dtype).float()          # halves: the difference of two large values
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    q = (x * 0.5 - low * 0.5).double() / (scale * 0.5).double()         # 64 bits: values next to a border
    codes = torch.where(scale > 0, q, 0.0).round().clamp(0, 15)
    finite = scale.isfinite() & x.isfinite().all(-1, keepdim=True)
    return torch.where(finite, codes, 0.0).float(), torch.where(finite, scale, math.nan), torch.where(finite, low, math.nan)


def _values(codes, scale, low, dtype):
    """What codes stand for: [..., D] in the rows' type."""
    return (codes * scale + low).flatten(-2).to(dtype)


def _pack(x):
    """16-bit rows [..., D] as rows of the cache, uint8 [..., bytes]."""
    codes, scale, low = _codes(x)
    code = codes.flatten(-2).to(torch.int16).unflatten(-1, (-1, 2, 2, 2))       # dims 8 w + 4 i + 2 j + h
    code = (code[..., 0, :] + 16 * code[..., 1, :]).transpose(-1, -2).to(torch.uint8).flatten(-3)    # bytes 4 w + 2 h + i
    params = torch.cat([scale, low], -1).to(x.dtype).flatten(-2).view(torch.uint8)
    out = torch.zeros(*x.shape[:-1], _row_bytes(x.shape[-1]), dtype=torch.uint8, device=x.device)
    out[..., :code.shape[-1]] = code
    out[..., code.shape[-1]:code.shape[-1] + params.shape[-1]] = params
    return out


def _unpack(rows, dim, dtype):
    """16-bit rows [..., D] of cache rows."""
    code = rows[..., :dim // 2].unflatten(-1, (-1, 2, 2)).transpose(-1, -2)             # [w, i, h]
    code = torch.stack([code & 15, code >> 4], -2).flatten(-4)                          # [w, i, j, h]
    params = rows[..., dim // 2:dim // 2 + dim // 8].contiguous().view(dtype).unflatten(-1, (-1, 2)).float()
    return _values(code.unflatten(-1, (-1, GROUP)).float(), params[..., :1], params[..., 1:], dtype)


def _dense(rows, tables):
    """[B, rows, Hkv, bytes] of a cache, gathered through its block tables when it is paged."""
    return rows if tables is None else rows[tables.long()].flatten(1, 2)


def _grouped(q, kv_heads):
    """[B, T, H, D] -> [B, Hkv, G * T, D], rows (head of the group, token)."""
    b, t, h, d = q.shape
    return q.view(b, t, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _plain_write(s):
    live = (torch.arange(s['k'].shape[1], device='cuda') < s['lengths'][:, None])[..., None, None]
    return tuple(torch.where(live, _values(*_codes(x), s['dtype']), 0) for x in (s['k'], s['v']))


def _plain_read(s):
    live = (torch.arange(s['rows'], device='cuda') < s['lengths'][:, None])[..., None, None]
    return tuple(torch.where(live, _unpack(_dense(x, s['tables'])[:, :s['rows']], s['dim'], s['dtype']), 0)
                 for x in (s['k4'], s['v4']))


def _plain_attention(s):
    k, v = (_unpack(_dense(x, s['tables']), s['dim'], s['dtype']).float() for x in (s['k4'], s['v4']))
    q = s['q'].float()
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
    return out.to(s['dtype']), lse


def _mass_scores(s):
    """Scores [B, Hkv, G * A, N] of the accepted rows, which keys each sees, and the rows' node numbers."""
    t = s['q'].shape[1]
    g = s['k4'].shape[2]
    at = s['rows'].long().clamp_min(0)
    q = s['q'].gather(1, at[:, :, None, None].expand(*at.shape, *s['q'].shape[2:])).float()
    k = _unpack(_dense(s['k4'], s['tables']), s['dim'], s['dtype']).float()
    scores = _grouped(q, g) @ k.permute(0, 2, 3, 1) * s['scale']
    i = torch.arange(t, device=q.device)
    end = s['lengths'][:, None] + (0 if s['context_only'] else i + 1)
    seen = (torch.arange(k.shape[1], device=q.device) < end.expand(-1, t)[:, :, None]) & (i < s['counts'][:, None])[:, :, None]
    return scores, seen.repeat(1, q.shape[2] // g, 1)[:, None], at


def _plain_mass(s):
    scores, seen, at = _mass_scores(s)
    b, t, h = s['lse'].shape
    g, n = s['mass'].shape[1:]
    lse = _grouped(s['lse'].gather(1, at[:, :, None].expand(b, t, h))[..., None], g)
    added = torch.exp(scores - lse).masked_fill(~seen, 0.0).sum(2)[:, :, :n]
    key = torch.arange(n, device=added.device)
    before = key < s['lengths'][:, None, None]
    fresh = (s['lengths'] + (0 if s['context_only'] else s['counts']))[:, None, None]
    new = torch.where(before, s['decay'] * s['mass'], 0.0) + added
    s['mass'].copy_(torch.where(key < fresh, new, s['mass']))
    return s['mass']


PLAIN = dict(write=_plain_write, read=_plain_read, attention=_plain_attention, mass=_plain_mass)


# -------------------------------------------------------------------- run --
def run(state):
    s = state
    if not own:
        return PLAIN[s['op']](s)
    from slimkv_b200 import cache4
    if s['op'] == 'write':
        # As a prompt's chunk does that goes on with the rows that later steps will see.
        cache4.write(s['k'], s['v'], s['k4'], s['v4'], s['starts'], counts=s['lengths'], block_tables=s['tables'])
        return cache4.read(s['k4'], s['v4'], s['lengths'], s['dtype'], rows=s['k'].shape[1], starts=s['starts'],
                           block_tables=s['tables'])
    if s['op'] == 'read':
        return cache4.read(s['k4'], s['v4'], s['lengths'], s['dtype'], rows=s['rows'], block_tables=s['tables'])
    if s['op'] == 'attention':
        return cache4.attention(s['q'], s['k4'], s['v4'], s['lengths'], s['scale'], mask=s['mask'],
                                block_tables=s['tables'], context_only=s['context_only'])
    return cache4.key_mass(s['q'], s['k4'], s['lse'], s['mass'], s['lengths'], s['scale'], rows=s['rows'],
                           counts=s['counts'], decay=s['decay'], block_tables=s['tables'],
                           context_only=s['context_only'])


# ------------------------------------------------------------------- work --
def work(case):
    op, b, g, d = case['op'], case['batch'], case['kv_heads'], case['dim']
    total = sum(_lengths(case))
    stored = d // 2 + d // 8                            # a row of the cache, without what fills it up
    if op == 'write':
        return dict(bytes=2 * total * g * (2 * d + stored + 2 * d) + 8 * b, flops=12 * 2 * total * g * d)
    if op == 'read':
        return dict(bytes=2 * total * g * (stored + 2 * d) + 4 * b, flops=2 * 2 * total * g * d)
    t, h = case['nodes'], case['heads']
    if op == 'attention':
        rows = total + (0 if case['context_only'] else b * t)
        return dict(bytes=2 * rows * g * stored + b * t * h * (4 * d + 4), flops=4 * t * h * d * total)
    counts = _mass_counts(case)
    picked = sum(counts)
    rows = total + (0 if case['context_only'] else picked)
    flops = sum(2 * c * h * d * n for c, n in zip(counts, _lengths(case)))
    return dict(bytes=rows * g * (stored + 8) + picked * h * (2 * d + 4), flops=flops)


# ------------------------------------------------------------------ exact --
F64 = torch.float64


def _quantised64(x):
    """16-bit rows [n, D] -> what the cache holds for them, rounded to their type, in 64 bits."""
    groups = x.to(F64).reshape(x.shape[0], -1, GROUP)
    low, _ = groups.min(-1, keepdim=True)
    high, _ = groups.max(-1, keepdim=True)
    step = ((high - low) / 15).to(x.dtype).to(F64)
    step[step < 2.0 ** -126] = 0
    away = (groups - low).float().to(F64)               # the format takes this difference in 32 bits
    code = torch.clamp(torch.round(away / step.masked_fill(step == 0, math.inf)), 0, 15)
    return (code * step + low).reshape(x.shape).to(x.dtype).to(F64)


ORDER = [0, 4, 1, 5, 2, 6, 3, 7]                        # where the dims 0..7 stand among the bytes' low and high halves


def _stored64(rows, dim, dtype):
    """What cache rows [n, bytes] stand for, in 64 bits."""
    byte = rows[:, :dim // 2].reshape(rows.shape[0], -1, 4).long()
    halves = torch.cat([byte[..., :1] % 16, byte[..., :1] // 16, byte[..., 1:2] % 16, byte[..., 1:2] // 16,
                        byte[..., 2:3] % 16, byte[..., 2:3] // 16, byte[..., 3:] % 16, byte[..., 3:] // 16], -1)
    code = halves[..., ORDER].reshape(rows.shape[0], -1, GROUP).to(F64)
    pair = rows[:, dim // 2:dim // 2 + dim // 8].clone().view(dtype).reshape(rows.shape[0], -1, 2).to(F64)
    return (code * pair[:, :, 0, None] + pair[:, :, 1, None]).reshape(rows.shape[0], dim).to(dtype).to(F64)


def _rows64(s, name, b, head, n):
    if s['tables'] is not None:
        page = s[name].shape[1]
        flat = s[name][s['tables'][b, :-(-n // page)].long(), :, head].flatten(0, 1)[:n]
    else:
        flat = s[name][b, :n, head]
    return _stored64(flat, s['dim'], s['dtype'])


def exact(case, seed):
    s = prepare(case, seed)
    lengths = s['lengths'].tolist()
    g, d = case['kv_heads'], case['dim']
    if case['op'] in ('write', 'read'):
        outs = []
        for name in 'kv':
            out = torch.zeros(case['batch'], case['hi'], g, d, dtype=F64, device='cuda')
            for b, n in enumerate(lengths):
                for j in range(g):
                    out[b, :n, j] = _quantised64(s[name][b, :n, j]) if case['op'] == 'write' else _rows64(s, name + '4', b, j, n)
            outs.append(out)
        return tuple(outs)
    t, h = case['nodes'], case['heads']
    per = h // g
    if case['op'] == 'attention':
        out = torch.zeros(case['batch'], t, h, d, dtype=F64, device='cuda')
        lse = torch.zeros(case['batch'], t, h, dtype=F64, device='cuda')
    else:
        mass = s['mass'].to(F64)
    for b, n in enumerate(lengths):
        if case['op'] == 'attention':
            rows = n + (0 if case['context_only'] else t)
            seen = torch.ones(t, rows, dtype=torch.bool, device='cuda')
            if not case['context_only']:
                if s['mask'] is None:
                    seen[:, n:] = torch.ones(t, t, device='cuda').tril().bool()
                else:
                    words = s['mask'][b, :, 0].tolist()
                    seen[:, n:] = torch.tensor([[bool(w >> i & 1) for i in range(t)] for w in words], device='cuda')
            for j in range(g):
                k, v = _rows64(s, 'k4', b, j, rows), _rows64(s, 'v4', b, j, rows)
                for i in range(per):
                    x = (s['q'][b, :, j * per + i].to(F64) @ k.T * s['scale']).masked_fill(~seen, -math.inf)
                    lse[b, :, j * per + i] = x.logsumexp(-1)
                    out[b, :, j * per + i] = x.softmax(-1) @ v
        else:
            count = int(s['counts'][b])
            end = n + (0 if case['context_only'] else count)
            mass[b, :, :n] *= s['decay']
            mass[b, :, n:end] = 0
            for j in range(g):
                k = _rows64(s, 'k4', b, j, end)
                for i, r in enumerate(s['rows'][b, :count].tolist()):
                    m = n if case['context_only'] else n + i + 1
                    x = s['q'][b, r, j * per:(j + 1) * per].to(F64) @ k[:m].T * s['scale']
                    mass[b, j, :m] += torch.exp(x - s['lse'][b, r, j * per:(j + 1) * per, None].to(F64)).sum(0)
    return (out, lse) if case['op'] == 'attention' else mass
