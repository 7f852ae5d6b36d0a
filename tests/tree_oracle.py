"""Plain 64-bit forms of the speculative-decoding and eviction operators, and
the error bounds of their kernels (tests only)."""
import math

import torch

F64 = torch.float64
# Unit roundoffs of the 16-bit types (8- and 11-bit significands): a probability
# and an output are each rounded to the type once.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ancestors(parents):
    """[T][T] truth values: node t sees node i (itself and its ancestors)."""
    seen = []
    for t, p in enumerate(parents):
        row = list(seen[p]) if 0 <= p < t else [False] * len(parents)
        row[t] = True
        seen.append(row)
    return torch.tensor(seen)


def words_of(seen):
    """int32 mask words of a [T, T] truth table."""
    t = seen.shape[-1]
    n = (t + 31) // 32
    out = torch.zeros(*seen.shape[:-1], n, dtype=torch.int64)
    for i in range(t):
        out[..., i // 32] |= seen[..., i].long() << (i % 32)
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)


def rows_of(cache, tables, b, n):
    """The first n rows [n, Hkv, D] of sequence b, in 64 bits on the CPU."""
    if tables is not None:
        page = cache.shape[1]
        used = tables[b, :-(-n // page)].long()
        return cache[used].flatten(0, 1)[:n].to(F64).cpu() if n else cache[:0].flatten(0, 1).to(F64).cpu()
    return cache[b if cache.shape[0] > 1 else 0, :n].to(F64).cpu()


def attention(q, k, v, lengths, scale, seen=None, nodes=None, tables=None, context_only=False):
    """(out, lse, bound of out, bound of lse); seen [B or 1, T, T] (default: a chain)."""
    B, T, H, D = q.shape
    G = k.shape[2]
    kind = q.dtype
    q = q.to(F64).cpu()
    out = torch.zeros(B, T, H, v.shape[3], dtype=F64)
    lse = torch.full((B, T, H), -math.inf, dtype=F64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        n, m = int(lengths[b]), T if nodes is None else int(nodes[b])
        rows = n + (0 if context_only else m)
        kb, vb = rows_of(k, tables, b, rows), rows_of(v, tables, b, rows)
        for t in range(m):
            vis = torch.zeros(rows, dtype=torch.bool)
            vis[:n] = True
            if not context_only:
                vis[n:] = (torch.arange(m) <= t) if seen is None else seen[b if seen.shape[0] > 1 else 0, t, :m]
            if not vis.any():
                continue
            for h in range(H):
                kk, vv = kb[vis, h * G // H], vb[vis, h * G // H]
                s = kk @ q[b, t, h] * scale
                lse[b, t, h] = s.logsumexp(-1)
                p = s.softmax(-1)
                out[b, t, h] = p @ vv
                # fp32 accumulation of D exact products, exponential and sum in fp32.
                e = D * 2.0 ** -24 * float((kk.abs() @ q[b, t, h].abs()).max()) * scale + 1e-5
                tol_lse[b, t, h] = e
                u = ROUND[kind]
                weight = p @ vv.abs()
                # P and the output rounded to the type; fp16 probabilities below 2^-14 by at most 2^-25.
                tol[b, t, h] = (u + 2 * e) * weight + u * out[b, t, h].abs() + 1e-6
                if kind == torch.float16:
                    tol[b, t, h] += len(kk) * 2.0 ** -25 * vv.abs().amax(0)
    return out, lse, tol, tol_lse


def check_attention(got, want):
    """A factor of 1.05 over the bounds leaves room for the terms of second order."""
    out, lse = got[0].to(F64).cpu(), got[1].to(F64).cpu()
    o, l, tol, tol_lse = want
    fine = o.isfinite()
    assert torch.equal(out.isnan(), o.isnan())
    assert torch.equal(out[~fine & ~o.isnan()], o[~fine & ~o.isnan()])
    off = ((out - o).abs() - 1.05 * tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f'out off its bound by {off.max():.3e}'
    empty = l == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
    live = ~empty & l.isfinite()
    assert ((lse - l).abs() <= 1.05 * tol_lse)[live].all(), (lse - l).abs()[live].max()


def mass(q, k, lse, old, lengths, scale, rows=None, counts=None, decay=1.0, tables=None, context_only=False):
    """(mass, bound)."""
    B, T, H, D = q.shape
    G = k.shape[2]
    new, tol = old.to(F64).cpu(), torch.zeros(old.shape, dtype=F64)
    q, lse = q.to(F64).cpu(), lse.to(F64).cpu()
    for b in range(B):
        n, c = int(lengths[b]), T if counts is None else int(counts[b])
        end = n + (0 if context_only else c)
        kb = rows_of(k, tables, b, end)
        new[b, :, :n] *= decay
        new[b, :, n:end] = 0
        tol[b, :, :end] = 2.0 ** -22 * new[b, :, :end].abs() + 1e-30
        for i in range(c):
            r = i if rows is None else int(rows[b, i])
            m = n if context_only else n + i + 1
            for h in range(H):
                x = lse[b, r, h]
                if x == math.inf:
                    continue
                g = h * G // H
                p = torch.exp(kb[:m, g] @ q[b, r, h] * scale - x)
                new[b, g, :m] += p
                # The score's fp32 accumulation, the exponent's rounding, 2^-22 of the exponential, the sum's.
                e = D * 2.0 ** -24 * (kb[:m, g].abs() @ q[b, r, h].abs()) * scale
                tol[b, g, :m] += p * (e + 2.0 ** -22 * (x.abs() + 40) + (c * H // G + 2) * 2.0 ** -24)
    return new, tol


def evict(k, v, mass, positions, lengths, keep, sinks=0, recent=0, tables=None):
    """(k, v, mass, positions, lengths), all rows exact."""
    B, G = mass.shape[:2]
    D, Dv = k.shape[3], v.shape[3]
    ok, ov = torch.zeros(B, keep, G, D, dtype=F64), torch.zeros(B, keep, G, Dv, dtype=F64)
    om, op = torch.zeros(B, G, keep, dtype=F64), torch.zeros(B, G, keep, dtype=torch.int32)
    ol = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = int(lengths[b])
        ol[b] = min(n, keep)
        kb, vb = rows_of(k, tables, b, n), rows_of(v, tables, b, n)
        for g in range(G):
            m = mass[b, g, :n].to(F64).cpu()

            def rank(i):
                if i < sinks or i >= n - recent:
                    return (0, 0.0, i)
                x = float(m[i])
                return (1, 0.0, i) if math.isnan(x) else (2, -x, i)
            kept = sorted(sorted(range(n), key=rank)[:keep])
            ok[b, :len(kept), g], ov[b, :len(kept), g] = kb[kept, g], vb[kept, g]
            om[b, g, :len(kept)] = m[kept]
            if positions is not None:
                op[b, g, :len(kept)] = positions[b, g].cpu()[kept]
    return ok, ov, om, op, ol


def accept(logits, tokens, parents, nodes=None):
    """(path, count, next) with python's own comparisons."""
    B, T, V = logits.shape
    x = logits.to(F64).cpu()
    path, count, after = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32), torch.full((B,), -1)
    for b in range(B):
        n = T if nodes is None else int(nodes[b])
        cur = 0 if n else -1
        while cur >= 0:
            path[b, count[b]] = cur
            count[b] += 1
            row = x[b, cur]
            nan = row.isnan().nonzero()
            best = int(nan[0]) if len(nan) else int((row == row.max()).nonzero()[0])
            after[b] = best
            cur = next((c for c in range(cur + 1, n) if int(parents[b, c]) == cur and int(tokens[b, c]) == best), -1)
    return path, count, after
