"""A cache kept within a budget by the attention its keys receive.

* :func:`key_mass` — adds the attention weights that the step's accepted rows
  gave each key to its running mass;
* :func:`evict` — keeps the sinks, the recent rows and the rows of the largest
  mass, in order, in a cache of ``keep`` rows.

Beacon latents carry no position, and raw keys are cached rotated, so a row
can leave without touching the others.  The reference never drops a cached
row.  Torch wrappers over ``include/slimkv_b200.h``; there is no CPU path.
"""
from ctypes import byref

import torch

from . import _lib
from .tree import _TYPES, _check_rows, _i32, _refuse, _run, _run_in_workspace, fill_cache


def _plane(t, dtype, device, batch, heads, rows, strides, what):
    """Pointer of a [B, Hkv, rows] plane (``rows``: at least so many), its strides into ``strides``."""
    shape = t.shape
    st = t.stride()
    if not (t.device == device and t.dtype == dtype and len(shape) == 3 and shape[0] == batch and shape[1] == heads and
            shape[2] >= rows and st[2] == 1):
        _refuse('%s must be %s [%d, %d, >= %d] on %s with contiguous rows', what, dtype, batch, heads, rows, device)
    strides[0], strides[1] = st[0], st[1]
    return t.data_ptr()


def mass_args(q, k, lse, mass, lengths, scale, rows, counts, decay, block_tables, context_only, wait_limit_ns,
              cache_type=None, cache_dim=None):
    """``slimkv_key_mass_args`` of a call.  ``cache_type``: that of the keys'
    elements (default: q's), ``cache_dim`` of them a row (default: the queries')."""
    kind = q.dtype
    if not (q.is_cuda and q.dim() == 4 and kind in (torch.bfloat16, torch.float16)):
        _refuse('q must be bf16 or fp16 [B, T, H, D] on CUDA')
    batch, t, heads, dim = q.shape
    qs, dev = q.stride(), q.device
    _check_rows(k, k, 4)
    if qs[3] != 1 or k.dtype != (cache_type or kind) or k.shape[3] != (cache_dim or dim) or k.device != dev:
        _refuse('q needs a contiguous last dimension, and a cache of its type, dim and device')
    if not (lse.device == dev and lse.dtype == torch.float32 and lse.shape == (batch, t, heads) and lse.is_contiguous()):
        _refuse('lse must be contiguous fp32 [B, T, H] on q\'s device')
    a = _lib.KeyMassArgs()
    fill_cache(a.cache, k, k, block_tables, batch)
    kv_heads = k.shape[2]
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim, a.type = batch, t, heads, kv_heads, dim, _TYPES[kind]
    a.q, a.lse, a.lengths = q.data_ptr(), lse.data_ptr(), _i32(lengths, (batch,), dev, 'lengths')
    x = a.q_stride
    x[0], x[1], x[2] = qs[:3]
    if rows is not None:
        a.rows = _i32(rows, (batch, t), dev, 'rows')
    if counts is not None:
        a.counts = _i32(counts, (batch,), dev, 'counts')
    a.mass = _plane(mass, torch.float32, dev, batch, kv_heads, 0, a.mass_stride, 'mass')
    a.mass_rows, a.context_only, a.scale, a.decay, a.wait_limit_ns = mass.shape[2], bool(context_only), scale, decay, wait_limit_ns
    return a


def key_mass(q, k, lse, mass, lengths, scale, rows=None, counts=None, decay=1.0, block_tables=None,
             context_only=False, wait_limit_ns=0):
    """Accumulates attention weights per key, in place (``slimkv_key_mass``).

    ``mass [B, Hkv, rows]`` (fp32): entry n becomes ``decay * mass[n] + sum_i
    sum_h exp(scale * q[b, r_i, h] . k[b, n] - lse[b, r_i, h])`` over the
    accepted rows ``r_i = rows[b, i]``, i < ``counts[b]`` (int32 ``[B, T]`` /
    ``[B]``: ``path`` and ``count`` of ``tree.tree_accept``; default: all rows)
    and the heads of the KV head's group, for the ``lengths[b]`` old rows and
    the accepted rows themselves, which follow them after ``tree.tree_commit``
    (row i sees n <= lengths[b] + i; a new row's mass starts from 0).
    ``context_only``: only the ``lengths[b]`` rows (Beacon latents).  ``q [B, T,
    H, D]`` and ``lse [B, T, H]`` as ``tree.tree_attention`` took and returned
    them; for a key set attended in parts, pass the merged lse.  The lse is taken
    as it is: a row that saw no key (lse -inf) would make the masses of its keys
    infinite for good, so leave it out of ``rows``; where ``tree_attention`` had
    ``nodes`` and every row counts, ``counts=nodes`` does.  Other entries of
    ``mass`` keep their values.  Returns ``mass``.
    """
    a = mass_args(q, k, lse, mass, lengths, scale, rows, counts, decay, block_tables, context_only, wait_limit_ns)
    _run(q.device, _lib.load().slimkv_key_mass, byref(a))
    return mass


def evict(k, v, mass, positions, lengths, keep, sinks=0, recent=0, block_tables=None, out=None):
    """Keeps ``min(lengths[b], keep)`` rows of each (sequence, KV head)
    (``slimkv_evict``).

    ``k`` / ``v [B, rows, Hkv, D]`` (or pages with ``block_tables``; any 1-, 2-
    or 4-byte type), ``mass [B, Hkv, rows]`` fp32, ``positions`` int32 of that
    shape or None.  The first ``sinks`` and the last ``recent`` rows stay, then
    those of the largest mass (ties: the lowest row), all in their order.
    Returns ``(k, v, mass, positions, lengths)`` of ``keep`` rows, zeros past a
    sequence's new length; ``out = (k, v, mass, positions)`` gives buffers (at
    least ``keep`` rows, nowhere over the inputs') to write instead of new ones.
    """
    _check_rows(k, v, 4)
    if mass.dim() != 3:
        _refuse('mass must be [B, Hkv, rows]')
    batch, heads, dim, dim_v, dev = mass.shape[0], k.shape[2], k.shape[3], v.shape[3], k.device
    a = _lib.EvictArgs()
    fill_cache(a.src, k, v, block_tables, batch)
    keep = int(keep)
    if keep < 1:
        _refuse('keep must be positive')
    if out is None:
        # Each (sequence, head) a contiguous run of rows.
        rows = heads * keep
        out_k = torch.empty_strided((batch, keep, heads, dim), (rows * dim, dim, keep * dim, 1), dtype=k.dtype, device=dev)
        out_v = torch.empty_strided((batch, keep, heads, dim_v), (rows * dim_v, dim_v, keep * dim_v, 1), dtype=k.dtype, device=dev)
        plane = (batch, heads, keep), (rows, keep, 1)
        out_mass = torch.empty_strided(*plane, dtype=torch.float32, device=dev)
        out_positions = None if positions is None else torch.empty_strided(*plane, dtype=torch.int32, device=dev)
        c = a.dst
        c.k, c.v, c.rows = out_k.data_ptr(), out_v.data_ptr(), keep
        x, y = c.k_stride, c.v_stride
        x[0], x[1], x[2] = rows * dim, dim, keep * dim
        y[0], y[1], y[2] = rows * dim_v, dim_v, keep * dim_v
        a.out_mass = out_mass.data_ptr()
        a.out_mass_stride[0], a.out_mass_stride[1] = rows, keep
        if positions is not None:
            a.out_positions = out_positions.data_ptr()
            a.out_positions_stride[0], a.out_positions_stride[1] = rows, keep
    else:
        out_k, out_v, out_mass, out_positions = out
        _check_rows(out_k, out_v, 4)
        if not (out_k.shape[0] == batch and out_k.shape[2:] == k.shape[2:] and out_v.shape[2:] == v.shape[2:] and
                out_k.dtype == k.dtype and out_k.device == dev and out_k.shape[1] >= keep):
            _refuse('out caches must be like the caches, with keep rows')
        if (positions is None) != (out_positions is None):
            _refuse('positions and their output go together')
        fill_cache(a.dst, out_k, out_v, None, batch)
        a.out_mass = _plane(out_mass, torch.float32, dev, batch, heads, keep, a.out_mass_stride, 'out mass')
        if positions is not None:
            a.out_positions = _plane(out_positions, torch.int32, dev, batch, heads, keep, a.out_positions_stride, 'out positions')
    a.batch, a.kv_heads, a.dim_qk, a.dim_v, a.elem_bytes = batch, heads, dim, dim_v, k.element_size()
    a.mass, a.mass_rows = _plane(mass, torch.float32, dev, batch, heads, 0, a.mass_stride, 'mass'), mass.shape[2]
    if positions is not None:
        a.positions = _plane(positions, torch.int32, dev, batch, heads, mass.shape[2], a.positions_stride, 'positions')
    new_lengths = torch.empty_strided((batch,), (1,), dtype=torch.int32, device=dev)
    a.lengths, a.new_lengths = _i32(lengths, (batch,), dev, 'lengths'), new_lengths.data_ptr()
    a.keep, a.sinks, a.recent = keep, sinks, recent
    lib = _lib.load()
    _run_in_workspace(dev, lib.slimkv_evict_workspace_size, lib.slimkv_evict, a)
    return out_k, out_v, out_mass, out_positions, new_lengths
